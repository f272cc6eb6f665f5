// Gradient of an embedding table, summed by sorted tokens: grad[v, :] (+)= scale * sum over the positions t with
// ids[t] == v of dout[t, :], every sum in one fixed order and no atomics.
//
// Three launches. (1) One cluster sorts the pairs (id, position) by id, equal ids by position: a radix sort from the
// low digit up whose per-warp digit counts live in shared memory and whose per-block totals are read through
// distributed shared memory. (2) Blocks walk `chunk` sorted positions each, so a frequent token is spread over many
// blocks; a run of equal ids inside a chunk is written at once, one that crosses a border leaves an fp32 partial sum.
// (3) The chunk where such a run begins adds its partial sums in order. dout is read once and every present row of
// the table is touched once. Ids outside the vocabulary sort behind all others and are left out.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "tx_host.h"

namespace cg = cooperative_groups;

namespace {

constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kMaxDigits = 1024;              // 10 bits a pass
constexpr int kSortCluster = 8;

struct SortArgs {
  const void* ids;
  int ids64;
  int T, V;
  int passes, bits;           // digit width
  int2* a;                    // [T]; the sorted pairs end up here
  int2* b;                    // [T]
};

// Pair `i` of the input of pass `p`.
__device__ __forceinline__ int2 sort_load(const SortArgs& s, const int2* src, int p, int i) {
  if (p > 0) return src[i];
  const long long id = s.ids64 ? static_cast<const long long*>(s.ids)[i] : static_cast<const int*>(s.ids)[i];
  return make_int2((id < 0 || id >= s.V) ? s.V : static_cast<int>(id), i);
}

// Every warp owns a contiguous part of its block's part of the pairs, which keeps each pass stable.
__global__ void __launch_bounds__(kSortThreads, 1) sort_ids_kernel(SortArgs s) {
  extern __shared__ int hist[];                                    // [warps][digits]
  __shared__ int total[kMaxDigits];                                // of this block, read by the others
  __shared__ int base[kMaxDigits];
  __shared__ int warp_sums[kSortWarps];
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int digits = 1 << s.bits;
  const int parts = blocks * kSortWarps;
  const int per = (s.T + parts - 1) / parts;
  const int lo = min(s.T, (rank * kSortWarps + warp) * per), hi = min(s.T, lo + per);
  int* mine = hist + warp * digits;
  for (int p = 0; p < s.passes; ++p) {
    // the last pass writes `a`
    int2* dst = ((s.passes - 1 - p) & 1) ? s.b : s.a;
    const int2* src = ((s.passes - 1 - p) & 1) ? s.a : s.b;
    const int shift = p * s.bits;
    for (int d = lane; d < digits; d += 32) mine[d] = 0;
    __syncwarp();
    for (int i0 = lo; i0 < hi; i0 += 32) {
      const int i = i0 + lane;
      const unsigned live = __ballot_sync(0xffffffffu, i < hi);
      if (i < hi) {
        const int d = (sort_load(s, src, p, i).x >> shift) & (digits - 1);
        const unsigned same = __match_any_sync(live, d);
        if ((same & ((1u << lane) - 1)) == 0) mine[d] += __popc(same);
      }
      __syncwarp();
    }
    __syncthreads();
    int sum = 0;
    if (tid < digits) {
      for (int w = 0; w < kSortWarps; ++w) {
        const int n = hist[w * digits + tid];
        hist[w * digits + tid] = sum;
        sum += n;
      }
      total[tid] = sum;
    }
    cluster.sync();
    int before = 0, all = 0;
    if (tid < digits) {
      for (int r = 0; r < blocks; ++r) {
        const int n = cluster.map_shared_rank(total, r)[tid];
        if (r < rank) before += n;
        all += n;
      }
    }
    int scan = all;                                                // inclusive over the digits
    for (int o = 1; o < 32; o <<= 1) {
      const int n = __shfl_up_sync(0xffffffffu, scan, o);
      if (lane >= o) scan += n;
    }
    if (lane == 31) warp_sums[warp] = scan;
    __syncthreads();
    if (warp == 0) {
      int v = warp_sums[lane];
      for (int o = 1; o < 32; o <<= 1) {
        const int n = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += n;
      }
      warp_sums[lane] = v;
    }
    __syncthreads();
    if (tid < digits) base[tid] = scan - all + (warp ? warp_sums[warp - 1] : 0) + before;
    __syncthreads();
    for (int i0 = lo; i0 < hi; i0 += 32) {
      const int i = i0 + lane;
      const unsigned live = __ballot_sync(0xffffffffu, i < hi);
      int2 pair;
      unsigned same = 0;
      int d = 0, at = 0;
      if (i < hi) {
        pair = sort_load(s, src, p, i);
        d = (pair.x >> shift) & (digits - 1);
        same = __match_any_sync(live, d);
        const unsigned below = same & ((1u << lane) - 1);
        at = base[d] + mine[d] + __popc(below);
        dst[at] = pair;
      }
      __syncwarp();
      if (i < hi && (same & ((1u << lane) - 1)) == 0) mine[d] += __popc(same);
      __syncwarp();
    }
    cluster.sync();                                                // pairs written, totals read
  }
}

__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&f)[8]) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

struct GradArgs {
  const int2* pairs;          // [T] sorted
  const __nv_bfloat16* dout;  // [T, D]
  float* partial;             // [2 * chunks, D]: sum of a run that came in, sum of a run that begins and goes on
  void* grad;                 // [V, D]
  int T, V, D, chunk;
  float scale;
  int vec;                    // grad is 16-byte aligned (a view into a flat buffer may not be)
};

// One row of the table is written by exactly one thread per column.
__device__ __forceinline__ void store_row(float* dst, const float (&v)[8], float scale, int vec) {
  if (!vec) {
#pragma unroll
    for (int e = 0; e < 8; ++e) dst[e] += v[e] * scale;
    return;
  }
  float4* p = reinterpret_cast<float4*>(dst);
  float4 a = p[0], b = p[1];
  a.x += v[0] * scale; a.y += v[1] * scale; a.z += v[2] * scale; a.w += v[3] * scale;
  b.x += v[4] * scale; b.y += v[5] * scale; b.z += v[6] * scale; b.w += v[7] * scale;
  p[0] = a;
  p[1] = b;
}
__device__ __forceinline__ void store_row(__nv_bfloat16* dst, const float (&v)[8], float scale, int vec) {
  if (!vec) {
#pragma unroll
    for (int e = 0; e < 8; ++e) dst[e] = __float2bfloat16_rn(v[e] * scale);
    return;
  }
  uint4 u;
  __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(v[2 * i] * scale, v[2 * i + 1] * scale);
  *reinterpret_cast<uint4*>(dst) = u;
}

constexpr int kMaxChunk = 32;

// Block (chunk, column tile); a thread owns 8 columns.
template <typename GT>
__global__ void sum_runs_kernel(GradArgs g) {
  __shared__ int2 sh[kMaxChunk + 2];                               // with the neighbours on both sides
  const int lo = blockIdx.x * g.chunk, n = min(g.chunk, g.T - lo);
  for (int i = threadIdx.x; i < n + 2; i += blockDim.x) {
    const int at = lo - 1 + i;
    sh[i] = (at >= 0 && at < g.T) ? g.pairs[at] : make_int2(-1, 0);
  }
  __syncthreads();
  const int col = (blockIdx.y * blockDim.x + threadIdx.x) * 8;
  if (col >= g.D) return;
  const int2* run = sh + 1;
  float acc[8] = {};
  for (int i0 = 0; i0 < n; i0 += 4) {
    float v[4][8];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (i0 + u < n) load8(g.dout + static_cast<long long>(run[i0 + u].y) * g.D + col, v[u]);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = i0 + u;
      if (i >= n) break;
      const int id = run[i].x;
      if (id >= g.V) return;                                       // only ids outside the vocabulary follow
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] += v[u][e];
      if (i + 1 < n && run[i + 1].x == id) continue;
      const bool in = run[-1].x == id, on = run[n].x == id;        // came in from the left, goes on to the right
      if (in || on) {
        float4* p = reinterpret_cast<float4*>(g.partial + (2ll * blockIdx.x + (in ? 0 : 1)) * g.D + col);
        p[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
        p[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
      } else {
        store_row(static_cast<GT*>(g.grad) + static_cast<long long>(id) * g.D + col, acc, g.scale, g.vec);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] = 0.f;
    }
  }
}

constexpr int kJoinGroups = 32;      // chunks of a run are summed in this many contiguous parts

// Block (chunk, 64 columns): 8 threads across, kJoinGroups parts. Only the chunk where a crossing run begins works.
template <typename GT>
__global__ void __launch_bounds__(8 * kJoinGroups) join_runs_kernel(GradArgs g) {
  __shared__ float sh[kJoinGroups][8][8];
  const int last = min(g.T, (static_cast<int>(blockIdx.x) + 1) * g.chunk) - 1;
  if (last + 1 >= g.T) return;
  const int id = g.pairs[last].x;
  if (id >= g.V || g.pairs[last + 1].x != id) return;
  const int lo = blockIdx.x * g.chunk;
  if (lo > 0 && g.pairs[lo - 1].x == id) return;                   // it began further left
  int a = last + 1, b = g.T;                                       // first position behind the run
  while (a < b) {
    const int mid = a + (b - a) / 2;
    if (g.pairs[mid].x == id) a = mid + 1; else b = mid;
  }
  const int end = (a - 1) / g.chunk;                               // the chunk that holds its last position
  const int count = end - static_cast<int>(blockIdx.x) + 1;
  const int tx = threadIdx.x & 7, part = threadIdx.x >> 3;
  const int col = blockIdx.y * 64 + tx * 8;
  const int per = (count + kJoinGroups - 1) / kJoinGroups;
  float acc[8] = {};
  if (col < g.D) {
    for (int i = part * per; i < min(count, (part + 1) * per); ++i) {
      const float4* p = reinterpret_cast<const float4*>(
          g.partial + (2ll * (blockIdx.x + i) + (i == 0 ? 1 : 0)) * g.D + col);
      const float4 x = p[0], y = p[1];
      acc[0] += x.x; acc[1] += x.y; acc[2] += x.z; acc[3] += x.w;
      acc[4] += y.x; acc[5] += y.y; acc[6] += y.z; acc[7] += y.w;
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) sh[part][tx][e] = acc[e];
  __syncthreads();
  if (part != 0 || col >= g.D) return;
  for (int q = 1; q < kJoinGroups; ++q)
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] += sh[q][tx][e];
  store_row(static_cast<GT*>(g.grad) + static_cast<long long>(id) * g.D + col, acc, g.scale, g.vec);
}

int chunk_of(int T) {
  // a few chunks per SM while there are few tokens, at most kMaxChunk positions
  const int c = (T + 4 * txh::sm_count() - 1) / (4 * txh::sm_count());
  return c < 4 ? 4 : (c > kMaxChunk ? kMaxChunk : c);
}

template <typename GT>
int launch_grad(const GradArgs& g, cudaStream_t s) {
  const int chunks = (g.T + g.chunk - 1) / g.chunk;
  const int threads = min(256, (g.D / 8 + 31) / 32 * 32);
  sum_runs_kernel<GT><<<dim3(chunks, (g.D / 8 + threads - 1) / threads), threads, 0, s>>>(g);
  join_runs_kernel<GT><<<dim3(chunks, (g.D + 63) / 64), 8 * kJoinGroups, 0, s>>>(g);
  return cudaGetLastError() == cudaSuccess ? 0 : 400;
}

}  // namespace

// Bytes of workspace for T tokens of D columns (16-byte aligned).
extern "C" long long tx_embedding_grad_workspace(int T, int D) {
  const long long chunks = (T + chunk_of(T) - 1) / chunk_of(T);
  return 2 * ((8ll * T + 15) / 16 * 16) + 2 * chunks * D * 4;
}

// ids int64 or int32 [T], dout bf16 [T, D] with D a multiple of 8. grad_bf16 == 0: grad is fp32 and added to; else it
// is bf16 and the present rows are overwritten (the caller has zeroed the others).
extern "C" int tx_embedding_grad(const void* ids, int ids64, const void* dout, void* grad, int grad_bf16, int T, int D,
                                 int V, float scale, void* workspace, cudaStream_t s) {
  if (D % 8 || D <= 0 || V <= 0 || V > 0x3fffffff) return 1;
  if (T <= 0) return 0;
  int2* a = static_cast<int2*>(workspace);
  int2* b = a + (T + 1ll) / 2 * 2;
  SortArgs so{ids, ids64, T, V, 1, 1, a, b};
  int bits = 1;
  while ((V >> bits) != 0) ++bits;                                 // V itself marks ids outside
  so.passes = (bits + 9) / 10;
  so.bits = (bits + so.passes - 1) / so.passes;
  const int bytes = kSortWarps * (1 << so.bits) * 4;
  static txh::DeviceFlag flag;
  if (!flag.cur()) {
    if (cudaFuncSetAttribute(sort_ids_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             kSortWarps * kMaxDigits * 4) != cudaSuccess) return 401;
    flag.cur() = true;
  }
  const int blocks = T <= 4096 ? 1 : kSortCluster;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(kSortThreads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = blocks;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, sort_ids_kernel, so) != cudaSuccess) return 402;
  const GradArgs g{a, static_cast<const __nv_bfloat16*>(dout), reinterpret_cast<float*>(b + (T + 1ll) / 2 * 2), grad, T,
                   V, D, chunk_of(T), scale, reinterpret_cast<uintptr_t>(grad) % 16 == 0};
  return grad_bf16 ? launch_grad<__nv_bfloat16>(g, s) : launch_grad<float>(g, s);
}
