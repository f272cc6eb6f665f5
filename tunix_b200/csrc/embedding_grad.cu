// Gradient of an embedding table, summed by sorted tokens: grad[v, :] (+)= scale * sum over the positions t with
// ids[t] == v of dout[t, :], every sum in fp32 and in one fixed order. Atomics (a reduction into the fp32 buffer, places
// in the list of long runs) only where their order cannot matter: each element gets one addition.
//
// Launches. (1) The pairs (id, position) are sorted by id, equal ids by position. Few tokens: every pair counts the
// pairs before it. More: one cluster, a radix sort from the low digit up whose per-warp digit counts live in shared
// memory and whose per-block totals are read through distributed shared memory (12 us for 16384 tokens, 27 us for
// 65536: latency of its few steps). A new gradient is cleared while the ids are sorted. (2) Blocks walk `chunk` sorted
// positions each. A run of equal ids is summed by the block where it begins, also a little into the next chunk; a run
// that covers a whole chunk (a frequent token, the padding id) is summed by every block it touches, into fp32 partial
// sums, so that one token cannot keep a block busy alone. (3) The partial sums of such a run are added in order. dout
// is read once and every present row of the table is touched once. Ids outside the vocabulary sort behind all others
// and are left out.
//
// Blocks of (2) and (3) are launched before their predecessor ends and wait for it on the device (with plain launches 4
// and 5 us more in the two cases below, 1 us of 7 for 512 tokens). Fetching a part of dout into L2 while the ids are
// sorted gained nothing.
//
// 16384 tokens x 4096 into an fp32 buffer: 96 us (134 MB of dout and 115 MB of rows read and written: 3.8 TB/s; latency
// of the sums, whose next rows are asked for when the last ones have come).
// 65536 x 1152, half of them one id, new table of 262144 rows: 145 us, of which 82 us write the table (604 MB).
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "tx_host.h"
#include "tx_ptx.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr int kMaxTokens = 0x7fff0000;        // indices run past the last token by a tile of the sort at most
constexpr int kSortThreads = 512;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kMaxDigits = 1024;              // 10 bits a pass
constexpr int kSortCluster = 8;
constexpr int kClearThreads = 512;
constexpr int kSortTile = 16;                 // pairs a lane has in flight
// Up to here every pair counts the pairs before it, from there on the radix sort (whole gradient of 64 columns, us:
// 512 tokens 6.9 and 12.8; 4096 tokens 12.4 and 13.8; 8192 tokens 28.8 and 16.6).
constexpr int kCountTokens = 4096;
constexpr int kCountThreads = 256;
constexpr int kCountPer = 8;                  // threads per pair

struct SortArgs {
  const void* ids;
  int ids64;
  int T, V;
  int passes;
  int2* a;                    // [T]; the sorted pairs end up here
  int2* b;                    // [T]
  int* n_long;                // set to 0 here: length of the list of long runs
  uint4* zero;                // a new gradient (n_zero vectors) that is cleared meanwhile, or none
  long long n_zero;
  int sort_blocks;            // of the counting sort; blocks behind these clear
};

// One block's tile. Tiles of 16 KB whose blocks end at once: 7.4 TB/s, where a few blocks per SM that loop over them
// write 6.1 TB/s.
constexpr int kClearTile = 1024;
__device__ __forceinline__ void clear_tile(const SortArgs& s, long long tile) {
  for (int i = threadIdx.x; i < kClearTile; i += blockDim.x) {
    const long long at = tile * kClearTile + i;
    if (at < s.n_zero) s.zero[at] = make_uint4(0, 0, 0, 0);
  }
}

// Ids outside the vocabulary become V.
__device__ __forceinline__ int id_at(const SortArgs& s, int i) {
  const long long id = s.ids64 ? static_cast<const long long*>(s.ids)[i] : static_cast<const int*>(s.ids)[i];
  return (id < 0 || id >= s.V) ? s.V : static_cast<int>(id);
}

// Pair `i` of the input of pass `p`.
__device__ __forceinline__ int2 sort_load(const SortArgs& s, const int2* src, int p, int i) {
  return p > 0 ? src[i] : make_int2(id_at(s, i), i);
}

__global__ void __launch_bounds__(kCountThreads) count_sort_kernel(SortArgs s) {
  __shared__ int4 ids4[kCountTokens / 4];
  int* ids = reinterpret_cast<int*>(ids4);
  if (static_cast<int>(blockIdx.x) >= s.sort_blocks) {
    clear_tile(s, blockIdx.x - s.sort_blocks);
    return;
  }
  const int padded = (s.T + 3) / 4 * 4;
  for (int i = threadIdx.x; i < padded; i += kCountThreads) ids[i] = i < s.T ? id_at(s, i) : 0x7fffffff;
  if (blockIdx.x == 0 && threadIdx.x == 0) *s.n_long = 0;
  __syncthreads();
  const int i = blockIdx.x * (kCountThreads / kCountPer) + threadIdx.x / kCountPer;
  const int id = i < s.T ? ids[i] : 0;
  int before = 0;
  for (int j = threadIdx.x % kCountPer; j < padded / 4; j += kCountPer) {
    const int4 o = ids4[j];
    const int p = 4 * j;
    before += (o.x < id || (o.x == id && p < i)) + (o.y < id || (o.y == id && p + 1 < i)) +
              (o.z < id || (o.z == id && p + 2 < i)) + (o.w < id || (o.w == id && p + 3 < i));
  }
#pragma unroll
  for (int o = 1; o < kCountPer; o <<= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
  if (i < s.T && threadIdx.x % kCountPer == 0) s.a[before] = make_int2(id, i);
}

// Every warp owns a contiguous part of its block's part of the pairs, which keeps each pass stable.
template <int BITS>
__global__ void __launch_bounds__(kSortThreads, 1) sort_ids_kernel(SortArgs s) {
  extern __shared__ int hist[];                                    // [warps][digits], then lane masks of the same shape
  __shared__ int total[kMaxDigits];                                // of this block, read by the others
  __shared__ int base[kMaxDigits];
  __shared__ int warp_sums[kSortWarps];
  cg::cluster_group cluster = cg::this_cluster();
  constexpr int blocks = kSortCluster;
  const int rank = static_cast<int>(cluster.block_rank());
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int digits = 1 << BITS;
  const int parts = blocks * kSortWarps;
  const int per = (s.T + parts - 1) / parts;
  const int lo = min(s.T, (rank * kSortWarps + warp) * per), hi = min(s.T, lo + per);
  int* mine = hist + warp * digits;
  unsigned* masks = reinterpret_cast<unsigned*>(hist + kSortWarps * digits) + warp * digits;
  for (int d = lane; d < digits; d += 32) masks[d] = 0;
  tx::griddep_launch_dependents();
  if (rank == 0 && tid == 0) *s.n_long = 0;
  for (int p = 0; p < s.passes; ++p) {
    // the last pass writes `a`
    int2* dst = ((s.passes - 1 - p) & 1) ? s.b : s.a;
    const int2* src = ((s.passes - 1 - p) & 1) ? s.a : s.b;
    const int shift = p * BITS;
    for (int d = lane; d < digits; d += 32) mine[d] = 0;
    __syncwarp();
    int2 pair[kSortTile];
    auto load_tile = [&](int i0) {
#pragma unroll
      for (int u = 0; u < kSortTile; ++u) {
        const int i = i0 + u * 32 + lane;
        pair[u] = i < hi ? sort_load(s, src, p, i) : make_int2(0, 0);
      }
    };
    for (int i0 = lo; i0 < hi; i0 += 32 * kSortTile) {
      load_tile(i0);
#pragma unroll
      for (int u = 0; u < kSortTile; ++u)
        if (i0 + u * 32 + lane < hi) atomicAdd(&mine[(pair[u].x >> shift) & (digits - 1)], 1);
    }
    __syncthreads();
    // counts before each warp, this block's totals
    constexpr int kPer = (digits + kSortThreads - 1) / kSortThreads;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const int d = tid + e * kSortThreads;
      if (d < digits) {
        int n[kSortWarps], sum = 0;
#pragma unroll
        for (int w = 0; w < kSortWarps; ++w) n[w] = hist[w * digits + d];
#pragma unroll
        for (int w = 0; w < kSortWarps; ++w) {
          hist[w * digits + d] = sum;
          sum += n[w];
        }
        total[d] = sum;
      }
    }
    cluster.sync();
    int before[kPer], all[kPer], mass = 0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const int d = tid * kPer + e;
      before[e] = all[e] = 0;
      if (d < digits) {
#pragma unroll
        for (int r = 0; r < blocks; ++r) {
          const int n = cluster.map_shared_rank(total, r)[d];
          if (r < rank) before[e] += n;
          all[e] += n;
        }
      }
      mass += all[e];
    }
    int scan = mass;                                               // inclusive over the threads
    for (int o = 1; o < 32; o <<= 1) {
      const int n = __shfl_up_sync(0xffffffffu, scan, o);
      if (lane >= o) scan += n;
    }
    if (lane == 31) warp_sums[warp] = scan;
    __syncthreads();
    int upto = scan - mass;
    for (int w = 0; w < warp; ++w) upto += warp_sums[w];
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      if (tid * kPer + e < digits) base[tid * kPer + e] = upto + before[e];
      upto += all[e];
    }
    __syncthreads();
    for (int i0 = lo; i0 < hi; i0 += 32 * kSortTile) {
      if (hi - lo > 32 * kSortTile) load_tile(i0);                 // else the tile is still in the registers
#pragma unroll
      for (int u = 0; u < kSortTile; ++u) {
        if (i0 + u * 32 >= hi) break;
        const bool in = i0 + u * 32 + lane < hi;
        // lanes with this lane's digit: every lane sets its bit in the digit's word (votes and matches take longer)
        const int d = (pair[u].x >> shift) & (digits - 1);
        if (in) atomicOr(&masks[d], 1u << lane);
        __syncwarp();
        const unsigned same = in ? masks[d] : 0, below = same & ((1u << lane) - 1);
        const int at = in ? base[d] + mine[d] + __popc(below) : 0;
        __syncwarp();
        if (in) {
          dst[at] = pair[u];
          if (below == 0) {
            mine[d] += __popc(same);
            masks[d] = 0;
          }
        }
        __syncwarp();
      }
    }
    cluster.sync();                                                // pairs written, totals read
  }
}

// Clears a new gradient on the SMs that the sort in front of it leaves free; its last block ends after the sort.
__global__ void __launch_bounds__(kClearThreads) clear_kernel(SortArgs s) {
  clear_tile(s, blockIdx.x);
  if (blockIdx.x == gridDim.x - 1) tx::griddep_wait();
}

struct GradArgs {
  const int2* pairs;          // [T] sorted
  const __nv_bfloat16* dout;  // [T, D]
  float* partial;             // [2 * chunks, D]: sum of a long run that came in, of one that begins and goes on
  int2* long_runs;            // [chunks]: chunk where it begins, chunk where it ends
  int* n_long;
  void* grad;                 // [V, D]
  int T, V, D, chunk;
  float scale;
  int vec;                    // grad is 16-byte aligned (a view into a flat buffer may not be)
};

// One row of the table is written by exactly one thread per column. The fp32 buffer is added to by a reduction without
// a return value: nothing waits for the old value, and with one addition per element the order cannot matter.
__device__ __forceinline__ void store_row(float* dst, const float (&v)[8], float scale, int vec) {
  if (!vec) {
#pragma unroll
    for (int e = 0; e < 8; ++e) dst[e] += v[e] * scale;
    return;
  }
#pragma unroll
  for (int h = 0; h < 8; h += 4)
    asm volatile("red.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(dst + h), "f"(v[h] * scale), "f"(v[h + 1] * scale),
                 "f"(v[h + 2] * scale), "f"(v[h + 3] * scale)
                 : "memory");
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
constexpr int kMinChunk = 4;
constexpr int kRows = 8;             // rows of dout a thread has in flight

// Block (chunk, column tile); a thread owns 8 columns. A run that crosses into the next chunk and ends there belongs to
// the chunk where it begins; one that covers a whole chunk or more is long.
template <typename GT>
__global__ void __launch_bounds__(256, 4) sum_runs_kernel(GradArgs g) {
  __shared__ int2 window[3 * kMaxChunk + 2];                       // the chunk before with one more, this one, the next with one more
  const int size = g.chunk, lo = blockIdx.x * size, n = min(size, g.T - lo);
  tx::griddep_wait();
  for (int i = threadIdx.x; i < 3 * size + 2; i += blockDim.x) {
    const int at = lo - size - 1 + i;
    window[i] = (at >= 0 && at < g.T) ? g.pairs[at] : make_int2(-1, 0);
  }
  __syncthreads();
  const int2* run = window + size + 1;                             // run[-size - 1 .. 2 size]
  int begin = 0, end = n;
  bool long_in = false, long_out = false;
  const int head = run[0].x, tail = run[n - 1].x;
  if (run[-1].x == head) {                                         // the first run came in
    int e = 1;
    while (e < n && run[e].x == head) ++e;
    const bool whole = e == n && run[n].x == head;                 // and goes on
    long_in = whole || run[-size - 1].x == head || (e == n && n == size);
    if (!long_in) begin = e;
  }
  if (n == size && run[n].x == tail && !(run[-1].x == tail && head == tail)) {       // the last run begins here and goes on
    int e = n + 1;
    while (e < 2 * size && run[e].x == tail) ++e;
    // it covers the next chunk
    long_out = e == 2 * size;
    if (!long_out) end = e;
  }
  const int col = (blockIdx.y * blockDim.x + threadIdx.x) * 8;
  if (long_out && blockIdx.y == 0 && threadIdx.x == 0 && tail < g.V) {
    int a = (lo / size) + 1, b = (g.T - 1) / size;                 // last chunk whose first position holds the id
    while (a < b) {
      const int mid = a + (b - a + 1) / 2;
      if (g.pairs[mid * size].x == tail) a = mid; else b = mid - 1;
    }
    g.long_runs[atomicAdd(g.n_long, 1)] = make_int2(blockIdx.x, a);
  }
  if (col >= g.D) return;
  float acc[8] = {};
  auto row = [&](int i) { return *reinterpret_cast<const uint4*>(g.dout + static_cast<long long>(run[i].y) * g.D + col); };
  auto add = [&](uint4 v) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      acc[2 * e] += __uint_as_float(w[e] << 16);
      acc[2 * e + 1] += __uint_as_float(w[e] & 0xffff0000u);
    }
  };
  for (int i0 = begin; i0 < end; i0 += kRows) {
    uint4 v[kRows];
    const int id0 = run[i0].x;
    if (id0 >= g.V) return;                                        // only ids outside the vocabulary follow
    if (i0 + kRows < end && run[i0 + kRows].x == id0) {            // in the middle of a run
#pragma unroll
      for (int u = 0; u < kRows; ++u) v[u] = row(i0 + u);
#pragma unroll
      for (int u = 0; u < kRows; ++u) add(v[u]);
      continue;
    }
#pragma unroll
    for (int u = 0; u < kRows; ++u)
      if (i0 + u < end) v[u] = row(i0 + u);
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
      const int i = i0 + u;
      if (i >= end) break;
      const int id = run[i].x;
      if (id >= g.V) return;
      add(v[u]);
      if (i + 1 < end && run[i + 1].x == id) continue;
      const bool in = long_in && id == head, on = long_out && id == tail;
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

constexpr int kJoinGroups = 32;      // chunks of a long run are summed in this many contiguous parts

// Work item: (long run, 64 columns); 8 threads across, kJoinGroups parts.
template <typename GT>
__global__ void __launch_bounds__(8 * kJoinGroups) join_runs_kernel(GradArgs g) {
  __shared__ float sh[kJoinGroups][8][8];
  tx::griddep_wait();
  const int tiles = (g.D + 63) / 64, items = *g.n_long * tiles;
  const int tx = threadIdx.x & 7, part = threadIdx.x >> 3;
  for (int item = blockIdx.x; item < items; item += gridDim.x) {
    const int2 run = g.long_runs[item / tiles];
    const int count = run.y - run.x + 1, col = (item % tiles) * 64 + tx * 8;
    const int per = (count + kJoinGroups - 1) / kJoinGroups;
    const int id = g.pairs[run.y * g.chunk].x;
    float acc[8] = {};
    if (col < g.D) {
#pragma unroll 4
      for (int i = part * per; i < min(count, (part + 1) * per); ++i) {
        const float4* p = reinterpret_cast<const float4*>(g.partial + (2ll * (run.x + i) + (i == 0 ? 1 : 0)) * g.D + col);
        const float4 x = p[0], y = p[1];
        acc[0] += x.x; acc[1] += x.y; acc[2] += x.z; acc[3] += x.w;
        acc[4] += y.x; acc[5] += y.y; acc[6] += y.z; acc[7] += y.w;
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) sh[part][tx][e] = acc[e];
    __syncthreads();
    if (part == 0 && col < g.D) {
      for (int q = 1; q < kJoinGroups; ++q)
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] += sh[q][tx][e];
      store_row(static_cast<GT*>(g.grad) + static_cast<long long>(id) * g.D + col, acc, g.scale, g.vec);
    }
    __syncthreads();
  }
}

int chunk_of(int T) {
  // a few chunks per SM while there are few tokens, at most kMaxChunk positions
  const int c = (T + 4 * txh::sm_count() - 1) / (4 * txh::sm_count());
  return c < kMinChunk ? kMinChunk : (c > kMaxChunk ? kMaxChunk : c);
}

template <typename GT>
int launch_grad(const GradArgs& g, cudaStream_t s) {
  const int chunks = (g.T + g.chunk - 1) / g.chunk;
  const int threads = min(256, (g.D / 8 + 31) / 32 * 32);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(chunks, (g.D / 8 + threads - 1) / threads);
  cfg.blockDim = dim3(threads);
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, sum_runs_kernel<GT>, g) != cudaSuccess) return 405;
  if (chunks < 2) return cudaGetLastError() == cudaSuccess ? 0 : 400;        // a long run covers a chunk behind its first
  const long long most = static_cast<long long>(chunks) * ((g.D + 63) / 64);
  const int grid = static_cast<int>(min(most, 4ll * txh::sm_count()));
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(8 * kJoinGroups);
  return cudaLaunchKernelEx(&cfg, join_runs_kernel<GT>, g) == cudaSuccess ? 0 : 406;
}

template <int BITS>
int launch_sort(SortArgs so, cudaStream_t s) {
  const int bytes = 2 * kSortWarps * (1 << BITS) * 4;
  static txh::DeviceFlag flag;                                     // one per width
  if (!flag.cur()) {
    if (cudaFuncSetAttribute(sort_ids_kernel<BITS>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
      return 401;
    flag.cur() = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(kSortCluster);
  cfg.blockDim = dim3(kSortThreads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = kSortCluster;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, sort_ids_kernel<BITS>, so) != cudaSuccess) return 402;
  if (so.n_zero == 0) return 0;
  cfg.gridDim = dim3(static_cast<unsigned>((so.n_zero + kClearTile - 1) / kClearTile));
  cfg.blockDim = dim3(kClearThreads);
  cfg.dynamicSmemBytes = 0;
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  return cudaLaunchKernelEx(&cfg, clear_kernel, so) == cudaSuccess ? 0 : 404;
}

}  // namespace

// Bytes of workspace for T tokens of D columns (16-byte aligned): two lists of pairs, the list of long runs and its
// length, the partial sums.
extern "C" long long tx_embedding_grad_workspace(int T, int D) {
  const long long chunks = (T + chunk_of(T) - 1) / chunk_of(T);
  return 2 * ((8ll * T + 15) / 16 * 16) + (8 * chunks + 15) / 16 * 16 + 16 + 2 * chunks * D * 4;
}

// ids int64 or int32 [T], T at most kMaxTokens, dout bf16 [T, D] with D a multiple of 8. grad_bf16 == 0: grad is fp32
// and added to; else it is bf16 and written whole.
extern "C" int tx_embedding_grad(const void* ids, int ids64, const void* dout, void* grad, int grad_bf16, int T, int D,
                                 int V, float scale, void* workspace, cudaStream_t s) {
  if (D % 8 || D <= 0 || V <= 0 || V > 0x3fffffff || T > kMaxTokens) return 1;
  if (T <= 0) return grad_bf16 && cudaMemsetAsync(grad, 0, 2ll * V * D, s) != cudaSuccess ? 403 : 0;
  const long long chunks = (T + chunk_of(T) - 1) / chunk_of(T);
  int2* a = static_cast<int2*>(workspace);
  int2* b = a + (T + 1ll) / 2 * 2;
  int2* long_runs = b + (T + 1ll) / 2 * 2;
  int* n_long = reinterpret_cast<int*>(long_runs + (chunks + 1) / 2 * 2);
  SortArgs so{ids, ids64, T, V, 1, a, b, n_long, nullptr, 0, 0};
  if (grad_bf16) {
    if (reinterpret_cast<uintptr_t>(grad) % 16 == 0) {
      so.zero = static_cast<uint4*>(grad);
      so.n_zero = static_cast<long long>(V) * D / 8;
    } else if (cudaMemsetAsync(grad, 0, 2ll * V * D, s) != cudaSuccess) {
      return 403;
    }
  }
  const GradArgs g{a, static_cast<const __nv_bfloat16*>(dout), reinterpret_cast<float*>(n_long + 4), long_runs, n_long,
                   grad, T, V, D, chunk_of(T), scale, reinterpret_cast<uintptr_t>(grad) % 16 == 0};
  if (T <= kCountTokens) {
    const int per = kCountThreads / kCountPer;
    so.sort_blocks = (T + per - 1) / per;
    const unsigned clear = static_cast<unsigned>((so.n_zero + kClearTile - 1) / kClearTile);
    count_sort_kernel<<<so.sort_blocks + clear, kCountThreads, 0, s>>>(so);
    return grad_bf16 ? launch_grad<__nv_bfloat16>(g, s) : launch_grad<float>(g, s);
  }
  int bits = 1;
  while ((V >> bits) != 0) ++bits;                                 // V itself marks ids outside
  so.passes = (bits + 9) / 10;
  const int width = (bits + so.passes - 1) / so.passes;
  const int rc = width > 9 ? launch_sort<10>(so, s) : (width > 8 ? launch_sort<9>(so, s) : launch_sort<8>(so, s));
  if (rc) return rc;
  return grad_bf16 ? launch_grad<__nv_bfloat16>(g, s) : launch_grad<float>(g, s);
}
