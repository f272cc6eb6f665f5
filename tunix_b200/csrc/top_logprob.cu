// Operators on rows of logits that report or learn from the k best entries of a row.
//
//  * tx_top_logprob_fwd: log-probability of one given token, the k largest logits (ids and log-probabilities, equal
//    values by the lowest id) and the entropy of softmax(x * inv_temp), in one pass over the row.
//  * tx_top_distill_fwd: per row the divergence from a teacher's list of (id, value) pairs and the cross entropy of
//    a label, in one pass over the student's row (none at all when only the listed entries matter).
//  * tx_top_bwd: the gradient of either with respect to the row, one read and one write.
//
// With m = max x, d_j = x_j - m and c = inv_temp * log2(e):  s = sum 2^(d_j c),  log p_j = d_j inv_temp - ln s.
// Everything is kept relative to m, so log-probabilities do not lose the bits of a large log-sum-exp, and the
// running maximum starts at the lowest finite float: a row of -inf sums to 0 instead of to NaN (it is reported as
// an empty row: ln s is stored as +inf, log-probabilities are -inf, losses and gradients 0).
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <stdint.h>

#include "tx_host.h"

namespace cg = cooperative_groups;

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kVec = 8;                       // elements a thread takes at a time
constexpr int kChunk = kThreads * kVec;       // elements the block takes per iteration
constexpr int kMaxTop = 256;                  // longest list of alternatives
constexpr int kMaxList = 1024;                // longest teacher's list
constexpr int kSlots = 4096;                  // candidate slots of a block
constexpr int kPicked = 1024;                 // of which this many may be left for the last sort
constexpr int kBins = 256;
constexpr int kMaxSplit = 8;                  // blocks (one cluster) a row is spread over when there are few rows
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Maximum that keeps a NaN.
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void from_f(float v, float* p) { *p = v; }
__device__ __forceinline__ void from_f(float v, __nv_bfloat16* p) { *p = __float2bfloat16_rn(v); }

// Eight consecutive elements from a 16-byte aligned address.
__device__ __forceinline__ void vec_load(const float* p, float (&z)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  z[0] = a.x; z[1] = a.y; z[2] = a.z; z[3] = a.w; z[4] = b.x; z[5] = b.y; z[6] = b.z; z[7] = b.w;
}
__device__ __forceinline__ void vec_load(const __nv_bfloat16* p, float (&z)[8]) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    z[2 * i] = __uint_as_float(w[i] << 16);
    z[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void vec_store(float* p, const float (&z)[8]) {
  *reinterpret_cast<float4*>(p) = make_float4(z[0], z[1], z[2], z[3]);
  *reinterpret_cast<float4*>(p + 4) = make_float4(z[4], z[5], z[6], z[7]);
}
__device__ __forceinline__ void vec_store(__nv_bfloat16* p, const float (&z)[8]) {
  uint4 u;
  __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(z[2 * i], z[2 * i + 1]);
  *reinterpret_cast<uint4*>(p) = u;
}

// How many elements an address lies behind the last 16-byte boundary.
template <typename T>
__device__ __forceinline__ int misalign(const T* p) {
  return static_cast<int>((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T));
}

// Elements j .. j+7 of a row; those outside [lo, hi) are -inf. `aligned`: the address of j is.
template <typename T>
__device__ __forceinline__ void load8(const T* row, int j, int lo, int hi, bool aligned, float (&z)[8]) {
  if (aligned && j >= lo && j + kVec <= hi) {
    vec_load(row + j, z);
  } else {
#pragma unroll
    for (int i = 0; i < kVec; ++i) z[i] = (j + i >= lo && j + i < hi) ? to_f(row[j + i]) : -INFINITY;
  }
}

__device__ __forceinline__ float max8(const float (&z)[8]) {
  return max_nan(max_nan(max_nan(z[0], z[1]), max_nan(z[2], z[3])), max_nan(max_nan(z[4], z[5]), max_nan(z[6], z[7])));
}

// Columns of a row that block `rank` of `blocks` takes: equal parts, cut at multiples of kVec from the first one.
__device__ __forceinline__ int2 part_of(int V, int rank, int blocks) {
  const int vecs = (V + kVec - 1) / kVec;
  const int per = (vecs + blocks - 1) / blocks * kVec;
  return make_int2(min(V, rank * per), min(V, rank * per + per));
}

// ---- softmax statistics --------------------------------------------------------------------------------
struct Stat {
  float m;    // running maximum, never below the lowest finite float
  float s;    // sum 2^(d c)
  float sd;   // sum 2^(d c) d, for the entropy; or the sum at a second temperature
};

constexpr int kNone = 0, kEntropy = 1, kSecond = 2;

__device__ __forceinline__ Stat stat_init() { return Stat{-FLT_MAX, 0.f, 0.f}; }

template <int X>
__device__ __forceinline__ void stat_rescale(Stat& a, float m, float c, float c2) {
  const float d = a.m - m;
  const float e = ex2(d * c);
  if (X == kEntropy) a.sd = e == 0.f ? 0.f : e * (a.sd + a.s * d);
  if (X == kSecond) a.sd *= ex2(d * c2);
  a.s *= e;
  a.m = m;
}

template <int X>
__device__ __forceinline__ void stat_push8(Stat& a, const float (&z)[8], float vm, float c, float c2) {
  if (vm > a.m) stat_rescale<X>(a, vm, c, c2);
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    const float d = z[i] - a.m;
    const float w = ex2(d * c);
    a.s += w;
    if (X == kEntropy) a.sd = fmaf(w, fmaxf(d, -FLT_MAX), a.sd);     // 0 * -inf would be NaN
    if (X == kSecond) a.sd += ex2(d * c2);
  }
}

template <int X>
__device__ __forceinline__ void stat_merge(Stat& a, Stat b, float c, float c2) {
  const float m = fmaxf(a.m, b.m);
  stat_rescale<X>(a, m, c, c2);
  stat_rescale<X>(b, m, c, c2);
  a.s += b.s;
  a.sd += b.sd;
}

// Leaves the block's statistics in every thread. `sh` holds kWarps entries.
template <int X>
__device__ __forceinline__ Stat stat_block(Stat a, Stat* sh, float c, float c2) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Stat b;
    b.m = __shfl_xor_sync(0xffffffffu, a.m, o);
    b.s = __shfl_xor_sync(0xffffffffu, a.s, o);
    b.sd = __shfl_xor_sync(0xffffffffu, a.sd, o);
    stat_merge<X>(a, b, c, c2);
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = a;
  __syncthreads();
  a = sh[0];
  for (int w = 1; w < kWarps; ++w) stat_merge<X>(a, sh[w], c, c2);
  return a;
}

// ln s, or +inf for a row without a finite logit.
__device__ __forceinline__ float log_sum(float s) { return s == 0.f ? INFINITY : logf(s); }

// ---- keys of candidates --------------------------------------------------------------------------------
// 64 bits that order by value from high to low (NaN highest, -0 equal to 0), equal values by the lowest index.
__device__ __forceinline__ unsigned long long key_of(float x, int idx) {
  const uint32_t b = __float_as_uint(x + 0.f);
  const uint32_t o = x != x ? 0xffffffffu : ((b & 0x80000000u) ? ~b : (b | 0x80000000u));
  return (static_cast<unsigned long long>(o) << 32) | (0xffffffffu - static_cast<uint32_t>(idx));
}
__device__ __forceinline__ float key_value(unsigned long long key) {
  const uint32_t o = static_cast<uint32_t>(key >> 32);
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);      // NaN's key gives a NaN back
}
__device__ __forceinline__ int key_index(unsigned long long key) {
  return static_cast<int>(0xffffffffu - static_cast<uint32_t>(key));
}

__device__ __forceinline__ unsigned long long shfl_key(unsigned long long k, int stride) {
  const uint32_t lo = __shfl_xor_sync(0xffffffffu, static_cast<uint32_t>(k), stride);
  const uint32_t hi = __shfl_xor_sync(0xffffffffu, static_cast<uint32_t>(k >> 32), stride);
  return (static_cast<unsigned long long>(hi) << 32) | lo;
}

// Sorts n keys in shared memory from high to low (bitonic; slots n .. P-1 are filled with 0, P the next power of 2).
// All threads call it. Up to one key per thread stays in a register and strides below a warp are shuffles.
__device__ __forceinline__ void sort_keys(unsigned long long* keys, int n) {
  int P = 32;
  while (P < n) P <<= 1;
  const int tid = threadIdx.x;
  if (P <= kThreads) {
    const bool in = (tid & ~31) < P;
    unsigned long long key = tid < n ? keys[tid] : 0;
    for (int size = 2; size <= P; size <<= 1) {
      for (int stride = size >> 1; stride > 0; stride >>= 1) {
        unsigned long long other = 0;
        if (stride >= 32) {
          __syncthreads();
          if (in) keys[tid] = key;
          __syncthreads();
          if (in) other = keys[tid ^ stride];
        } else if (in) {
          other = shfl_key(key, stride);
        }
        const bool larger = ((tid & stride) == 0) == ((tid & size) == 0);
        if (larger == (other > key)) key = other;
      }
    }
    __syncthreads();
    if (in) keys[tid] = key;
    __syncthreads();
    return;
  }
  for (int i = n + tid; i < P; i += kThreads) keys[i] = 0;
  __syncthreads();
  for (int size = 2; size <= P; size <<= 1) {
    for (int stride = size >> 1; stride > 0; stride >>= 1) {
      for (int i = tid; i < P / 2; i += kThreads) {
        const int a = 2 * i - (i & (stride - 1));
        const int b = a + stride;
        const unsigned long long x = keys[a], y = keys[b];
        if ((x < y) == ((a & size) == 0)) {
          keys[a] = y;
          keys[b] = x;
        }
      }
      __syncthreads();
    }
  }
}

// ---- forward: given token, k best, entropy --------------------------------------------------------------
struct TopArgs {
  const void* logits;
  long long ld;
  int T, V, k;
  float inv_temp;
  const long long* targets;    // [T] or null
  long long* ids;              // [T, k]
  float* top;                  // [T, k]
  float* target;               // [T] or null
  float* entropy;              // [T] or null
  float2* stats;               // [T]: m, ln s
};

// Selection state of a block.
//
// A candidate is an element that is not below a threshold which k elements of the block's part are known to reach.
// The first threshold comes from the first iteration: the smallest over the warps of the ceil(k / warps)-th largest of
// a warp's per-thread maxima (of the warps that have 256 elements). From then on candidates are counted in bins of equal width above it, and every 64
// candidates the threshold moves up to half a bin below the lowest bin that k of them reach. Bin numbers and that
// edge are computed with monotone roundings, so an element of such a bin is never below the edge.
struct Select {
  unsigned long long keys[kSlots];
  unsigned long long picked[kPicked];
  int bins[kBins];
  int count, n_picked;
  float thr0, width, thr;
  float warp_nth[kWarps], warp_max[kWarps];
  Stat stat[kWarps];
  Stat part;                   // this block's statistics, read by the cluster's first block
};

__device__ __forceinline__ int bin_of(float x, float thr0, float inv_width) {
  return static_cast<int>(fminf((x - thr0) * inv_width, static_cast<float>(kBins - 1)));     // NaN: the last one
}

// Lowest bin that k counted candidates reach or pass (0 while there are fewer), by one warp.
__device__ __forceinline__ int cut_bin(const volatile int* bins, int k) {
  const int lane = threadIdx.x & 31;
  const int top = kBins - 1 - lane * (kBins / 32);           // lane 0 has the highest bins
  int n[kBins / 32], sum = 0;
#pragma unroll
  for (int i = 0; i < kBins / 32; ++i) {
    n[i] = bins[top - i];
    sum += n[i];
  }
  int upto = sum;
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += v;
  }
  const unsigned reach = __ballot_sync(0xffffffffu, upto >= k);
  if (reach == 0) return 0;
  const int who = __ffs(reach) - 1;
  int b = top, seen = upto - sum;
#pragma unroll
  for (int i = 0; i < kBins / 32; ++i) {
    seen += n[i];
    if (seen < k) b = top - i - 1;
  }
  return __shfl_sync(0xffffffffu, b, who);
}

// The k best of columns [lo, hi) into keys[0 .. k), sorted, for rows whose candidates do not fit: elements come in
// order of their index, one per thread and iteration, so from the first full set on only larger ones than the k-th
// can enter.
template <typename LT>
__device__ void select_in_order(Select& s, const LT* x, int lo, int hi, int k) {
  const int limit = kSlots - kThreads;
  float thr = -INFINITY;
  bool any = true;                                   // no threshold yet
  __syncthreads();
  if (threadIdx.x == 0) s.count = 0;
  __syncthreads();
  for (int base = lo; base < hi; base += kThreads) {
    const int j = base + threadIdx.x;
    int over = 0;
    if (j < hi) {
      const float v = to_f(x[j]);
      if (any || !(v <= thr)) {
        const int pos = atomicAdd(&s.count, 1);
        s.keys[pos] = key_of(v, j);                  // below the limit before this iteration
        over = pos >= limit - 1;
      }
    }
    // the first set is cut at once: it holds every element so far
    if (__syncthreads_or(over || (any && base + kThreads - lo >= k))) {
      sort_keys(s.keys, s.count);
      any = s.count < k;
      if (!any) thr = key_value(s.keys[k - 1]);
      __syncthreads();
      if (threadIdx.x == 0) s.count = min(s.count, k);
      __syncthreads();
    }
  }
  sort_keys(s.keys, s.count);
}

template <typename LT, int X>
__global__ void __launch_bounds__(kThreads, 2) top_fwd_kernel(TopArgs a) {
  extern __shared__ unsigned char shared[];
  Select& s = *reinterpret_cast<Select*>(shared);
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int row = blockIdx.x / blocks, tid = threadIdx.x, lane = tid & 31;
  const LT* x = static_cast<const LT*>(a.logits) + static_cast<long long>(row) * a.ld;
  const float c = a.inv_temp * kLog2e;
  const int k = a.k;
  const int2 part = part_of(a.V, rank, blocks);
  const int lo = part.x, hi = part.y;
  for (int i = tid; i < kBins; i += kThreads) s.bins[i] = 0;
  if (tid == 0) {
    s.count = 0;
    s.n_picked = 0;
  }
  Stat st = stat_init();
  // ---- first iteration: the first threshold
  const int base = lo - misalign(x + lo);
  float z[8];
  const int j0 = base + tid * kVec;
  load8(x, j0, lo, hi, true, z);
  const float v0 = max8(z);
  stat_push8<X>(st, z, v0, c, 0.f);
  float v = v0 != v0 ? INFINITY : v0;
  for (int size = 2; size <= 32; size <<= 1)
    for (int stride = size >> 1; stride > 0; stride >>= 1) {
      const float o = __shfl_xor_sync(0xffffffffu, v, stride);
      const bool larger = ((lane & stride) == 0) == ((lane & size) == 0);
      v = larger ? fmaxf(v, o) : fminf(v, o);
    }
  // only warps whose 256 elements all lie in the part count; too few of them give no threshold
  const int whole = min(kWarps, max(0, hi - base) / (32 * kVec));
  const int nth_of = whole ? (k + whole - 1) / whole : 33;
  const float nth = __shfl_sync(0xffffffffu, v, min(nth_of, 32) - 1);
  if (lane == 0) {
    s.warp_nth[tid >> 5] = nth;
    s.warp_max[tid >> 5] = v;
  }
  __syncthreads();
  float thr0 = INFINITY, most = s.warp_max[0];
  for (int w = 0; w < kWarps; ++w) {
    if (w < whole) thr0 = fminf(thr0, s.warp_nth[w]);
    most = fmaxf(most, s.warp_max[w]);
  }
  if (nth_of > 32) thr0 = -INFINITY;
  // 64 bins up to the first iteration's maximum; any positive width is correct
  float width = (most - thr0) * (1.f / 64.f);
  if (!(width > 1e-30f && width < 1e30f)) width = 1.f;
  const float inv_width = 1.f / width;
  if (tid == 0) s.thr = thr0;
  float thr = thr0;
  __syncthreads();
  auto offer = [&](const float (&e)[8], int j, float vm) {
    bool full = false;
    if (!(vm < thr)) {
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        if (!(e[i] < thr) && j + i >= lo && j + i < hi) {
          const int pos = atomicAdd(&s.count, 1);
          if (pos < kSlots) s.keys[pos] = key_of(e[i], j + i);
          atomicAdd(&s.bins[bin_of(e[i], thr0, inv_width)], 1);
          full |= (pos & 63) == 63;
        }
      }
    }
    if (__any_sync(0xffffffffu, full)) {
      const int b = cut_bin(s.bins, k);
      const float t = fmaf(b - 0.5f, width, thr0);
      if (lane == 0 && b > 0 && t > *const_cast<volatile float*>(&s.thr)) *const_cast<volatile float*>(&s.thr) = t;
      __syncwarp();
    }
  };
  offer(z, j0, v0);
  for (int at = base + kChunk; at < hi; at += 2 * kChunk) {
    const int j = at + tid * kVec;
    float y[8];
    load8(x, j, lo, hi, true, z);
    load8(x, j + kChunk, lo, hi, true, y);
    const float vz = max8(z), vy = max8(y);
    stat_push8<X>(st, z, vz, c, 0.f);
    stat_push8<X>(st, y, vy, c, 0.f);
    thr = *const_cast<volatile float*>(&s.thr);
    offer(z, j, vz);
    offer(y, j + kChunk, vy);
  }
  __syncthreads();
  // ---- the block's k best, sorted
  const int n = s.count;
  const int want = min(k, hi - lo);
  const unsigned long long* best = s.keys;
  if (n > kSlots) {
    select_in_order(s, x, lo, hi, k);
  } else if (n <= 128) {
    sort_keys(s.keys, n);
  } else {
    const int b = cut_bin(s.bins, k);
    for (int i = tid; i < n; i += kThreads) {
      const unsigned long long key = s.keys[i];
      if (bin_of(key_value(key), thr0, inv_width) >= b) {
        const int pos = atomicAdd(&s.n_picked, 1);
        if (pos < kPicked) s.picked[pos] = key;
      }
    }
    __syncthreads();
    if (s.n_picked <= kPicked) {
      best = s.picked;
      sort_keys(s.picked, s.n_picked);
    } else {
      sort_keys(s.keys, n);
    }
  }
  st = stat_block<X>(st, s.stat, c, 0.f);
  // ---- over the cluster: the first block collects lists and statistics
  if (blocks > 1) {
    if (best != s.picked) {
      for (int i = tid; i < want; i += kThreads) s.picked[i] = best[i];
    }
    if (tid == 0) {
      s.part = st;
      s.n_picked = want;
    }
    cluster.sync();
    if (rank == 0) {
      int at = 0;
      for (int r = 0; r < blocks; ++r) {
        const Select* o = cluster.map_shared_rank(&s, r);
        const int m = o->n_picked;
        for (int i = tid; i < m; i += kThreads) s.keys[at + i] = o->picked[i];
        at += m;
        if (r > 0) stat_merge<X>(st, o->part, c, 0.f);
      }
      __syncthreads();
      sort_keys(s.keys, at);
      best = s.keys;
    }
    cluster.sync();                      // the others' shared memory was read
    if (rank != 0) return;
  }
  const float ls = log_sum(st.s);
  for (int i = tid; i < k; i += kThreads) {
    const unsigned long long key = best[i];
    a.ids[static_cast<long long>(row) * k + i] = key_index(key);
    a.top[static_cast<long long>(row) * k + i] = (key_value(key) - st.m) * a.inv_temp - ls;
  }
  if (tid == 0) {
    if (a.target) {
      const long long t = a.targets[row];
      a.target[row] = (t >= 0 && t < a.V) ? (to_f(x[t]) - st.m) * a.inv_temp - ls : 0.f;
    }
    if (a.entropy) a.entropy[row] = st.s == 0.f ? 0.f : ls - a.inv_temp * (st.sd / st.s);
    a.stats[row] = make_float2(st.m, ls);
  }
}

// ---- forward: divergence from a teacher's list, cross entropy of a label ---------------------------------
struct DistillArgs {
  const void* logits;
  long long ld;
  int T, V, k;
  float inv_temp;
  int full;                    // 0: both sides normalised over the list, 1: over the vocabulary
  const long long* ids;        // [T, k]; an id outside the vocabulary is an absent entry
  const float* values;         // [T, k]
  const long long* labels;     // [T] or null; a label outside the vocabulary is ignored
  float* kl;                   // [T]
  float* nll;                  // [T] or null
  float4* stats;               // [T]: m, ln s at temperature 1, ln s at the temperature, unused
};

struct List {                  // statistics of the list, the same in every lane
  float mt, st, mx, sx;        // teacher: max, sum; student: max, sum (relative to the max)
};

__device__ __forceinline__ float warp_max(float v) {
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Statistics of a row's list normalised over the list itself, by one warp.
template <typename LT>
__device__ __forceinline__ List list_stats(const LT* x, const long long* ids, const float* values, int V, int k,
                                           float c) {
  List l{-FLT_MAX, 0.f, -FLT_MAX, 0.f};
  const int lane = threadIdx.x & 31;
  for (int i = lane; i < k; i += 32) {
    const long long id = ids[i];
    if (id < 0 || id >= V) continue;
    l.mt = fmaxf(l.mt, values[i]);
    l.mx = fmaxf(l.mx, to_f(x[id]));
  }
  l.mt = warp_max(l.mt);
  l.mx = warp_max(l.mx);
  for (int i = lane; i < k; i += 32) {
    const long long id = ids[i];
    if (id < 0 || id >= V) continue;
    l.st += ex2((values[i] - l.mt) * c);
    l.sx += ex2((to_f(x[id]) - l.mx) * c);
  }
  l.st = warp_sum(l.st);
  l.sx = warp_sum(l.sx);
  return l;
}

// PASSES: how many softmax sums of the row are needed. 0 (only the listed entries matter: one warp per row), 1 (scale
// c1 in the exponent) or 2 (c1 and c2).
template <typename LT, int PASSES>
__global__ void __launch_bounds__(PASSES ? kThreads : 32) distill_fwd_kernel(DistillArgs a, float c1, float c2) {
  __shared__ Stat sh_stat[kWarps];
  __shared__ Stat sh_part;
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = PASSES ? static_cast<int>(cluster.num_blocks()) : 1;
  const int rank = PASSES ? static_cast<int>(cluster.block_rank()) : 0;
  const int row = blockIdx.x / blocks, tid = threadIdx.x;
  const LT* x = static_cast<const LT*>(a.logits) + static_cast<long long>(row) * a.ld;
  const int V = a.V, k = a.k;
  Stat st = stat_init();
  constexpr int X = PASSES == 2 ? kSecond : kNone;
  if (PASSES > 0) {
    const int2 part = part_of(V, rank, blocks);
    const int lo = part.x, hi = part.y;
    for (int j = lo - misalign(x + lo) + tid * kVec; j < hi; j += 2 * kChunk) {
      float z[8], y[8];
      load8(x, j, lo, hi, true, z);
      load8(x, j + kChunk, lo, hi, true, y);
      stat_push8<X>(st, z, max8(z), c1, c2);
      stat_push8<X>(st, y, max8(y), c1, c2);
    }
    st = stat_block<X>(st, sh_stat, c1, c2);
    if (blocks > 1) {
      if (tid == 0) sh_part = st;
      cluster.sync();
      if (rank == 0)
        for (int r = 1; r < blocks; ++r) stat_merge<X>(st, *cluster.map_shared_rank(&sh_part, r), c1, c2);
      cluster.sync();
      if (rank != 0) return;
    }
  }
  if (tid >= 32) return;
  // With one pass both sums are the same number and only the one that is asked for gets used.
  const float ls1 = log_sum(st.s);
  const float ls2 = PASSES == 2 ? log_sum(st.sd) : ls1;
  const long long* ids = a.ids + static_cast<long long>(row) * k;
  const float* values = a.values + static_cast<long long>(row) * k;
  float kl = 0.f;
  if (a.full) {
    for (int i = tid; i < k; i += 32) {
      const long long id = ids[i];
      if (id < 0 || id >= V) continue;
      const float t = values[i], q = expf(t);
      if (q == 0.f) continue;
      kl += q * (t - ((to_f(x[id]) - st.m) * a.inv_temp - ls2));
    }
    kl = warp_sum(kl);
    if (ls2 == INFINITY) kl = 0.f;
  } else {
    const float c = a.inv_temp * kLog2e;
    const List l = list_stats(x, ids, values, V, k, c);
    const float lt = logf(l.st), lx = logf(l.sx);
    for (int i = tid; i < k; i += 32) {
      const long long id = ids[i];
      if (id < 0 || id >= V) continue;
      const float lq = (values[i] - l.mt) * a.inv_temp - lt;
      const float q = expf(lq);
      if (q == 0.f) continue;
      kl += q * (lq - ((to_f(x[id]) - l.mx) * a.inv_temp - lx));
    }
    kl = warp_sum(kl);
    if (l.st == 0.f || l.sx == 0.f) kl = 0.f;
  }
  if (tid == 0) {
    a.kl[row] = kl;
    if (a.nll) {
      const long long t = a.labels[row];
      a.nll[row] = (t >= 0 && t < V && ls1 != INFINITY) ? ls1 - (to_f(x[t]) - st.m) : 0.f;
    }
    a.stats[row] = make_float4(st.m, ls1, ls2, 0.f);
  }
}

// ---- backward -------------------------------------------------------------------------------------------
constexpr int kScore = 0, kListed = 1, kFull = 2;

struct BwdArgs {
  const void* logits;
  long long ld;
  int T, V, k, mode;
  float inv_temp;
  const long long* ids;        // [T, k]
  const float* values;         // [T, k] teacher's values (distillation) or gradients of the list (score); may be null
  const long long* given;      // [T] label or target, or null
  const float* g_list;         // [T] gradient of the divergence; unused by score
  const float* g_given;        // [T] gradient of nll / of the target's log-probability, or null
  const float* g_entropy;      // [T] or null
  const float* entropy;        // [T] when g_entropy
  const float* m;              // row statistics: m, ln s at temperature 1, ln s at the temperature, `stat_stride` floats
  int stat_stride, stat_one, stat_temp;
  void* dx;
  long long ldd;
  int blocks;                  // a row's columns are cut into this many parts
};

// d_j = A p_j (temperature) + B p_j (temperature 1) - G p_j (log p_j + H), then the listed columns get their own
// terms on top: they are computed from the same fp32 value and rounded once, by the thread of the first occurrence.
template <typename LT, int DENSE>   // bit 0: temperature, bit 1: temperature 1, bit 2: entropy
__global__ void __launch_bounds__(kThreads) top_bwd_kernel(BwdArgs a) {
  __shared__ int sh_id[kMaxList + 1];
  __shared__ float sh_coef[kMaxList + 1];
  __shared__ float sh_dense[2];
  const int row = blockIdx.x / a.blocks, tid = threadIdx.x;
  const int2 part = part_of(a.V, blockIdx.x - row * a.blocks, a.blocks);
  const int lo = part.x, hi = part.y;
  const LT* x = static_cast<const LT*>(a.logits) + static_cast<long long>(row) * a.ld;
  LT* dx = static_cast<LT*>(a.dx) + static_cast<long long>(row) * a.ldd;
  const int V = a.V, k = a.k;
  const float* st = a.m + static_cast<long long>(row) * a.stat_stride;
  const float m = st[0], ls1 = st[a.stat_one], lst = st[a.stat_temp];
  const float c = a.inv_temp * kLog2e;
  if (tid < 32) {
    const long long* ids = a.ids + static_cast<long long>(row) * k;
    const float* values = a.values ? a.values + static_cast<long long>(row) * k : nullptr;
    const float g = a.g_list ? a.g_list[row] : 0.f;
    float sum = 0.f;                      // of what multiplies p at the temperature
    List l{};
    float lt = 0.f, lx = 0.f;
    bool live = true;
    if (a.mode == kListed) {
      l = list_stats(x, ids, values, V, k, c);
      lt = logf(l.st);
      lx = logf(l.sx);
      live = l.st != 0.f && l.sx != 0.f;
    } else {
      live = lst != INFINITY;
    }
    live = live && (a.mode == kScore ? values != nullptr : a.g_list != nullptr);
    for (int i = tid; i < k; i += 32) {
      const long long id = ids[i];
      int at = -1;
      float coef = 0.f;
      if (live && id >= 0 && id < V) {
        at = static_cast<int>(id);
        if (a.mode == kScore) {
          coef = values[i];
          sum -= coef;
        } else if (a.mode == kFull) {
          const float q = expf(values[i]);
          coef = -g * q;
          sum -= coef;
        } else {
          const float q = expf((values[i] - l.mt) * a.inv_temp - lt);
          const float p = expf((to_f(x[id]) - l.mx) * a.inv_temp - lx);
          coef = g * (p - q);
        }
      }
      sh_id[i] = at;
      sh_coef[i] = coef * a.inv_temp;
    }
    sum = warp_sum(sum);
    if (tid == 0) {
      int at = -1;
      float coef = 0.f;
      if (a.g_given) {
        const long long t = a.given[row];
        if (t >= 0 && t < V && (a.mode == kScore ? lst : ls1) != INFINITY) {
          at = static_cast<int>(t);
          coef = a.g_given[row];
        }
      }
      sh_id[k] = at;
      sh_coef[k] = a.mode == kScore ? coef * a.inv_temp : -coef;
      if (a.mode == kScore) sum -= coef;
      sh_dense[0] = sum * a.inv_temp;
      sh_dense[1] = a.mode == kScore ? 0.f : coef;
    }
  }
  __syncthreads();
  const float A = sh_dense[0], B = sh_dense[1];
  const float lst2 = lst * kLog2e, ls12 = ls1 * kLog2e;
  float G = 0.f, H = 0.f;
  if (DENSE & 4) {
    G = a.g_entropy[row] * a.inv_temp;
    H = a.entropy[row];
  }
  auto dense = [&](float v) -> float {
    const float d = v - m;
    float r = 0.f;
    if (DENSE & 5) {
      const float p = ex2(fmaf(d, c, -lst2));
      r = A * p;
      if (DENSE & 4) r -= p == 0.f ? 0.f : G * p * (d * a.inv_temp - lst + H);
    }
    if (DENSE & 2) r = fmaf(B, ex2(fmaf(d, kLog2e, -ls12)), r);
    return r;
  };
  const int shift = misalign(dx + lo);
  const bool aligned = misalign(x + lo) == shift;
  for (int j = lo - shift + tid * kVec; j < hi; j += kChunk) {
    float z[8];
    if (DENSE) {
      load8(x, j, lo, hi, aligned, z);
#pragma unroll
      for (int i = 0; i < kVec; ++i) z[i] = dense(z[i]);
    } else {
#pragma unroll
      for (int i = 0; i < kVec; ++i) z[i] = 0.f;
    }
    if (j >= lo && j + kVec <= hi) {
      vec_store(dx + j, z);
    } else {
#pragma unroll
      for (int i = 0; i < kVec; ++i)
        if (j + i >= lo && j + i < hi) from_f(z[i], dx + j + i);
    }
  }
  __syncthreads();
  for (int i = tid; i <= k; i += kThreads) {
    const int at = sh_id[i];
    if (at < lo || at >= hi) continue;
    float sum = 0.f;
    bool mine = true;
    for (int n = 0; n <= k; ++n) {
      if (sh_id[n] != at) continue;
      if (n < i) mine = false;
      sum += sh_coef[n];
    }
    if (mine) from_f((DENSE ? dense(to_f(x[at])) : 0.f) + sum, dx + at);
  }
}

// Blocks per row of a forward pass: one while the rows fill the GPU, else up to kMaxSplit as long as a part is a full
// iteration of its block.
int split_of(int T, int V) {
  int n = 1;
  while (n < kMaxSplit && 2ll * n * T <= 2ll * txh::sm_count() && V / (2 * n) >= kChunk) n *= 2;
  return n;
}

template <auto Kernel, typename... Args>       // static flag: one per kernel, instantiations share a type
int launch_rows(int T, int blocks, int bytes, cudaStream_t s, Args... args) {
  static txh::DeviceFlag flag;
  if (bytes > 48 * 1024 && !flag.cur()) {
    if (cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return 401;
    flag.cur() = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(T) * blocks);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = blocks;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, Kernel, args...) == cudaSuccess ? 0 : 400;
}

template <typename LT>
int launch_bwd(BwdArgs a, int dense, cudaStream_t s) {
  const int want = 4 * txh::sm_count(), most = (a.V + kChunk - 1) / kChunk;
  a.blocks = min(most, a.T >= want ? 1 : (want + a.T - 1) / a.T);
#define TX_BWD(D) case D: top_bwd_kernel<LT, D><<<a.T * a.blocks, kThreads, 0, s>>>(a); break
  switch (dense) {
    TX_BWD(0); TX_BWD(1); TX_BWD(2); TX_BWD(3); TX_BWD(5);
    default: return 2;
  }
#undef TX_BWD
  return cudaGetLastError() == cudaSuccess ? 0 : 400;
}

}  // namespace

extern "C" int tx_top_max_k() { return kMaxTop; }
extern "C" int tx_top_max_list() { return kMaxList; }

// logits [T, V] with row stride ld (elements), fp32 or bf16; 1 <= k <= min(V, tx_top_max_k()).
extern "C" int tx_top_logprob_fwd(const void* logits, int logits_fp32, long long ld, int T, int V, int k,
                                  float inv_temp, const long long* targets, long long* ids, float* top, float* target,
                                  float* entropy, float* stats, cudaStream_t s) {
  if (T <= 0) return 0;
  if (V < 1 || k < 1 || k > kMaxTop || k > V || V > 0x7fff0000) return 1;
  const TopArgs a{logits, ld, T, V, k, inv_temp, targets, ids, top, target, entropy, reinterpret_cast<float2*>(stats)};
  const int n = split_of(T, V), bytes = sizeof(Select);
  if (logits_fp32)
    return entropy ? launch_rows<top_fwd_kernel<float, kEntropy>>(T, n, bytes, s, a)
                   : launch_rows<top_fwd_kernel<float, kNone>>(T, n, bytes, s, a);
  return entropy ? launch_rows<top_fwd_kernel<__nv_bfloat16, kEntropy>>(T, n, bytes, s, a)
                 : launch_rows<top_fwd_kernel<__nv_bfloat16, kNone>>(T, n, bytes, s, a);
}

extern "C" int tx_top_distill_fwd(const void* logits, int logits_fp32, long long ld, int T, int V, int k,
                                  float inv_temp, int full, const long long* ids, const float* values,
                                  const long long* labels, float* kl, float* nll, float* stats, cudaStream_t s) {
  if (T <= 0) return 0;
  if (V < 1 || k < 1 || k > kMaxList || V > 0x7fff0000) return 1;
  const DistillArgs a{logits, ld, T, V, k, inv_temp, full, ids, values, labels, kl, nll, reinterpret_cast<float4*>(stats)};
  const float c = inv_temp * kLog2e;
  const int passes = (nll ? 1 : 0) + (full ? 1 : 0) - (nll && full && inv_temp == 1.f ? 1 : 0);
  const float c1 = nll ? kLog2e : c;
  const int n = split_of(T, V);
#define TX_FWD(LT)                                                                          \
  if (passes == 1) return launch_rows<distill_fwd_kernel<LT, 1>>(T, n, 0, s, a, c1, c);      \
  if (passes == 2) return launch_rows<distill_fwd_kernel<LT, 2>>(T, n, 0, s, a, c1, c);      \
  distill_fwd_kernel<LT, 0><<<T, 32, 0, s>>>(a, c1, c)
  if (logits_fp32) { TX_FWD(float); } else { TX_FWD(__nv_bfloat16); }
#undef TX_FWD
  return cudaGetLastError() == cudaSuccess ? 0 : 400;
}

// Gradient of tx_top_logprob_fwd: values = gradients of the list (or null), given = targets.
extern "C" int tx_top_logprob_bwd(const void* logits, int logits_fp32, long long ld, int T, int V, int k,
                                  float inv_temp, const long long* ids, const float* g_top, const long long* targets,
                                  const float* g_target, const float* g_entropy, const float* entropy,
                                  const float* stats, void* dx, long long ldd, cudaStream_t s) {
  if (T <= 0) return 0;
  if (V < 1 || k < 1 || k > kMaxTop || V > 0x7fff0000) return 1;
  const BwdArgs a{logits, ld, T, V, k, kScore, inv_temp, ids, g_top, targets, nullptr, g_target, g_entropy, entropy,
                  stats, 2, 1, 1, dx, ldd, 1};
  const int dense = g_entropy ? 5 : 1;
  return logits_fp32 ? launch_bwd<float>(a, dense, s) : launch_bwd<__nv_bfloat16>(a, dense, s);
}

// Gradient of tx_top_distill_fwd; g_kl or g_nll may be null.
extern "C" int tx_top_distill_bwd(const void* logits, int logits_fp32, long long ld, int T, int V, int k,
                                  float inv_temp, int full, const long long* ids, const float* values,
                                  const long long* labels, const float* g_kl, const float* g_nll, const float* stats,
                                  void* dx, long long ldd, cudaStream_t s) {
  if (T <= 0) return 0;
  if (V < 1 || k < 1 || k > kMaxList || V > 0x7fff0000) return 1;
  const BwdArgs a{logits, ld, T, V, k, full ? kFull : kListed, inv_temp, ids, values, labels, g_kl, g_nll, nullptr,
                  nullptr, stats, 4, 1, 2, dx, ldd, 1};
  const int dense = (full && g_kl ? 1 : 0) | (g_nll ? 2 : 0);
  return logits_fp32 ? launch_bwd<float>(a, dense, s) : launch_bwd<__nv_bfloat16>(a, dense, s);
}
