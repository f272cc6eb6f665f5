// Operators on rows of logits that report or learn from the k best entries of a row.
//
//  * tx_top_logprob_fwd: log-probability of one given token, the k largest logits (ids and log-probabilities, equal
//    values by the lowest id) and the entropy of softmax(x * inv_temp), in one pass over the row.
//  * tx_top_distill_fwd: per row the divergence from a teacher's list of (id, value) pairs and the cross entropy of
//    a label, in one pass over the student's row (none at all when only the listed entries matter).
//  * tx_top_logprob_bwd, tx_top_distill_bwd: the gradient of either with respect to the row, one read and one write
//    (one write alone where the dense part of the gradient is zero).
//
// With m = max x, d_j = x_j - m and c = inv_temp * log2(e):  s = sum 2^(d_j c),  log p_j = d_j inv_temp - ln s.
// What is reported is kept relative to m, so log-probabilities do not lose the bits of a large log-sum-exp. Sums,
// maxima and the list's statistics are fp32. A row of -inf is an empty row: ln s is stored as +inf, log-probabilities
// are -inf, losses and gradients 0.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <stdint.h>

#include "tx_host.h"

namespace cg = cooperative_groups;

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kUnroll = 4;                    // 16-byte vectors a thread has in flight
constexpr int kMaxTop = 256;                  // longest list of alternatives
constexpr int kMaxList = 1024;                // longest teacher's list
constexpr int kCand = 2560;                   // candidates of a block
constexpr int kKept = 1024;                   // of which this many may reach the last threshold
constexpr int kKeys = 2048;                   // elements that do
constexpr int kBins = 256;
constexpr int kMaxSplit = 8;                  // blocks (one cluster) a row is spread over when there are few rows
constexpr int kMinPart = 4096;                // columns of a part of the backward pass at least
constexpr int kBwdPart = 32768;               // columns a block of the backward pass takes at most
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr double kLog2eFine = 1.4426950408889634;
constexpr float kFloor = -1e37f;              // lowest running maximum

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
__device__ __forceinline__ uint32_t max_nan_bf16x2(uint32_t a, uint32_t b) {
  uint32_t y;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
  return y;
}

// Two floats in one 64-bit register: half the instructions of the scalar forms.
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pack2(float a, float b) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpack2(f32x2 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// 2^t for two t <= 0 without the special function unit: 2^n from the exponent, n the nearest integer, times a
// polynomial in the rest (|f| <= 1/2; degree 5, fitted for the smallest relative error: 2.2e-7 with fp32 roundings, as
// ex2). Below -126 the result stays at 2^-126.
__device__ __forceinline__ f32x2 ex2_by_fma(float a, float b) {
  const float kShift = 12582912.f;                 // 1.5 * 2^23: the sum's low bits are the nearest integer
  const f32x2 t = pack2(fmaxf(a, -126.f), fmaxf(b, -126.f));
  const f32x2 n = add2(t, pack2(kShift, kShift));
  const f32x2 f = fma2(add2(n, pack2(-kShift, -kShift)), pack2(-1.f, -1.f), t);
  f32x2 p = fma2(f, pack2(0.0013276472f, 0.0013276472f), pack2(0.009675541f, 0.009675541f));
  p = fma2(f, p, pack2(0.05550713f, 0.05550713f));
  p = fma2(f, p, pack2(0.2402212f, 0.2402212f));
  p = fma2(f, p, pack2(0.69314694f, 0.69314694f));
  p = fma2(f, p, pack2(1.0000001f, 1.0000001f));
  const float2 q = unpack2(p), e = unpack2(n);
  return pack2(__int_as_float(__float_as_int(q.x) + (__float_as_int(e.x) << 23)),
               __int_as_float(__float_as_int(q.y) + (__float_as_int(e.y) << 23)));
}

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void from_f(float v, float* p) { *p = v; }
__device__ __forceinline__ void from_f(float v, __nv_bfloat16* p) { *p = __float2bfloat16_rn(v); }

// ---- 16-byte vectors of a row ---------------------------------------------------------------------------
template <typename T>
constexpr int kVec = 16 / static_cast<int>(sizeof(T));
template <typename T>
constexpr int kChunk = kThreads * kVec<T>;    // elements the block takes with one vector per thread

__device__ __forceinline__ void unpack(uint4 u, float (&z)[4]) {
  z[0] = __uint_as_float(u.x); z[1] = __uint_as_float(u.y); z[2] = __uint_as_float(u.z); z[3] = __uint_as_float(u.w);
}
__device__ __forceinline__ void unpack(uint4 u, float (&z)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    z[2 * i] = __uint_as_float(w[i] << 16);
    z[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ uint4 pack(const float (&z)[4]) {
  return make_uint4(__float_as_uint(z[0]), __float_as_uint(z[1]), __float_as_uint(z[2]), __float_as_uint(z[3]));
}
__device__ __forceinline__ uint4 pack(const float (&z)[8]) {
  uint4 u;
  __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(z[2 * i], z[2 * i + 1]);
  return u;
}
// Element e of a vector.
template <typename T>
__device__ __forceinline__ float element(uint4 u, int e) {
  const int word = sizeof(T) == 2 ? e / 2 : e;
  const uint32_t v = word < 2 ? (word == 0 ? u.x : u.y) : (word == 2 ? u.z : u.w);
  return __uint_as_float(sizeof(T) == 4 ? v : (e & 1 ? v & 0xffff0000u : v << 16));
}
// Maxima of vectors, kept packed for bf16: `scalar` is the one number.
template <typename T>
struct Top;
template <>
struct Top<float> {
  float v;
  __device__ __forceinline__ static Top of(uint4 u) {
    return Top{max_nan(max_nan(__uint_as_float(u.x), __uint_as_float(u.y)), max_nan(__uint_as_float(u.z), __uint_as_float(u.w)))};
  }
  __device__ __forceinline__ static Top max(Top a, Top b) { return Top{max_nan(a.v, b.v)}; }
  __device__ __forceinline__ float scalar() const { return v; }
};
template <>
struct Top<__nv_bfloat16> {
  uint32_t v;
  __device__ __forceinline__ static Top of(uint4 u) {
    return Top{max_nan_bf16x2(max_nan_bf16x2(u.x, u.y), max_nan_bf16x2(u.z, u.w))};
  }
  __device__ __forceinline__ static Top max(Top a, Top b) { return Top{max_nan_bf16x2(a.v, b.v)}; }
  __device__ __forceinline__ float scalar() const {
    return max_nan(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  }
};

// How many elements an address lies behind the last 16-byte boundary.
template <typename T>
__device__ __forceinline__ int misalign(const T* p) {
  return static_cast<int>((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T));
}

// The vector that begins at element j of a row; elements outside [lo, hi) are -inf. `aligned`: the address of j is.
template <typename T>
__device__ __forceinline__ uint4 load_vec(const T* row, int j, int lo, int hi, bool aligned) {
  if (aligned && j >= lo && j + kVec<T> <= hi) return *reinterpret_cast<const uint4*>(row + j);
  const uint32_t none = sizeof(T) == 2 ? 0xff80ff80u : 0xff800000u;
  if (j >= hi) return make_uint4(none, none, none, none);
  float z[kVec<T>];
#pragma unroll
  for (int i = 0; i < kVec<T>; ++i) z[i] = (j + i >= lo && j + i < hi) ? to_f(row[j + i]) : -INFINITY;
  return pack(z);
}

template <typename T>
__device__ __forceinline__ void store_vec(T* row, int j, int lo, int hi, const float (&z)[kVec<T>]) {
  if (j >= lo && j + kVec<T> <= hi) {
    *reinterpret_cast<uint4*>(row + j) = pack(z);
  } else {
#pragma unroll
    for (int i = 0; i < kVec<T>; ++i)
      if (j + i >= lo && j + i < hi) from_f(z[i], row + j + i);
  }
}

// Columns of a row that block `rank` of `blocks` takes: equal parts, cut at multiples of 8 from the first one.
__device__ __forceinline__ int2 part_of(int V, int rank, int blocks) {
  const int vecs = (V + 7) / 8;
  const int per = (vecs + blocks - 1) / blocks * 8;
  return make_int2(min(V, rank * per), min(V, rank * per + per));
}

// ---- softmax statistics --------------------------------------------------------------------------------
// A thread sums 2^(x c - M) with M = m c rounded: one packed multiply-add per two elements. The rounding of M is the
// same in every term and is taken back from the logarithm at the end. Where m c leaves fp32, or every element lies
// below the floor of the running maximum, the sum comes out as 0 (far below 1, where it should not) or NaN and the row
// is summed again the careful way.
constexpr int kNone = 0, kEntropy = 1, kSecond = 2;

struct Stat {
  float m;    // maximum
  float s;    // sum 2^(x c - M)
  float t;    // kEntropy: sum 2^(x c - M) (x c - M); kSecond: the sum at the scale c2
};

__device__ __forceinline__ float scaled_max(float m, float c) { return fmaxf(m * c, -FLT_MAX); }

template <int X>
struct Acc {
  float m, M, M2;
  f32x2 s, t;

  __device__ __forceinline__ void init(float first, float c, float c2) {
    m = fmaxf(first, kFloor);
    M = scaled_max(m, c);
    if (X == kSecond) M2 = scaled_max(m, c2);
    s = t = 0;
  }
  __device__ __forceinline__ void raise(float v, float c, float c2) {
    const float n = scaled_max(v, c), d = M - n, e = ex2(d);
    const f32x2 ee = pack2(e, e);
    if (X == kEntropy) t = e == 0.f ? 0 : mul2(fma2(s, pack2(d, d), t), ee);
    if (X == kSecond) {
      const float n2 = scaled_max(v, c2), e2 = ex2(M2 - n2);
      t = mul2(t, pack2(e2, e2));
      M2 = n2;
    }
    s = mul2(s, ee);
    m = v;
    M = n;
  }
  // Adds a vector none of whose elements is above m.
  template <typename LT>
  __device__ __forceinline__ void push(uint4 u, float c, float c2) {
    float z[kVec<LT>];
    unpack(u, z);
    const f32x2 cc = pack2(c, c), mm = pack2(-M, -M);
    const f32x2 cc2 = pack2(c2, c2), mm2 = pack2(-M2, -M2);
#pragma unroll
    for (int i = 0; i < kVec<LT>; i += 2) {
      const f32x2 zz = pack2(z[i], z[i + 1]);
      const float2 g = unpack2(fma2(zz, cc, mm));
      const f32x2 w = pack2(ex2(g.x), ex2(g.y));
      s = add2(s, w);
      if (X == kEntropy) t = fma2(w, pack2(fmaxf(g.x, -1e30f), fmaxf(g.y, -1e30f)), t);     // 0 * -inf would be NaN
      if (X == kSecond) {
        const float2 h = unpack2(fma2(zz, cc2, mm2));
        // two exponentials per bf16 element are more than the special function unit has time for while the row streams
        // in: of 16 per vector it takes 12 (4096 x 151936: 266 us; 313 us with all 16, 289 us with 14, 287 us with 10)
        t = add2(t, sizeof(LT) == 2 && i >= 4 ? ex2_by_fma(h.x, h.y) : pack2(ex2(h.x), ex2(h.y)));
      }
    }
  }
  __device__ __forceinline__ Stat stat() const {
    const float2 a = unpack2(s), b = unpack2(t);
    return Stat{m, a.x + a.y, b.x + b.y};
  }
};

template <int X>
__device__ __forceinline__ void stat_raise(Stat& a, float m, float c, float c2) {
  const float d = scaled_max(a.m, c) - scaled_max(m, c), e = ex2(d);
  if (X == kEntropy) a.t = e == 0.f ? 0.f : e * fmaf(a.s, d, a.t);
  if (X == kSecond) a.t *= ex2(scaled_max(a.m, c2) - scaled_max(m, c2));
  a.s *= e;
  a.m = m;
}

template <int X>
__device__ __forceinline__ void stat_merge(Stat& a, Stat b, float c, float c2) {
  if (a.m != b.m) {
    const float m = fmaxf(a.m, b.m);
    stat_raise<X>(a, m, c, c2);
    stat_raise<X>(b, m, c, c2);
  }
  a.s += b.s;
  a.t += b.t;
}

__device__ __forceinline__ float warp_max_of(float v) {
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float warp_sum_of(float v) {
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The block's statistics in every thread, the maximum first, then sums relative to it. Between the steps, and before
// `sh` (kWarps entries) is used again, the block synchronises.
__device__ __forceinline__ void stat_max(const Stat& a, Stat* sh) {
  const float m = warp_max_of(a.m);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5].m = m;
}
template <int X>
__device__ __forceinline__ void stat_sums(Stat& a, Stat* sh, float c, float c2) {
  float m = sh[0].m;
  for (int w = 1; w < kWarps; ++w) m = fmaxf(m, sh[w].m);
  if (a.m != m) stat_raise<X>(a, m, c, c2);
  a.s = warp_sum_of(a.s);
  if (X != kNone) a.t = warp_sum_of(a.t);
  if ((threadIdx.x & 31) == 0) {
    sh[threadIdx.x >> 5].s = a.s;
    sh[threadIdx.x >> 5].t = a.t;
  }
}
template <int X>
__device__ __forceinline__ Stat stat_all(Stat a, const Stat* sh) {
  a.s = a.t = 0.f;
  for (int w = 0; w < kWarps; ++w) {
    a.s += sh[w].s;
    if (X != kNone) a.t += sh[w].t;
  }
  return a;
}

// What a row's softmax comes to. ls = +inf marks a row without an element above -inf.
struct Row {
  float m, ls;      // maximum, ln sum exp((x - m) at the scale)
  float x;          // kEntropy: the entropy; kSecond: ln of the sum at the scale c2
  bool careful;     // from differences to the true maximum: there is no sum 2^(x c - M)
};

__device__ __forceinline__ float log_sum(float s) { return s == 0.f ? INFINITY : logf(s); }

// ln s of a positive, finite and normal s: the logarithm's argument is brought near 1, where its rounding is small.
__device__ __forceinline__ double log_fine(float s) {
  int e;
  float f = frexpf(s, &e);                                   // in [0.5, 1)
  if (f < 0.75f) {
    f += f;
    --e;
  }
  return fma(static_cast<double>(e), 0.69314718055994531, static_cast<double>(logf(f)));
}
// ln sum exp((x - m) at the scale), from s = sum 2^(x c - M) with M rounded.
__device__ __forceinline__ double log_fine(float s, float m, float c) {
  const double rounded = fma(static_cast<double>(m), static_cast<double>(c), -static_cast<double>(scaled_max(m, c)));
  return fma(-0.69314718055994531, rounded, log_fine(s));
}

// Row statistics from differences to the true maximum, by the whole block over the whole row.
template <typename LT, int X>
__device__ __noinline__ Row careful_row(const LT* x, int V, Stat* sh, float c, float c2) {
  float m = -INFINITY;
  for (int j = threadIdx.x; j < V; j += kThreads) m = fmaxf(m, to_f(x[j]));
  Stat a{m, 0.f, 0.f};
  __syncthreads();
  for (int o = 16; o > 0; o >>= 1) a.m = fmaxf(a.m, __shfl_xor_sync(0xffffffffu, a.m, o));
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = a;
  __syncthreads();
  m = -FLT_MAX;
  for (int w = 0; w < kWarps; ++w) m = fmaxf(m, sh[w].m);
  float s = 0.f, t = 0.f;
  for (int j = threadIdx.x; j < V; j += kThreads) {
    const float d = to_f(x[j]) - m, w = ex2(d * c);
    s += w;
    if (X == kEntropy) t = fmaf(w, fmaxf(d * c, -1e30f), t);
    if (X == kSecond) t += ex2(d * c2);
  }
  for (int o = 16; o > 0; o >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    t += __shfl_xor_sync(0xffffffffu, t, o);
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = Stat{m, s, t};
  __syncthreads();
  s = t = 0.f;
  for (int w = 0; w < kWarps; ++w) {
    s += sh[w].s;
    t += sh[w].t;
  }
  Row r{m, log_sum(s), 0.f, true};
  if (X == kEntropy) r.x = s == 0.f ? 0.f : r.ls - kLn2 * (t / s);
  if (X == kSecond) r.x = log_sum(t);
  return r;
}

// All threads of the block call it with the row's statistics.
template <typename LT, int X>
__device__ __forceinline__ Row finish_row(const Stat& a, const LT* x, int V, Stat* sh, float c, float c2) {
  // the maximum alone contributes 1
  if (!(a.s > 0.5f && a.s < INFINITY && (X != kSecond || (a.t > 0.5f && a.t < INFINITY))))
    return careful_row<LT, X>(x, V, sh, c, c2);
  Row r;
  r.careful = false;
  r.m = a.m;
  const float ln = logf(a.s);
  r.ls = fmaf(-kLn2, fmaf(a.m, c, -scaled_max(a.m, c)), ln);          // M - m c, exactly
  r.x = 0.f;
  if (X == kEntropy) r.x = ln - kLn2 * (a.t / a.s);
  if (X == kSecond) r.x = fmaf(-kLn2, fmaf(a.m, c2, -scaled_max(a.m, c2)), logf(a.t));
  return r;
}

// Asks for what the warp reads in the iteration that begins at element `at`, 128 bytes per lane, so that its loads find
// it in L2: a block's threads wait for each other only at a row's ends, but each has only one iteration's loads in
// flight. One iteration ahead 8192 x 128256 bf16 with k = 64 takes 360 us, two 366 us, four 374 us, none 388 us; bulk
// prefetches of 512 bytes 375 us. In the backward pass it pays where an element takes two terms (1000 x 262144 bf16
// with entropy: 163 us, 172 us without); with one, 4096 x 128256 takes 323 us instead of 326 us for itself, but 340 us
// instead of 333 us in long runs under the power cap.
template <typename LT>
__device__ __forceinline__ void ask_ahead(const LT* x, int at, int hi) {
  constexpr int line = 128 / sizeof(LT);                     // a warp's vectors side by side are four lines
  const int lane = threadIdx.x & 31;
  const int j = at + (threadIdx.x >> 5) * 4 * line + lane / 4 * kChunk<LT> + lane % 4 * line;
  if (lane < 4 * kUnroll && j < hi) asm volatile("prefetch.global.L2 [%0];" ::"l"(x + j));
}

// The block's vectors of columns [lo, hi) from element `from` on, kUnroll per thread at a time: fn(first element of the
// thread, vectors, how many of them begin inside; the last may reach out and is then filled with -inf).
template <typename LT, typename Fn>
__device__ __forceinline__ void each_vec(const LT* x, int from, int lo, int hi, Fn fn) {
  constexpr int step = kUnroll * kChunk<LT>;
  int at = from;
  uint4 u[kUnroll];
  for (; at >= lo && at + step <= hi; at += step) {
    const int j = at + threadIdx.x * kVec<LT>;
    ask_ahead(x, at + step, hi);
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) u[i] = *reinterpret_cast<const uint4*>(x + j + i * kChunk<LT>);
    fn(j, u, kUnroll);
  }
  for (; at < hi; at += step) {
    const int j = at + threadIdx.x * kVec<LT>, n = min(kUnroll, (hi - at + kChunk<LT> - 1) / kChunk<LT>);
#pragma unroll
    for (int i = 0; i < kUnroll; ++i)
      if (i < n) u[i] = load_vec(x, j + i * kChunk<LT>, lo, hi, true);
    fn(j, u, n);
  }
}

// The maximum of n vectors.
template <typename LT>
__device__ __forceinline__ float max_vecs(const uint4 (&u)[kUnroll], int n) {
  Top<LT> all = Top<LT>::of(u[0]);
#pragma unroll
  for (int i = 1; i < kUnroll; ++i)
    if (i < n) all = Top<LT>::max(all, Top<LT>::of(u[i]));
  return all.scalar();
}

// Adds n vectors of the given maximum.
template <typename LT, int X>
__device__ __forceinline__ void add_vecs(Acc<X>& acc, const uint4 (&u)[kUnroll], int n, float most, float c, float c2) {
  if (most > acc.m) acc.raise(most, c, c2);
#pragma unroll
  for (int i = 0; i < kUnroll; ++i)
    if (i < n) acc.template push<LT>(u[i], c, c2);
}

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

// Sorts n keys (all different) in shared memory from high to low. All threads call it. Short lists: four or two threads
// count how many keys are above theirs. Longer ones: bitonic (slots n .. P-1 are filled with 0, P the next power of 2);
// up to one key per thread stays in a register and strides below a warp are shuffles.
__device__ __forceinline__ void sort_keys(unsigned long long* keys, int n) {
  if (n <= kThreads / 2) {
    const int per = n <= kThreads / 4 ? 4 : 2, i = threadIdx.x / per, sub = threadIdx.x % per;
    const unsigned long long key = i < n ? keys[i] : 0;
    int above = 0;
    for (int j = sub; i < n && j < n; j += per) above += keys[j] > key;
    above += __shfl_xor_sync(0xffffffffu, above, 1);
    if (per == 4) above += __shfl_xor_sync(0xffffffffu, above, 2);
    __syncthreads();
    if (i < n && sub == 0) keys[above] = key;
    __syncthreads();
    return;
  }
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

// The row's target and its logit.
struct Given {
  long long at;
  float value;
};

// Numbers in the order of floats; a NaN counts as +inf.
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t b = __float_as_uint(x != x ? INFINITY : x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_order(uint32_t o) {
  return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}

// The n-th largest number of a warp (1 <= n <= 32), neither 0 nor ~0 among them, from the nearer end: the extreme one
// is taken away until it is that one's turn (8192 x 32000 bf16 with k = 20: 129 us, 135 us with a sort of the warp;
// with k = 64, eight rounds, both are the same).
__device__ __forceinline__ uint32_t nth_largest(uint32_t v, int n) {
  const bool down = n <= 16;
  int left = down ? n : 33 - n;
  if (!down) v = ~v;
  uint32_t top;
  while (true) {
    top = __reduce_max_sync(0xffffffffu, v);
    left -= __popc(__ballot_sync(0xffffffffu, v == top));
    if (left <= 0) break;
    if (v == top) v = 0;
  }
  return down ? top : ~top;
}

// Selection state of a block.
//
// A candidate is what a thread takes in one iteration (kUnroll vectors), when its largest element is not below a
// threshold that k elements of the block's part are known to reach. The first threshold comes from the first iteration:
// the smallest over the warps of the ceil(k / warps)-th largest of a warp's per-thread maxima (of the warps that have a
// whole vector per thread). From then on the maxima of candidates are counted in bins of equal width above it, and in
// every other iteration one warp moves the threshold up to a bin below the lowest bin that k of them reach. Bin numbers
// (rounded to the nearest) and that edge are computed with monotone roundings, so an element of such a bin is never
// below the edge. At the end the candidates that still reach the threshold are read again (from L2), a vector per
// thread, and their elements that do are sorted: little more than k. Every step is dense over the block's threads: for
// all but the smallest k the kernel is bound by the instructions it issues, not by the memory.
struct Select {
  unsigned long long keys[kKeys];
  union {
    uint32_t cand[kCand];                // largest element as bf16, rounded up | iteration * kThreads + thread
    unsigned long long binned[kCand / 2];
  };
  uint16_t kept[kKept];
  int bins[kBins], next[kBins];
  int widest;
  int count, n_kept, n_keys;
  float thr;
  float warp_nth[kWarps], warp_max[kWarps];
  Stat stat[kWarps];
  Stat part;                   // this block's statistics, read by the cluster's first block
};

__device__ __forceinline__ int bin_of(float x, float thr0, float inv_width) {
  return __float_as_int(fminf((x - thr0) * inv_width, static_cast<float>(kBins - 1)) + 8388608.f) & (kBins - 1);
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

// The k best of columns [lo, hi) into keys[0 .. k), sorted, for rows whose candidates do not fit (many equal or masked
// elements): elements come in order of their index, one per thread and iteration, so from the first full set on only
// larger ones than the k-th can enter.
template <typename LT>
__device__ __noinline__ void select_in_order(Select& s, const LT* x, int lo, int hi, int k) {
  constexpr int limit = kKeys - kThreads;
  static_assert(limit > kMaxTop, "");
  float thr = -INFINITY;
  bool any = true;                                   // no threshold yet
  __syncthreads();
  if (threadIdx.x == 0) s.n_keys = 0;
  __syncthreads();
  for (int base = lo; base < hi; base += kThreads) {
    const int j = base + threadIdx.x;
    int over = 0;
    if (j < hi) {
      const float v = to_f(x[j]);
      if (any || !(v <= thr)) {
        const int pos = atomicAdd(&s.n_keys, 1);
        s.keys[pos] = key_of(v, j);                  // below the limit before this iteration
        over = pos >= limit - 1;
      }
    }
    // the first full set is cut at once: it holds every element so far
    if (__syncthreads_or(over || (any && base + kThreads - lo >= k))) {
      sort_keys(s.keys, s.n_keys);
      any = s.n_keys < k;
      if (!any) thr = key_value(s.keys[k - 1]);
      __syncthreads();
      if (threadIdx.x == 0) s.n_keys = min(s.n_keys, k);
      __syncthreads();
    }
  }
  sort_keys(s.keys, s.n_keys);
}

// Sorts the first k of n keys from high to low with the bins they were counted in: a key goes behind the keys of higher
// bins, its place among those of its own (a few, as long as few elements are equal) is counted. All threads call it.
// 8192 rows of 8000 with k = 200 (before the steps around it became shorter): 191 us, 277 us with a bitonic sort.
__device__ __forceinline__ void sort_binned(Select& s, int n, int k, float thr0, float inv_width) {
  const int tid = threadIdx.x;
  if (n <= kThreads / 4) {                                   // counting all of them is less
    sort_keys(s.keys, n);
    return;
  }
  if (tid < 32) {                                            // lane 0 has the highest bins
    const int top = kBins - 1 - tid * (kBins / 32);
    int c[kBins / 32], sum = 0, most = 0;
#pragma unroll
    for (int i = 0; i < kBins / 32; ++i) {
      c[i] = s.bins[top - i];
      sum += c[i];
      most = max(most, c[i]);
    }
    int upto = sum;
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (tid >= o) upto += v;
    }
    upto -= sum;
#pragma unroll
    for (int i = 0; i < kBins / 32; ++i) {
      s.next[top - i] = upto;
      upto += c[i];
    }
    for (int o = 16; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
    if (tid == 0) s.widest = most;
  }
  __syncthreads();
  if (s.widest > 64 || n > kCand / 2) {                      // many in one bin
    sort_keys(s.keys, n);
    return;
  }
  for (int i = tid; i < n; i += kThreads) {
    const unsigned long long key = s.keys[i];
    s.binned[atomicAdd(&s.next[bin_of(key_value(key), thr0, inv_width)], 1)] = key;
  }
  __syncthreads();
  for (int i = tid; i < n; i += kThreads) {
    const unsigned long long key = s.binned[i];
    const int b = bin_of(key_value(key), thr0, inv_width);
    const int end = s.next[b], begin = end - s.bins[b];
    if (begin >= k) continue;
    int at = begin;
    for (int q = begin; q < end; ++q) at += s.binned[q] > key;
    s.keys[at] = key;
  }
  __syncthreads();
}

// The k best of columns [lo, hi) into s.keys, sorted, and the statistics of the part. `base`: the first column of the
// first vector.
template <typename LT, int X>
__device__ __forceinline__ Stat top_of_part(Select& s, const LT* x, int base, int lo, int hi, int k, float c,
                                            const long long* targets, int V, Given& given) {
  constexpr int N = kVec<LT>, chunk = kChunk<LT>;
  const int tid = threadIdx.x, lane = tid & 31;
  for (int i = tid; i < kBins; i += kThreads) s.bins[i] = 0;
  if (tid == 0) s.count = s.n_kept = s.n_keys = 0;
  // ---- first iteration: the first threshold
  Acc<X> acc;
  uint4 u[kUnroll];
  ask_ahead(x, base + kUnroll * chunk, hi);
  const int count = min(kUnroll, (hi - base + chunk - 1) / chunk);
#pragma unroll
  for (int i = 0; i < kUnroll; ++i)
    if (i < count) u[i] = load_vec(x, base + tid * N + i * chunk, lo, hi, true);
  const float most = max_vecs<LT>(u, count);
  const int whole = min(kWarps, max(0, hi - base) / (32 * N));
  const int nth_of = whole ? (k + whole - 1) / whole : 33;             // more than a warp's threads: no threshold
  const uint32_t order = order_of(most);
  const float warp_max = of_order(__reduce_max_sync(0xffffffffu, order));
  const float nth = of_order(nth_largest(order, min(nth_of, 32)));
  if (lane == 0) {
    s.warp_nth[tid >> 5] = nth;
    s.warp_max[tid >> 5] = warp_max;
  }
  acc.init(warp_max, c, 0.f);                                          // later maxima are rare
  add_vecs<LT, X>(acc, u, count, most, c, 0.f);
  __syncthreads();
  float thr0 = INFINITY, block_max = s.warp_max[0];
  for (int w = 0; w < kWarps; ++w) {
    if (w < whole) thr0 = fminf(thr0, s.warp_nth[w]);
    block_max = fmaxf(block_max, s.warp_max[w]);
  }
  if (nth_of > 32) thr0 = -INFINITY;
  // 128 bins up to the first iteration's maximum; any positive width is correct
  float width = (block_max - thr0) * (1.f / 128.f);
  if (!(width > 1e-30f && width < 1e30f)) width = 1.f;
  const float inv_width = 1.f / width;
  if (tid == 0) s.thr = thr0;
  float thr = thr0;
  __syncthreads();
  volatile float* shared_thr = &s.thr;
  int it = 0;
  auto offer = [&](float most) {
    if (!(most < thr)) {
      const uint32_t bits = __float_as_uint(most);
      const uint32_t up = (bits + (most >= 0.f ? 0xffffu : 0u)) & 0xffff0000u;
      const int pos = atomicAdd(&s.count, 1);
      if (pos < kCand) s.cand[pos] = up | static_cast<uint32_t>(it * kThreads + tid);
      atomicAdd(&s.bins[bin_of(most, thr0, inv_width)], 1);
    }
    if ((it & 1) && ((it >> 1) & (kWarps - 1)) == tid >> 5) {
      const int b = cut_bin(s.bins, k);
      const float t = fmaf(b - 1.f, width, thr0);
      if (lane == 0 && b > 1 && t > *shared_thr) *shared_thr = t;
      __syncwarp();
    }
    ++it;
  };
  offer(most);
  each_vec(x, base + kUnroll * chunk, lo, hi, [&](int, const uint4 (&w)[kUnroll], int n) {
    thr = *shared_thr;
    const float t = max_vecs<LT>(w, n);
    add_vecs<LT, X>(acc, w, n, t, c, 0.f);
    offer(t);
  });
  Stat st = acc.stat();
  stat_max(st, s.stat);
  __syncthreads();
  if (tid == 0 && targets) given.at = *targets;              // the loads come back while the candidates are sorted
  stat_sums<X>(st, s.stat, c, 0.f);
  // ---- the candidates' elements, sorted
  const int n = s.count;
  bool fits = n <= kCand && hi - base <= 65536 / kThreads * kUnroll * chunk;
  if (fits) {
    if (tid < 32) {
      const int b = cut_bin(s.bins, k);
      const float t = fmaf(b - 1.f, width, thr0);
      if (tid == 0 && b > 1 && t > *shared_thr) *shared_thr = t;
    }
    __syncthreads();
    thr = *shared_thr;
    for (int i = tid; i < n; i += kThreads) {
      const uint32_t word = s.cand[i];
      if (__uint_as_float(word & 0xffff0000u) < thr) continue;
      const int pos = atomicAdd(&s.n_kept, 1);
      if (pos < kKept) s.kept[pos] = static_cast<uint16_t>(word);
    }
    for (int i = tid; i < kBins; i += kThreads) s.bins[i] = 0;
    __syncthreads();
    fits = s.n_kept <= kKept;
  }
  if (given.at >= 0 && given.at < V) given.value = to_f(x[given.at]);
  if (fits) {
    for (int i = tid; i < s.n_kept * kUnroll; i += kThreads) {
      const int at = s.kept[i / kUnroll];
      const int j = base + (at / kThreads * kUnroll + i % kUnroll) * chunk + at % kThreads * N;
      const uint4 w = load_vec(x, j, lo, hi, true);
      if (Top<LT>::of(w).scalar() < thr) continue;
      float z[N];
      unpack(w, z);
      unsigned above = 0;                                    // its elements that reach the threshold, usually one
#pragma unroll
      for (int e = 0; e < N; ++e) above |= !(z[e] < thr) && j + e >= lo && j + e < hi ? 1u << e : 0u;
      int pos = atomicAdd(&s.n_keys, __popc(above));
      for (; above; above &= above - 1) {
        const int e = __ffs(above) - 1;
        const float v = element<LT>(w, e);
        if (pos < kKeys) s.keys[pos] = key_of(v, j + e);
        ++pos;
        atomicAdd(&s.bins[bin_of(v, thr0, inv_width)], 1);
      }
    }
    __syncthreads();
    fits = s.n_keys <= kKeys;
  }
  if (fits)
    sort_binned(s, s.n_keys, k, thr0, inv_width);
  else
    select_in_order(s, x, lo, hi, k);
  return stat_all<X>(st, s.stat);
}

// A row per cluster of 1 .. kMaxSplit blocks, each with a part of the columns.
//
// Long rows with small k are bound by memory (8192 x 128256 bf16, k = 1: 312 us, 6.7 TB/s), with larger k by the
// instructions of the selection, a fifth on top of those of the sums at k = 64 (349 us, 6.0 TB/s; k = 256: 430 us).
// Five blocks of 256 threads per SM hide one row's serial parts (first threshold, last sort) behind the others'
// streaming. Short rows are mostly those parts: 8192 x 32000, k = 20: 130 us, 4.0 TB/s (blocks of 128 threads take 113
// us there, but 357 us where this takes 349 us). Tried at 8192 x 128256, k = 64: a ring of asynchronous copies with two
// blocks per SM 649 us where this took 415 us, two blocks per row 557 us and six blocks with 40 registers 390 us where
// it took 361 us. 2047 x 151936 fp32 with entropy, k = 8: 198 us (6.3 TB/s). Under the power cap of a long run the
// clock falls and these times grow by up to a tenth.
template <typename LT, int X>
__global__ void __launch_bounds__(kThreads, X == kNone ? 5 : 4) top_fwd_kernel(TopArgs a) {
  extern __shared__ __align__(16) unsigned char shared[];
  Select& s = *reinterpret_cast<Select*>(shared);
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int row = blockIdx.x / blocks, tid = threadIdx.x, k = a.k;
  const LT* x = static_cast<const LT*>(a.logits) + static_cast<long long>(row) * a.ld;
  const float c = a.inv_temp * kLog2e;
  const int2 part = part_of(a.V, rank, blocks);
  const int lo = part.x, hi = part.y, base = lo - misalign(x + lo);
  Given given{-1, 0.f};
  Stat st = top_of_part<LT, X>(s, x, base, lo, hi, k, c, a.target && rank == 0 ? a.targets + row : nullptr, a.V, given);
  int at = tid;                          // place of this thread's key among the k best of the row
  if (blocks > 1) {
    const int mine = min(k, hi - lo);
    if (tid == 0) {
      s.part = st;
      s.n_keys = mine;
    }
    cluster.sync();
    // Every block takes in all parts, in the same order, and counts for its own keys those above them in the others'
    // sorted lists: binary searches through distributed shared memory, side by side.
    Stat parts[kMaxSplit];
    int l[kMaxSplit], h[kMaxSplit];
#pragma unroll
    for (int r = 0; r < kMaxSplit; ++r) {
      const Select* o = cluster.map_shared_rank(&s, r < blocks ? r : 0);
      parts[r] = o->part;
      l[r] = 0;
      h[r] = r < blocks ? o->n_keys : 0;
    }
    st = parts[0];
#pragma unroll
    for (int r = 1; r < kMaxSplit; ++r)
      if (r < blocks) stat_merge<X>(st, parts[r], c, 0.f);
    at = k;
    if (tid < mine) {
      const unsigned long long key = s.keys[tid];
      for (int span = 1; span <= k; span *= 2) {                       // loads of all lists first, without branches
        unsigned long long v[kMaxSplit];
#pragma unroll
        for (int r = 0; r < kMaxSplit; ++r)
          v[r] = cluster.map_shared_rank(&s, r < blocks ? r : 0)->keys[(l[r] + h[r]) / 2];
#pragma unroll
        for (int r = 0; r < kMaxSplit; ++r) {
          const int mid = (l[r] + h[r]) / 2;
          const bool more = l[r] < h[r], above = v[r] > key;
          l[r] = more && above ? mid + 1 : l[r];
          h[r] = more && !above ? mid : h[r];
        }
      }
      at = 0;
#pragma unroll
      for (int r = 0; r < kMaxSplit; ++r) at += l[r];
    }
    cluster.sync();                      // nobody reads another block's shared memory any more
  }
  const Row r = finish_row<LT, X>(st, x, a.V, s.stat, c, 0.f);
  if (at < k) {
    const unsigned long long key = s.keys[tid];
    a.ids[static_cast<long long>(row) * k + at] = key_index(key);
    a.top[static_cast<long long>(row) * k + at] = (key_value(key) - r.m) * a.inv_temp - r.ls;
  }
  if (tid == 0 && rank == 0) {
    if (a.target) a.target[row] = given.at >= 0 && given.at < a.V ? (given.value - r.m) * a.inv_temp - r.ls : 0.f;
    if (a.entropy) a.entropy[row] = r.x;
    a.stats[row] = make_float2(r.m, r.ls);
  }
}

// ---- forward: divergence from a teacher's list, cross entropy of a label ---------------------------------
struct DistillArgs {
  const void* logits;
  long long ld;
  int T, V, k;
  double inv_temp;
  int full;                    // 0: both sides normalised over the list, 1: over the vocabulary
  const long long* ids;        // [T, k]; an id outside the vocabulary is an absent entry
  const float* values;         // [T, k]
  const long long* labels;     // [T] or null; a label outside the vocabulary is ignored
  float* kl;                   // [T]
  float* nll;                  // [T] or null
  float* stats;                // [T, kDistillStats]
};

// Per row: m, ln s at temperature 1, ln s at the temperature, the list's teacher mass (full); then for a list that is
// normalised over itself the teacher's maximum and ln sum, the student's maximum and ln sum (+inf: nothing usable).
constexpr int kDistillStats = 8;

// The list of one row, by one warp; writes the row's outputs. ls1, ls2: ln s at temperature 1 and at the temperature.
// A divergence is a sum of differences of log-probabilities that can be much smaller than these: they are formed in 64
// bits, a few operations per entry, where roundings in 32 bits were 2e-6 of the result and more.
template <typename LT>
__device__ __forceinline__ void distill_list(const DistillArgs& a, int row, const LT* x, float m, float ls1,
                                             double ls2) {
  const int lane = threadIdx.x & 31, V = a.V, k = a.k;
  const long long* ids = a.ids + static_cast<long long>(row) * k;
  const float* values = a.values + static_cast<long long>(row) * k;
  float kl = 0.f, mass = 0.f, mt = -FLT_MAX, mx = -FLT_MAX, lt = 0.f, lx = 0.f;
  if (a.full) {
    for (int i = lane; i < k; i += 32) {
      const long long id = ids[i];
      if (id < 0 || id >= V) continue;
      const float t = values[i], q = expf(t);
      mass += q;
      if (q == 0.f) continue;
      kl += q * static_cast<float>(t - ((static_cast<double>(to_f(x[id])) - m) * a.inv_temp - ls2));
    }
    mass = warp_sum_of(mass);
    kl = warp_sum_of(kl);
    if (ls2 == INFINITY) kl = 0.f;
  } else {
    const float c = static_cast<float>(a.inv_temp * kLog2eFine);
    float st = 0.f, sx = 0.f;
    for (int i = lane; i < k; i += 32) {
      const long long id = ids[i];
      if (id < 0 || id >= V) continue;
      mt = fmaxf(mt, values[i]);
      mx = fmaxf(mx, to_f(x[id]));
    }
    mt = warp_max_of(mt);
    mx = warp_max_of(mx);
    for (int i = lane; i < k; i += 32) {
      const long long id = ids[i];
      if (id < 0 || id >= V) continue;
      st += ex2((values[i] - mt) * c);
      sx += ex2((to_f(x[id]) - mx) * c);
    }
    st = warp_sum_of(st);
    sx = warp_sum_of(sx);
    lt = log_sum(st);
    lx = log_sum(sx);
    const bool usable = st > 0.5f && st < INFINITY && sx > 0.5f && sx < INFINITY;      // a maximum alone counts 1
    const double both = usable ? log_fine(sx) - log_fine(st) : static_cast<double>(lx) - lt;
    for (int i = lane; i < k; i += 32) {
      const long long id = ids[i];
      if (id < 0 || id >= V) continue;
      const double t = static_cast<double>(values[i]) - mt, s = static_cast<double>(to_f(x[id])) - mx;
      const float q = expf(static_cast<float>(t * a.inv_temp) - lt);
      if (q == 0.f) continue;
      kl += q * static_cast<float>((t - s) * a.inv_temp + both);
    }
    kl = warp_sum_of(kl);
    if (lt == INFINITY || lx == INFINITY) kl = 0.f;
  }
  if (lane == 0) {
    a.kl[row] = kl;
    if (a.nll) {
      const long long t = a.labels[row];
      a.nll[row] = (t >= 0 && t < V && ls1 != INFINITY) ? ls1 - (to_f(x[t]) - m) : 0.f;
    }
    float4* out = reinterpret_cast<float4*>(a.stats + static_cast<long long>(row) * kDistillStats);
    out[0] = make_float4(m, ls1, static_cast<float>(ls2), mass);
    out[1] = make_float4(mt, lt, mx, lx);
  }
}

// Only the listed entries matter: one warp per row.
template <typename LT>
__global__ void __launch_bounds__(kThreads) distill_list_kernel(DistillArgs a) {
  const int row = blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (row >= a.T) return;
  const LT* x = static_cast<const LT*>(a.logits) + static_cast<long long>(row) * a.ld;
  distill_list(a, row, x, -FLT_MAX, INFINITY, INFINITY);
}

// X: kNone (one softmax sum of the row, scale c1 in the exponent) or kSecond (c1 and c2). One sum is bound by memory
// (4096 x 128256 bf16: 162 us, 6.5 TB/s), two by the exponentials (4096 x 151936 bf16: 266 us, 4.7 TB/s).
template <typename LT, int X>
__global__ void __launch_bounds__(kThreads) distill_fwd_kernel(DistillArgs a, float c1, float c2) {
  __shared__ Stat sh_stat[kWarps];
  __shared__ Stat sh_part;
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int row = blockIdx.x / blocks, tid = threadIdx.x;
  const LT* x = static_cast<const LT*>(a.logits) + static_cast<long long>(row) * a.ld;
  const int2 part = part_of(a.V, rank, blocks);
  const int lo = part.x, hi = part.y;
  Acc<X> acc;
  acc.init(-INFINITY, c1, c2);
  bool fresh = true;
  each_vec(x, lo - misalign(x + lo), lo, hi, [&](int, const uint4 (&u)[kUnroll], int count) {
    const float most = max_vecs<LT>(u, count);
    if (fresh) {                         // begin with the warp's maximum: later ones are rare
      acc.init(warp_max_of(most), c1, c2);
      fresh = false;
    }
    add_vecs<LT, X>(acc, u, count, most, c1, c2);
  });
  Stat st = acc.stat();
  stat_max(st, sh_stat);
  __syncthreads();
  stat_sums<X>(st, sh_stat, c1, c2);
  __syncthreads();
  st = stat_all<X>(st, sh_stat);
  if (blocks > 1) {
    if (tid == 0) sh_part = st;
    cluster.sync();
    if (rank == 0) {
      Stat parts[kMaxSplit];
#pragma unroll
      for (int r = 1; r < kMaxSplit; ++r) parts[r] = *cluster.map_shared_rank(&sh_part, r < blocks ? r : 0);
#pragma unroll
      for (int r = 1; r < kMaxSplit; ++r)
        if (r < blocks) stat_merge<X>(st, parts[r], c1, c2);
    }
    cluster.sync();
    if (rank != 0) return;
  }
  const Row r = finish_row<LT, X>(st, x, a.V, sh_stat, c1, c2);
  // With one sum both logarithms are the same number and only the one that is asked for gets used.
  if (tid < 32) {
    const float rough = X == kSecond ? r.x : r.ls;
    distill_list(a, row, x, r.m, r.ls,
                 r.careful ? rough : (X == kSecond ? log_fine(st.t, st.m, c2) : log_fine(st.s, st.m, c1)));
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
  const float* stats;          // [T, 2] (score: m, ln s) or [T, kDistillStats]
  void* dx;                    // [T, V], dense
  int blocks;                  // a row's columns are cut into this many parts
  int one;                     // both softmaxes are the same: their factors are added
};

// d_j = A p_j (temperature) + B p_j (temperature 1) - G p_j (log p_j + H), then the listed columns get their own
// terms on top: they are computed from the same fp32 value and rounded once, by the thread of the first occurrence.
//
// Bound by memory: 4096 x 151936 bf16 with both temperatures 385 us (6.5 TB/s), 1000 x 262144 bf16 with entropy 163 us
// (6.4 TB/s), soft part alone on 2048 x 151936 fp32 186 us (6.7 TB/s written).
//
// A block has a part of kBwdPart columns: the blocks at work at a time then cover few rows from end to end, which the
// memory takes 4 to 8 % faster than a block per row (4096 x 128256 bf16: 325 us, against 354 us for whole rows and
// 392 us for parts of 8192, whose lists cost more). Without a dense term the gradient was cleared before.
template <typename LT, int DENSE>   // bit 0: temperature, bit 1: temperature 1, bit 2: entropy
__global__ void __launch_bounds__(kThreads) top_bwd_kernel(BwdArgs a) {
  __shared__ __align__(16) int sh_id[kMaxList];
  __shared__ float sh_coef[kMaxList];
  __shared__ float sh_sum[kWarps];
  constexpr int N = kVec<LT>, chunk = kChunk<LT>;
  const int row = blockIdx.x / a.blocks, tid = threadIdx.x;
  const int2 part = part_of(a.V, blockIdx.x - row * a.blocks, a.blocks);
  const int lo = part.x, hi = part.y;
  const LT* x = static_cast<const LT*>(a.logits) + static_cast<long long>(row) * a.ld;
  LT* dx = static_cast<LT*>(a.dx) + static_cast<long long>(row) * a.V;
  const int V = a.V, k = a.k, mode = a.mode;
  const int from = lo - misalign(dx + lo);
  const bool aligned = misalign(x + lo) == misalign(dx + lo);
  uint4 u[kUnroll];
  auto load = [&](int j) {
#pragma unroll
    for (int i = 0; i < kUnroll; ++i)
      if (j + i * chunk < hi) u[i] = load_vec(x, j + i * chunk, lo, hi, aligned);
  };
  const bool ahead = (DENSE == 3 || DENSE == 5) && aligned;
  if (ahead) ask_ahead(x, from + kUnroll * chunk, hi);
  if (DENSE) load(from + tid * N);                 // on their way while the list is looked at
  const float* st = a.stats + static_cast<long long>(row) * (mode == kScore ? 2 : kDistillStats);
  const float m = st[0], ls1 = st[1], lst = mode == kScore ? st[1] : st[2];
  const float c = a.inv_temp * kLog2e;
  // ---- factors of the list
  const long long* ids = a.ids + static_cast<long long>(row) * k;
  const float* values = a.values ? a.values + static_cast<long long>(row) * k : nullptr;
  const float g = a.g_list ? a.g_list[row] : 0.f;
  float mt = 0.f, lt = 0.f, mx = 0.f, lx = 0.f;
  bool live = mode == kScore ? values != nullptr : a.g_list != nullptr;
  if (mode == kListed) {
    mt = st[4]; lt = st[5]; mx = st[6]; lx = st[7];
    live = live && lt != INFINITY && lx != INFINITY;
  } else {
    live = live && lst != INFINITY;
  }
  float sum = 0.f;
  for (int i = tid; i < (k + 3) / 4 * 4; i += kThreads) {
    int at = -1;
    float coef = 0.f;
    if (live && i < k) {
      const long long id = ids[i];
      if (id >= 0 && id < V) {
        at = static_cast<int>(id);
        if (mode == kScore) {
          coef = values[i];
          sum += coef;
        } else if (mode == kFull) {
          coef = -g * expf(values[i]);
        } else {
          const float q = expf((values[i] - mt) * a.inv_temp - lt);
          const float p = expf((to_f(x[id]) - mx) * a.inv_temp - lx);
          coef = g * (p - q);
        }
      }
    }
    sh_id[i] = at;
    if (i < k) sh_coef[i] = coef * a.inv_temp;
  }
  if (mode == kScore) {
    sum = warp_sum_of(sum);
    if ((tid & 31) == 0) sh_sum[tid >> 5] = sum;
  }
  int given = -1;
  float g_given = 0.f;
  if (a.g_given) {
    const long long t = a.given[row];
    if (t >= 0 && t < V && (mode == kScore ? lst : ls1) != INFINITY) {
      given = static_cast<int>(t);
      g_given = a.g_given[row];
    }
  }
  __syncthreads();
  float A = 0.f, B = 0.f, given_coef = 0.f;
  if (mode == kScore) {
    A = 0.f;
    for (int w = 0; w < kWarps; ++w) A += sh_sum[w];
    A = -(A + g_given) * a.inv_temp;
    given_coef = g_given * a.inv_temp;
  } else {
    if (mode == kFull && live) A = g * a.inv_temp * st[3];
    if (a.one) A += g_given; else B = g_given;
    given_coef = -g_given;
  }
  const float lst2 = lst * kLog2e, ls12 = ls1 * kLog2e;
  float G = 0.f;
  if (DENSE & 4) {
    const float ge = a.g_entropy[row] * a.inv_temp;
    G = -ge * kLn2;                                // p (A - ge (log p + H)) = p (A - ge H + G log2 p)
    A -= ge * a.entropy[row];
  }
  const f32x2 mm = pack2(-m, -m), cc = pack2(c, c), ll = pack2(-lst2, -lst2), AA = pack2(A, A), GG = pack2(G, G);
  const f32x2 cc1 = pack2(kLog2e, kLog2e), ll1 = pack2(-ls12, -ls12), BB = pack2(B, B);
  auto dense2 = [&](f32x2 v) -> f32x2 {
    const f32x2 d = add2(v, mm);
    f32x2 r = 0;
    if (DENSE & 5) {
      const float2 e = unpack2(fma2(d, cc, ll));
      const f32x2 p = pack2(ex2(e.x), ex2(e.y));
      if (DENSE & 4)
        // below 2^-126 p is 0: the exponent is bounded there, or its product with G could leave fp32 and 0 * inf is NaN
        r = mul2(p, fma2(GG, pack2(fmaxf(e.x, -200.f), fmaxf(e.y, -200.f)), AA));
      else
        r = mul2(p, AA);
    }
    if (DENSE & 2) {
      const float2 e = unpack2(fma2(d, cc1, ll1));
      r = fma2(pack2(ex2(e.x), ex2(e.y)), BB, r);
    }
    return r;
  };
  // ---- the whole part
  if (DENSE) {
    for (int at = from; at < hi; at += kUnroll * chunk) {
      const int j = at + tid * N;
      if (ahead && at != from) ask_ahead(x, at + kUnroll * chunk, hi);
      if (at != from) load(j);
#pragma unroll
      for (int i = 0; i < kUnroll; ++i) {
        const int ji = j + i * chunk;
        if (ji >= hi) break;
        float z[N];
        unpack(u[i], z);
#pragma unroll
        for (int e = 0; e < N; e += 2) {
          const float2 r = unpack2(dense2(pack2(z[e], z[e + 1])));
          z[e] = r.x;
          z[e + 1] = r.y;
        }
        store_vec(dx, ji, lo, hi, z);
      }
    }
  }
  __syncthreads();
  // ---- the listed columns of the part
  auto put = [&](int at, float extra) {
    const float v = DENSE ? to_f(x[at]) : 0.f;
    from_f((DENSE ? unpack2(dense2(pack2(v, v))).x : 0.f) + extra, dx + at);
  };
  for (int i = tid; i < k; i += kThreads) {
    const int at = sh_id[i];
    if (at < lo || at >= hi) continue;
    int same = 0;
    for (int n = 0; n < k; n += 4) {
      const int4 o = *reinterpret_cast<const int4*>(sh_id + n);
      same += (o.x == at) + (o.y == at) + (o.z == at) + (o.w == at);
    }
    float extra = sh_coef[i];
    bool mine = true;
    if (same > 1) {                                // a column that is listed more than once
      extra = 0.f;
      for (int n = 0; n < k; ++n) {
        if (sh_id[n] != at) continue;
        if (n < i) mine = false;
        extra += sh_coef[n];
      }
    }
    if (mine) put(at, extra + (at == given ? given_coef : 0.f));
  }
  if (given >= lo && given < hi) {
    int listed = 0;
    for (int i = tid; i < k; i += kThreads) listed |= sh_id[i] == given;
    listed = __syncthreads_or(listed);             // `given` is the same in all threads
    if (tid == 0 && !listed) put(given, given_coef);
  }
}

// Blocks per row of a forward pass: up to kMaxSplit while all of them are at most three per SM and each has `least`
// bytes of the row. Measured on rows of 151936 bf16 with k = 20 (us with 1, 2, 4, 8 blocks): one row 16.5, 13.5, 10.6,
// 10.4; 32 rows 17.2, 13.6, 11.2, 12.4; 64 rows 17.3, 13.8, 13.0, 15.9; 148 rows 17.7, 16.5, 19.1, 20.9; 200 rows 21.7,
// 19.8, 19.9, 20.9; rows of 32000: 64 rows 8.7, 9.4, 9.1, 10.5. Without a selection less is enough (one row 12.3, 9.3,
// 6.8, 5.9).
int split_of(int T, long long bytes, int least) {
  int n = 1;
  while (n < kMaxSplit && 2ll * n * T <= 3ll * txh::sm_count() && bytes / (2 * n) >= least) n *= 2;
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

// n bytes (a multiple of 2) from a 16-byte boundary. Blocks of 16 KB that end at once: 7.4 TB/s, where 1184 blocks that
// loop over the same tiles write 6.1 TB/s (1.24 GB).
constexpr int kClearThreads = 512, kClearVecs = 2;
__global__ void __launch_bounds__(kClearThreads) clear_kernel(unsigned char* p, long long n) {
  const long long at = blockIdx.x * static_cast<long long>(kClearThreads * kClearVecs) + threadIdx.x;
#pragma unroll
  for (int i = 0; i < kClearVecs; ++i) {
    const long long byte = (at + i * kClearThreads) * 16;
    if (byte + 16 <= n) {
      *reinterpret_cast<uint4*>(p + byte) = make_uint4(0, 0, 0, 0);
    } else {
      for (long long b = byte; b < n; b += 2) *reinterpret_cast<uint16_t*>(p + b) = 0;
    }
  }
}

template <typename LT>
int launch_bwd(BwdArgs a, int dense, cudaStream_t s) {
  // few rows: more and smaller parts, so that every SM has some
  const int want = 8 * txh::sm_count(), most = (a.V + kMinPart - 1) / kMinPart;
  a.blocks = max((a.V + kBwdPart - 1) / kBwdPart, min(most, (want + a.T - 1) / a.T));
  if (dense == 0) {
    a.blocks = 1;
    const long long bytes = static_cast<long long>(sizeof(LT)) * a.T * a.V, tile = 16 * kClearThreads * kClearVecs;
    clear_kernel<<<static_cast<unsigned>((bytes + tile - 1) / tile), kClearThreads, 0, s>>>(
        static_cast<unsigned char*>(a.dx), bytes);
  }
#define TX_BWD(D) case D: top_bwd_kernel<LT, D><<<a.T * a.blocks, kThreads, 0, s>>>(a); break
  switch (dense) {
    TX_BWD(0); TX_BWD(1); TX_BWD(2); TX_BWD(3); TX_BWD(5);
    default: return 2;
  }
#undef TX_BWD
  return cudaGetLastError() == cudaSuccess ? 0 : 400;
}

}  // namespace

// logits [T, V] with row stride ld (elements), fp32 or bf16; 1 <= k <= min(V, 256).
extern "C" int tx_top_logprob_fwd(const void* logits, int logits_fp32, long long ld, int T, int V, int k,
                                  float inv_temp, const long long* targets, long long* ids, float* top, float* target,
                                  float* entropy, float* stats, cudaStream_t s) {
  if (T <= 0) return 0;
  if (V < 1 || k < 1 || k > kMaxTop || k > V || V > 0x7fff0000) return 1;
  const TopArgs a{logits, ld, T, V, k, inv_temp, targets, ids, top, target, entropy, reinterpret_cast<float2*>(stats)};
  const int n = split_of(T, V * (logits_fp32 ? 4ll : 2ll), 65536);
  const int bytes = sizeof(Select);
  if (logits_fp32)
    return entropy ? launch_rows<top_fwd_kernel<float, kEntropy>>(T, n, bytes, s, a)
                   : launch_rows<top_fwd_kernel<float, kNone>>(T, n, bytes, s, a);
  return entropy ? launch_rows<top_fwd_kernel<__nv_bfloat16, kEntropy>>(T, n, bytes, s, a)
                 : launch_rows<top_fwd_kernel<__nv_bfloat16, kNone>>(T, n, bytes, s, a);
}

// 1 <= k <= 1024; stats [T, 8].
extern "C" int tx_top_distill_fwd(const void* logits, int logits_fp32, long long ld, int T, int V, int k,
                                  double inv_temp, int full, const long long* ids, const float* values,
                                  const long long* labels, float* kl, float* nll, float* stats, cudaStream_t s) {
  if (T <= 0) return 0;
  if (V < 1 || k < 1 || k > kMaxList || V > 0x7fff0000) return 1;
  const DistillArgs a{logits, ld, T, V, k, inv_temp, full, ids, values, labels, kl, nll, stats};
  const float c = static_cast<float>(inv_temp * kLog2eFine), c1 = nll ? kLog2e : c;
  const int n = split_of(T, V * (logits_fp32 ? 4ll : 2ll), 32768);
  if (!nll && !full) {
    const int grid = (T + kWarps - 1) / kWarps;
    if (logits_fp32) distill_list_kernel<float><<<grid, kThreads, 0, s>>>(a);
    else             distill_list_kernel<__nv_bfloat16><<<grid, kThreads, 0, s>>>(a);
    return cudaGetLastError() == cudaSuccess ? 0 : 400;
  }
  if (nll && full && inv_temp != 1.0)
    return logits_fp32 ? launch_rows<distill_fwd_kernel<float, kSecond>>(T, n, 0, s, a, c1, c)
                       : launch_rows<distill_fwd_kernel<__nv_bfloat16, kSecond>>(T, n, 0, s, a, c1, c);
  return logits_fp32 ? launch_rows<distill_fwd_kernel<float, kNone>>(T, n, 0, s, a, c1, c)
                     : launch_rows<distill_fwd_kernel<__nv_bfloat16, kNone>>(T, n, 0, s, a, c1, c);
}

// Gradient of tx_top_logprob_fwd: g_top or null, g_target with targets or null, g_entropy with entropy or null. dx is
// [T, V], dense, from a 16-byte boundary.
extern "C" int tx_top_logprob_bwd(const void* logits, int logits_fp32, long long ld, int T, int V, int k,
                                  float inv_temp, const long long* ids, const float* g_top, const long long* targets,
                                  const float* g_target, const float* g_entropy, const float* entropy,
                                  const float* stats, void* dx, cudaStream_t s) {
  if (T <= 0) return 0;
  if (V < 1 || k < 1 || k > kMaxTop || V > 0x7fff0000) return 1;
  const BwdArgs a{logits, ld, T, V, k, kScore, inv_temp, ids, g_top, targets, nullptr, g_target, g_entropy, entropy,
                  stats, dx, 1, 0};
  const int dense = g_entropy ? 5 : 1;
  return logits_fp32 ? launch_bwd<float>(a, dense, s) : launch_bwd<__nv_bfloat16>(a, dense, s);
}

// Gradient of tx_top_distill_fwd; g_kl or g_nll may be null. dx as above.
extern "C" int tx_top_distill_bwd(const void* logits, int logits_fp32, long long ld, int T, int V, int k,
                                  float inv_temp, int full, const long long* ids, const float* values,
                                  const long long* labels, const float* g_kl, const float* g_nll, const float* stats,
                                  void* dx, cudaStream_t s) {
  if (T <= 0) return 0;
  if (V < 1 || k < 1 || k > kMaxList || V > 0x7fff0000) return 1;
  const int both = full && g_kl && g_nll && inv_temp == 1.f;
  const BwdArgs a{logits, ld, T, V, k, full ? kFull : kListed, inv_temp, ids, values, labels, g_kl, g_nll, nullptr,
                  nullptr, stats, dx, 1, both};
  const int dense = (full && g_kl ? 1 : 0) | (g_nll && !both ? 2 : 0);
  return logits_fp32 ? launch_bwd<float>(a, dense, s) : launch_bwd<__nv_bfloat16>(a, dense, s);
}
