// Device helpers shared by the kernels that read a language model's logits (token_logprobs.cu,
// distill_topk.cu): element access, the running softmax state of a row and the order of a row's
// top list.
//
// With c = log2(e) / temperature and a base m near the row's largest logit, a part of a row is
// summed as
//   s = sum 2^(c (x - m)),   a = sum 2^(c (x - m)) c (x - m)
// so that the row's log normaliser is  m / temperature + ln s  and its entropy  ln s - ln2 a / s.
// Exponents are clamped at -200, where 2^t is already 0 in fp32, so that a masked (-inf) element adds
// 0 to both sums, not -inf * 0. Maxima are the NaN-propagating ones: a NaN logit ends up in every
// result of its row.
//
// The inner loops take c x - b with a whole number b near c m: one fused multiply-add, exact but for
// its last rounding (c m itself would be rounded, by 2^-24 |c m| for the whole sum), and rescaling by
// powers of two. Where |c m| is past kWide that has no digits left, or overflows (a row filled with
// the type's lowest value as a mask): such rows take the differences x - m before the scaling.
#pragma once

#include <cstdint>
#include <type_traits>

#include "bdh_sm100.h"
#include "common.cuh"
#include "internal.h"

namespace bdh {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kExpFloor = -200.0f;
constexpr int kTopMax = BDH_TOP_MAX;  // entries of a top list

__device__ __forceinline__ float neg_inf() { return __uint_as_float(0xff800000u); }
__device__ __forceinline__ float quiet_nan() { return __uint_as_float(0x7fc00000u); }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// One instruction on sm_100.
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float y;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}

template <typename T>
__device__ __forceinline__ float logit_at(const T* p, int64_t i);
template <>
__device__ __forceinline__ float logit_at<float>(const float* p, int64_t i) {
  return p[i];
}
template <>
__device__ __forceinline__ float logit_at<uint16_t>(const uint16_t* p, int64_t i) {
  return __uint_as_float(static_cast<uint32_t>(p[i]) << 16);
}
__device__ __forceinline__ void logit_put(float* p, int64_t i, float v) { p[i] = v; }
__device__ __forceinline__ void logit_put(uint16_t* p, int64_t i, float v) {
  p[i] = static_cast<uint16_t>(f32_to_bf16_bits(v));
}

// ------------------------------------------------------------------------ vectors ----
// A row is read as 16-byte vectors of kVec<T> elements between its first and last 16-byte
// boundary, and element by element before and after them (rows start at any element, so the
// vectors of two rows may lie differently). Nothing outside the row is read.
template <typename T>
constexpr int kVec = 16 / static_cast<int>(sizeof(T));

struct RowSpan {
  int head, vecs, tail;  // elements, vectors, elements
};
template <typename T>
__device__ __forceinline__ RowSpan row_span(const T* p, int n) {
  RowSpan r;
  r.head = static_cast<int>(((16u - (reinterpret_cast<uintptr_t>(p) & 15u)) & 15u) / sizeof(T));
  if (r.head > n) r.head = n;
  r.vecs = (n - r.head) / kVec<T>;
  r.tail = n - r.head - r.vecs * kVec<T>;
  return r;
}

// The elements of a 16-byte vector as fp32.
__device__ __forceinline__ void unpack(const uint4& u, float (&x)[4]) {
  x[0] = __uint_as_float(u.x);
  x[1] = __uint_as_float(u.y);
  x[2] = __uint_as_float(u.z);
  x[3] = __uint_as_float(u.w);
}
__device__ __forceinline__ void unpack(const uint4& u, float (&x)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = bf16x2_lo(w[i]);
    x[2 * i + 1] = bf16x2_hi(w[i]);
  }
}
// The other way, and to a 16-byte aligned place.
__device__ __forceinline__ uint4 pack(const float (&x)[4]) {
  return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]),
                    __float_as_uint(x[3]));
}
__device__ __forceinline__ uint4 pack(const float (&x)[8]) {
  return make_uint4(cvt_bf16x2(x[0], x[1]), cvt_bf16x2(x[2], x[3]), cvt_bf16x2(x[4], x[5]),
                    cvt_bf16x2(x[6], x[7]));
}
template <typename T, int N>
__device__ __forceinline__ void store_vec(T* p, const float (&x)[N]) {
  *reinterpret_cast<uint4*>(p) = pack(x);
}
// The largest element of N vectors (bf16 in pairs, where one instruction compares two).
template <int N>
__device__ __forceinline__ float max_of(const uint4 (&w)[N], float) {
  float m = neg_inf();
#pragma unroll
  for (int u = 0; u < N; ++u) {
    float x[4];
    unpack(w[u], x);
    m = max_nan(max_nan(m, x[0], x[1]), x[2], x[3]);
  }
  return m;
}
__device__ __forceinline__ uint32_t max_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <int N>
__device__ __forceinline__ float max_of(const uint4 (&w)[N], uint16_t) {
  uint32_t m = 0xff80ff80u;
#pragma unroll
  for (int u = 0; u < N; ++u)
    m = max_bf16x2(m, max_bf16x2(max_bf16x2(w[u].x, w[u].y), max_bf16x2(w[u].z, w[u].w)));
  return max_nan(bf16x2_lo(m), bf16x2_hi(m));
}
// A vector with what is below `least` raised to it. An entropy's sum multiplies an element's exponential by
// its exponent, so that a masked one must not have an infinite exponent: -2 kWide / c (from the host, in the
// logits' type, bf16 twice) has an exponential of 0 beside every base, which is above -kWide, and -2 kWide as
// its exponent, at every temperature.
__device__ __forceinline__ uint4 at_least(const uint4& w, float, uint32_t least) {
  const float to = __uint_as_float(least);
  return make_uint4(__float_as_uint(max_nan(__uint_as_float(w.x), to)),
                    __float_as_uint(max_nan(__uint_as_float(w.y), to)),
                    __float_as_uint(max_nan(__uint_as_float(w.z), to)),
                    __float_as_uint(max_nan(__uint_as_float(w.w), to)));
}
__device__ __forceinline__ uint4 at_least(const uint4& w, uint16_t, uint32_t least) {
  return make_uint4(max_bf16x2(w.x, least), max_bf16x2(w.y, least), max_bf16x2(w.z, least),
                    max_bf16x2(w.w, least));
}
// A vector of -inf: what a place past the end of a row counts as.
template <typename T>
__device__ __forceinline__ uint4 void_vec();
template <>
__device__ __forceinline__ uint4 void_vec<float>() {
  return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u);
}
template <>
__device__ __forceinline__ uint4 void_vec<uint16_t>() {
  return make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u);
}

constexpr int kUnroll = 4;  // vectors that a thread has in flight (a batch)

// How many of a batch's vectors b + u G + tid this warp has any of.
template <int G>
__device__ __forceinline__ int batch_fill(int b, int v1, int tid) {
  return (v1 - b - (tid & ~31) + G - 1) / G;  // may be more than there are
}
// A group of G threads over the vectors [v0, v1): f(w, b, fill, refill) for every batch w of its kUnroll
// vectors b + u G + tid (-inf past the end). f calls refill(u) as soon as it has taken vector u out of
// its register, so that the next batch's loads are under way while this one is worked on, without
// registers of their own. `w` is asked for by the caller (load_batch) as early as it can. While this
// batch and the next are whole (fill: the constant kUnroll), nothing is checked per vector.
template <typename T, int G>
__device__ __forceinline__ void load_batch(uint4 (&w)[kUnroll], const uint4* vec, int b, int v1, int tid) {
#pragma unroll
  for (int u = 0; u < kUnroll; ++u)
    if (b < v1) w[u] = __ldg(vec + min(b + u * G + tid, v1 - 1));  // (a vector past the end: any inside)
}
template <typename T, int G, typename F>
__device__ __forceinline__ void stream(uint4 (&w)[kUnroll], const uint4* vec, int v0, int v1, int tid, F f) {
  constexpr int kStep = G * kUnroll;
  int b = v0;
  const uint4* next = vec + v0 + kStep + tid;
  for (; b + 2 * kStep <= v1; b += kStep, next += kStep)
    f(w, b, std::integral_constant<int, kUnroll>(), [&](int u) { w[u] = __ldg(next + u * G); });
  for (; b < v1; b += kStep) {
    if (b + kStep > v1) {
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (b + u * G + tid >= v1) w[u] = void_vec<T>();
    }
    f(w, b, batch_fill<G>(b, v1, tid),
      [&](int u) { w[u] = __ldg(vec + min(b + kStep + u * G + tid, v1 - 1)); });
  }
}

// The same for a slice that is read twice: with an L2 cache policy on its loads, and with the next batch
// in registers of its own, asked for before this one is looked at, which costs the copies but has the
// loads under way longer (f's refill does nothing).
__device__ __forceinline__ uint4 ld_vec(const uint4* p, uint64_t policy) {
  uint4 r;
  asm volatile("ld.global.nc.L2::cache_hint.v4.u32 {%0, %1, %2, %3}, [%4], %5;"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p), "l"(policy));
  return r;
}
template <int G>
__device__ __forceinline__ void load_batch(uint4 (&w)[kUnroll], const uint4* vec, int b, int v1, int tid,
                                           uint64_t policy) {
#pragma unroll
  for (int u = 0; u < kUnroll; ++u)
    if (b < v1) w[u] = ld_vec(vec + min(b + u * G + tid, v1 - 1), policy);
}
template <typename T, int G, typename F>
__device__ __forceinline__ void stream_early(uint4 (&next)[kUnroll], const uint4* vec, int v0, int v1, int tid,
                                             uint64_t policy, F f) {
  constexpr int kStep = G * kUnroll;
  for (int b = v0; b < v1; b += kStep) {
    uint4 w[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) w[u] = next[u];
    load_batch<G>(next, vec, b + kStep, v1, tid, policy);
    if (b + kStep > v1) {
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (b + u * G + tid >= v1) w[u] = void_vec<T>();
    }
    f(w, b, batch_fill<G>(b, v1, tid), [](int) {});
  }
}

// d[i] = f(x[i]) for n elements by a group of G threads, or zeros without reading. Vectors where x and
// d lie alike; else vectors are read and elements written.
template <typename T, int G, typename F>
__device__ __forceinline__ void map_row(const T* x, T* d, int n, int tid, bool zero, F f) {
  constexpr int kV = kVec<T>;
  const RowSpan span = row_span(x, n);
  const bool aligned = (reinterpret_cast<uintptr_t>(d + span.head) & 15u) == 0;
  const uint4* vec = reinterpret_cast<const uint4*>(x + span.head);
  T* out = d + span.head;
  for (int e = tid; e < span.head + span.tail; e += G) {
    const int at = e < span.head ? e : n - span.tail + (e - span.head);
    logit_put(d, at, zero ? 0.0f : f(logit_at<T>(x, at)));
  }
  for (int b = 0; b < span.vecs; b += G * kUnroll) {
    uint4 w[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int v = b + u * G + tid;
      if (v < span.vecs && !zero) w[u] = __ldg(vec + v);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int v = b + u * G + tid;
      if (v >= span.vecs) break;
      float xs[kV], ds[kV];
      if (zero) {
#pragma unroll
        for (int e = 0; e < kV; ++e) ds[e] = 0.0f;
      } else {
        unpack(w[u], xs);
#pragma unroll
        for (int e = 0; e < kV; ++e) ds[e] = f(xs[e]);
      }
      if (aligned) {
        store_vec(out + static_cast<int64_t>(v) * kV, ds);
      } else {
#pragma unroll
        for (int e = 0; e < kV; ++e) logit_put(out, static_cast<int64_t>(v) * kV + e, ds[e]);
      }
    }
  }
}

// Softmax state of a part of a row: maximum, sum, and exponent-weighted sum (see above).
struct SoftState {
  float m, s, a;
};  // m: a value of the row, -inf for none above it
__device__ __forceinline__ SoftState soft_empty() { return {neg_inf(), 0.0f, 0.0f}; }
__device__ __forceinline__ void soft_add(SoftState& st, float x, float c) {
  const float m = max_nan(st.m, x);
  if (m != st.m) {  // also when it becomes NaN
    const float d = max_nan((st.m - m) * c, kExpFloor);
    const float f = ex2(d);
    st.a = f * fmaf(d, st.s, st.a);
    st.s *= f;
    st.m = m;
  }
  if (m == neg_inf()) return;
  const float t = max_nan((x - m) * c, kExpFloor);
  const float e = ex2(t);
  st.s += e;
  st.a = fmaf(e, t, st.a);
}
__device__ __forceinline__ SoftState soft_merge(const SoftState& x, const SoftState& y, float c) {
  const float m = max_nan(x.m, y.m);
  if (m == neg_inf()) return soft_empty();
  const float dx = max_nan((x.m - m) * c, kExpFloor), dy = max_nan((y.m - m) * c, kExpFloor);
  const float fx = ex2(dx), fy = ex2(dy);
  return {m, fmaf(x.s, fx, y.s * fy), fmaf(fx, fmaf(dx, x.s, x.a), fy * fmaf(dy, y.s, y.a))};
}
// Raise the state's base to m (not below it; NaN stays).
__device__ __forceinline__ void soft_raise(SoftState& st, float m, float c) {
  const float d = max_nan((st.m - m) * c, kExpFloor);
  const float f = ex2(d);
  st.a = f * fmaf(d, st.s, st.a);
  st.s *= f;
  st.m = m;
}

// 2^n for a whole n <= 0.
__device__ __forceinline__ float pow2(float n) {
  return n < -126.0f ? 0.0f : __int_as_float((static_cast<int>(n) + 127) << 23);
}
// A thread's running sums over vectors. The base may be below the largest element so far by up to
// kBaseSlack in the exponent (terms stay below 2^kBaseSlack), so that the sums are rescaled a few
// times a row and not whenever a new maximum comes. A thread that meets a base it cannot use stops
// and says so (`wide`); its part is then summed with soft_add.
constexpr float kBaseSlack = 8.0f;
template <bool ENTROPY>
struct SoftSums {
  float m = neg_inf(), limit = neg_inf(), base = 0.0f;  // the base's element, the largest it serves
  float s[2] = {0.0f, 0.0f}, a[2] = {0.0f, 0.0f};
  bool wide = false;
  __device__ __forceinline__ void raise(float largest, float c, float slack) {
    const float b = largest * c;
    if (!(fabsf(b) < kWide)) {  // NaN too
      wide = true;
      return;
    }
    const float to = rintf(b);
    if (m != neg_inf()) {
      const float d = base - to, f = pow2(d);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (ENTROPY) a[i] = f * fmaf(max_nan(d, kExpFloor), s[i], a[i]);
        s[i] *= f;
      }
    }
    base = to;
    m = largest;
    limit = largest + slack;
  }
  // N vectors whose largest element is `largest`; of a row's last ones, `fill` of them. `least`: see
  // at_least. taken(u): vector u is out of its register.
  template <typename T, int N, typename Fill, typename Taken>
  __device__ __forceinline__ void add(const uint4 (&w)[N], float largest, float c, float slack, uint32_t least,
                                      Fill fill, Taken taken) {
    if (!(largest <= limit)) raise(largest, c, slack);  // a NaN too
    const bool sum = !wide && m != neg_inf();
    float ps[2] = {0.0f, 0.0f}, pa[2] = {0.0f, 0.0f};  // (a batch's own sums: fewer terms in a row)
#pragma unroll
    for (int u = 0; u < N; ++u) {
      float x[kVec<T>];
      unpack(ENTROPY ? at_least(w[u], T(), least) : w[u], x);
      taken(u);
      if (u > 0 && u >= fill) continue;
#pragma unroll
      for (int i = 0; i < kVec<T>; ++i) {
        const float t = fmaf(x[i], c, -base), e = ex2(t);
        ps[i % 2] += e;
        if (ENTROPY) pa[i % 2] = fmaf(e, t, pa[i % 2]);
      }
    }
    if (!sum) return;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      s[i] += ps[i];
      if (ENTROPY) a[i] += pa[i];
    }
  }
  __device__ __forceinline__ SoftState state(float c) const {
    if (m == neg_inf()) return soft_empty();
    const float t = fmaf(m, c, -base), f = ex2(-t), sum = s[0] + s[1];
    return {m, sum * f, ENTROPY ? f * fmaf(-t, sum, a[0] + a[1]) : 0.0f};
  }
};
// The same for a thread's part of the vectors [v0, v1) where it was too wide.
template <typename T, int G>
__device__ __forceinline__ SoftState soft_slowly(const uint4* vec, int v0, int v1, int tid, float c) {
  SoftState st = soft_empty();
  const T* x = reinterpret_cast<const T*>(vec);
#pragma unroll 1
  for (int v = v0 + tid; v < v1; v += G)
#pragma unroll 1
    for (int e = 0; e < kVec<T>; ++e) soft_add(st, logit_at<T>(x, static_cast<int64_t>(v) * kVec<T> + e), c);
  return st;
}

// An element's exponential times what the row has for all: p (k0 + k1 log2 p) with
// log2 p = c (x - m) - l2, for a row's base m and log2 sum l2. As 2^t (K0 + K1 t) with t = c x - b.
struct RowMap {
  float c, b, k0, k1;
  float m, l2, w0, w1;  // the plain form, for a wide row
  bool wide, with_log;
  __device__ __forceinline__ RowMap(float c_, float m_, float l2_, float w0_, float w1_)
      : c(c_), m(m_), l2(l2_), w0(w0_), w1(w1_) {
    wide = !(fabsf(m * c) < kWide);
    with_log = w1 != 0.0f;  // NaN counts
    b = rintf(m * c);
    const float shift = -fmaf(m, c, -b) - l2, f = exp2f(shift);
    k0 = fmaf(w1, shift, w0) * f;
    k1 = w1 * f;
  }
  __device__ __forceinline__ float plain(float x) const {
    const float y = fmaf(x - m, c, -l2);
    return ex2(y) * (with_log ? fmaf(w1, max_nan(y, kExpFloor), w0) : w0);
  }
  __device__ __forceinline__ float of(float x) const { return wide ? plain(x) : (*this)(x); }
  __device__ __forceinline__ float operator()(float x) const {
    const float t = fmaf(x, c, -b);
    return ex2(t) * (with_log ? fmaf(k1, max_nan(t, kExpFloor), k0) : k0);
  }
};
template <int G>
__device__ __forceinline__ float row_map(const RowMap& map, float x) {
  return G <= 32 ? map.plain(x) : map.of(x);
}
// d = map(x) for n elements of a row by a group of G threads. A warp's rows are short and do not wait
// for arithmetic: the plain form, in which a single token's probability is exactly 1.
template <typename T, int G>
__device__ __forceinline__ void map_row(const T* x, T* d, int n, int tid, bool zero, const RowMap& map) {
  if (G <= 32) {
    map_row<T, G>(x, d, n, tid, zero, [&](float v) { return map.plain(v); });
  } else if (map.wide && !zero) {
#pragma unroll 1
    for (int e = tid; e < n; e += G) logit_put(d, e, map.of(logit_at<T>(x, e)));
  } else if (map.with_log) {
    map_row<T, G>(x, d, n, tid, zero, [&](float v) {
      const float t = fmaf(v, map.c, -map.b);
      return ex2(t) * fmaf(map.k1, max_nan(t, kExpFloor), map.k0);
    });
  } else {
    map_row<T, G>(x, d, n, tid, zero, [&](float v) { return ex2(fmaf(v, map.c, -map.b)) * map.k0; });
  }
}

// Over the warp, or over each L neighbouring lanes of it (all lanes take part).
template <int L = 32>
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int d = L / 2; d > 0; d >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, d));
  return v;
}
template <int L = 32>
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = L / 2; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}
// The lanes' states as one.
__device__ __forceinline__ SoftState soft_join(SoftState st, float c) {
  const float m = warp_max(st.m);
  if (m == neg_inf()) return soft_empty();
  soft_raise(st, m, c);
  st.s = warp_sum(st.s);
  st.a = warp_sum(st.a);
  return st;
}
// Softmax state of a row that L lanes hold N elements each of: the maximum first, then the sums.
template <bool ENTROPY, int L, int N>
__device__ __forceinline__ SoftState soft_of_lanes(const float (&x)[N], float c) {
  float m = x[0];
#pragma unroll
  for (int i = 1; i + 1 < N; i += 2) m = max_nan(m, x[i], x[i + 1]);
  if (N % 2 == 0) m = max_nan(m, x[N - 1]);
  m = warp_max<L>(m);
  const float from = m == neg_inf() ? 0.0f : m;  // (all lanes go on: other lanes' rows may have more)
  float s = 0.0f, a = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float t = max_nan((x[i] - from) * c, kExpFloor), e = ex2(t);
    s += e;
    if (ENTROPY) a = fmaf(e, t, a);
  }
  return {m, warp_sum<L>(s), ENTROPY ? warp_sum<L>(a) : 0.0f};
}

// Order of a row's top list: larger values first, an equal value's lower index first; -0 equals
// +0, and NaN comes before everything (as torch.sort places it). Larger key, earlier place;
// key 0 stands for "no element" and is below every element's, ~0 is above.
__device__ __forceinline__ uint32_t value_key(float x) {
  if (x != x) return 0xff800001u;  // one above +inf's
  const uint32_t b = __float_as_uint(x + 0.0f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);  // NaN comes back as one
}
__device__ __forceinline__ uint64_t top_key(float x, uint32_t i) {
  return (static_cast<uint64_t>(value_key(x)) << 32) | (0xffffffffu - i);
}
__device__ __forceinline__ uint32_t key_index(uint64_t k) {
  return 0xffffffffu - static_cast<uint32_t>(k);
}

// ------------------------------------------------------------------------ clusters ----
__device__ __forceinline__ uint32_t cta_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// Address of the local shared variable at `p` in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t peer_smem(const void* p, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ void peer_store(uint32_t addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}
__device__ __forceinline__ void peer_store(uint32_t addr, uint64_t v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}
__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}

}  // namespace bdh
