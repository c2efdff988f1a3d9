// Device helpers shared by the kernels that read a language model's logits (token_logprobs.cu,
// distill_topk.cu): element access, the running softmax state of a row and the order of a row's
// top list.
//
// With c = log2(e) / temperature and the row's running maximum m (of the raw logits), a part of
// a row is summed as
//   s = sum 2^(c (x - m)),   a = sum 2^(c (x - m)) c (x - m)
// so that the row's log normaliser is  m / temperature + ln s  and its entropy  ln s - ln2 a / s.
// Differences x - m are formed before the scaling: a row filled with the type's lowest value (a
// mask) then gives zeros, where c x - c m would overflow. Exponents are clamped at -200, where
// 2^t is already 0 in fp32, so that a masked (-inf) element adds 0 to both sums, not -inf * 0.
// Maxima are the NaN-propagating ones: a NaN logit ends up in every result of its row.
#pragma once

#include <cstdint>

#include "bdh_sm100.h"
#include "common.cuh"

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

// Two fp32 in a register pair: sm_100's packed arithmetic does both with one instruction, each
// rounded as its scalar form.
struct F2 {
  uint64_t v;
};
__device__ __forceinline__ F2 f2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void f2_split(const F2& x, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x.v));
}
__device__ __forceinline__ F2 f2_add(const F2& a, const F2& b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 f2_mul(const F2& a, const F2& b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 f2_fma(const F2& a, const F2& b, const F2& c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
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
// The other way, to a 16-byte aligned place.
__device__ __forceinline__ void store_vec(float* p, const float (&x)[4]) {
  *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
}
__device__ __forceinline__ void store_vec(uint16_t* p, const float (&x)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(cvt_bf16x2(x[0], x[1]), cvt_bf16x2(x[2], x[3]),
                                            cvt_bf16x2(x[4], x[5]), cvt_bf16x2(x[6], x[7]));
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

// d[i] = f(x[i]) for n elements by a group of G threads: `pair` on two elements, `single` on one,
// or zeros. Vectors where x and d lie alike; else vectors are read and elements written.
template <typename T, int G, typename Single, typename Pair>
__device__ __forceinline__ void map_row(const T* x, T* d, int n, int tid, bool zero, Single single,
                                        Pair pair) {
  constexpr int kV = kVec<T>;
  const RowSpan span = row_span(x, n);
  const bool aligned = (reinterpret_cast<uintptr_t>(d + span.head) & 15u) == 0;
  const uint4* vec = reinterpret_cast<const uint4*>(x + span.head);
  T* out = d + span.head;
  for (int e = tid; e < span.head + span.tail; e += G) {
    const int at = e < span.head ? e : n - span.tail + (e - span.head);
    logit_put(d, at, zero ? 0.0f : single(logit_at<T>(x, at)));
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
        for (int e = 0; e < kV; e += 2) pair(xs[e], xs[e + 1], ds[e], ds[e + 1]);
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
};
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
// Raise the state's maximum to m (not below it; NaN stays).
__device__ __forceinline__ void soft_raise(SoftState& st, float m, float c) {
  const float d = max_nan((st.m - m) * c, kExpFloor);
  const float f = ex2(d);
  st.a = f * fmaf(d, st.s, st.a);
  st.s *= f;
  st.m = m;
}
// Add N elements none of which is above the state's maximum, which is not -inf.
template <bool ENTROPY, int N>
__device__ __forceinline__ void soft_sum(SoftState& st, const float (&x)[N], float c) {
  const F2 nm = f2(-st.m, -st.m), cc = f2(c, c);
  F2 s = f2(0.0f, 0.0f), a = f2(0.0f, 0.0f);
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    float t0, t1;
    f2_split(f2_mul(f2_add(f2(x[i], x[i + 1]), nm), cc), t0, t1);
    if (ENTROPY) {
      t0 = max_nan(t0, kExpFloor);
      t1 = max_nan(t1, kExpFloor);
    }
    const F2 e = f2(ex2(t0), ex2(t1));
    s = f2_add(s, e);
    if (ENTROPY) a = f2_fma(e, f2(t0, t1), a);
  }
  float s0, s1, a0, a1;
  f2_split(s, s0, s1);
  st.s += s0 + s1;
  if (ENTROPY) {
    f2_split(a, a0, a1);
    st.a += a0 + a1;
  }
}

// A thread's running softmax state over vectors: the two sums in pairs, and a base m that is a value
// of the row but may be below its largest by up to kBaseSlack in the exponent, so that the sums are
// rescaled a few times a row and not whenever a new maximum comes (terms stay below 2^kBaseSlack).
constexpr float kBaseSlack = 8.0f;
struct SoftSums {
  float m;
  F2 s, a;
  __device__ __forceinline__ explicit SoftSums(const SoftState& st)
      : m(st.m), s(f2(st.s, 0.0f)), a(f2(st.a, 0.0f)) {}
  // N vectors whose largest element is `largest`.
  template <bool ENTROPY, typename T, int N>
  __device__ __forceinline__ void add(const uint4 (&w)[N], float largest, float c, float slack) {
    if (!(largest <= m + slack)) {  // a NaN too
      const float to = max_nan(largest, m);
      const float d = max_nan((m - to) * c, kExpFloor), f = ex2(d);
      const F2 ff = f2(f, f);
      if (ENTROPY) a = f2_mul(ff, f2_fma(f2(d, d), s, a));
      s = f2_mul(ff, s);
      m = to;
    }
    if (m == neg_inf()) return;
    const F2 nm = f2(-m, -m), cc = f2(c, c);
    F2 ps = f2(0.0f, 0.0f), pa = f2(0.0f, 0.0f);
#pragma unroll
    for (int u = 0; u < N; ++u) {
      float x[kVec<T>];
      unpack(w[u], x);
#pragma unroll
      for (int i = 0; i < kVec<T>; i += 2) {
        float t0, t1;
        f2_split(f2_mul(f2_add(f2(x[i], x[i + 1]), nm), cc), t0, t1);
        if (ENTROPY) {
          t0 = max_nan(t0, kExpFloor);
          t1 = max_nan(t1, kExpFloor);
        }
        const F2 e = f2(ex2(t0), ex2(t1));
        ps = f2_add(ps, e);
        if (ENTROPY) pa = f2_fma(e, f2(t0, t1), pa);
      }
    }
    s = f2_add(s, ps);
    if (ENTROPY) a = f2_add(a, pa);
  }
  __device__ __forceinline__ SoftState state() const {
    float s0, s1, a0, a1;
    f2_split(s, s0, s1);
    f2_split(a, a0, a1);
    return {m, s0 + s1, a0 + a1};
  }
};

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, d));
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
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
// Softmax state of a row that a warp holds N elements a lane of: the maximum first, then the sums.
template <bool ENTROPY, int N>
__device__ __forceinline__ SoftState soft_of_warp(const float (&x)[N], float edge, float c) {
  float m = edge;
#pragma unroll
  for (int i = 0; i < N; ++i) m = max_nan(m, x[i]);
  SoftState st = {warp_max(m), 0.0f, 0.0f};
  if (st.m == neg_inf()) return st;
  soft_sum<ENTROPY>(st, x, c);
  const float t = max_nan((edge - st.m) * c, kExpFloor), e = ex2(t);
  st.s = warp_sum(st.s + e);
  if (ENTROPY) st.a = warp_sum(fmaf(e, t, st.a));
  return st;
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
