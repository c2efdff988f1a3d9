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

// Offset of row r of a two-level layout (outer stride, inner stride) in elements.
struct RowLayout {
  int64_t so = 0, si = 0;
  __host__ __device__ __forceinline__ int64_t at(int64_t outer, int64_t inner) const {
    return outer * so + inner * si;
  }
};

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
__device__ __forceinline__ SoftState soft_warp(SoftState st, float c) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const SoftState other = {__shfl_xor_sync(0xffffffffu, st.m, o),
                             __shfl_xor_sync(0xffffffffu, st.s, o),
                             __shfl_xor_sync(0xffffffffu, st.a, o)};
    st = soft_merge(st, other, c);
  }
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

}  // namespace bdh
