// Distillation from the log probabilities that a teacher kept for its top tokens, and its
// gradient. With the student's z = x / temperature and p = softmax(z), and a row's list of K
// (token, teacher value) slots:
//
//   q_j   : tail = 0: softmax of the list's values; tail = 1: exp(value_j), and the class "every
//           other token" with r = max(0, 1 - sum_j q_j) against s = sum of p over unlisted tokens
//   loss  = w [ sum_j q_j (ln q_j - ln p[token_j]) + r (ln r - ln s) ]
//   dx_i  = w/temperature [ p_i (sum_j q_j + r) - r (p_i / s) [i unlisted] - sum_j q_j [i = token_j] ]
//
// A slot with token < 0 is empty; a repeated token's masses add; a row of weight 0 is not read.
// The unlisted tokens are summed by themselves, so that s keeps its digits when the list holds
// nearly everything. A row's slice is copied to shared memory (cp.async), the listed tokens are
// struck out there (-inf), the rest is summed from it and, in the same call, turned into the
// gradient from it, so that the logits cross HBM once. A warp takes a short row; else a CTA, or a
// cluster whose CTAs hold a slice each and exchange their sums through distributed shared memory.
// The backward from stored statistics has nothing to sum and streams.
//
// Repeated tokens are found while striking out: every slot writes its number in place of its token's
// logit and reads it back, and where one finds another's number the masses are added up by a search
// (K^2 comparisons, which as a rule cost more than the row itself and are seldom needed).
#include <algorithm>
#include <string>

#include "bdh_sm100.h"
#include "internal.h"
#include "logits.cuh"
#include "tma_host.h"

namespace bdh {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kPiece = 16384;             // elements of a row per CTA of the streaming backward
constexpr int kSliceBytes = 68 * 1024;    // of a row per CTA, while the cluster may grow
static_assert(kThreads >= kTopMax, "one thread per slot");

constexpr int kStats = 8;  // floats per row: see RowStats

// What the forward leaves for the gradient.
struct RowStats {
  float m, ln_s;            // a base near the largest logit, ln of the sum of exp((x - m) / temperature)
  float rest_m, ln_rest;    // the same of the unlisted tokens
  float total, r;           // mass of the list, and of the class beside it
  float shift;              // ln q = teacher's value - shift
  float repeated;           // 1: a token is in the list twice
};
static_assert(sizeof(RowStats) == kStats * sizeof(float), "stored as it is");

// What the gradient needs of a row: dx_i = 2^(c (x_i - m) + shift) coef for unlisted tokens.
struct RowGradient {
  float m, shift, coef;        // unlisted: with a tail relative to their own sum s, however small
  float top_m, top_shift;      // listed: p = 2^(c (z - top_m) + top_shift)
  float scale, total;          // listed: scale (p total - mass)
  bool none;                   // no logit above -inf in the row
};
__device__ __forceinline__ RowGradient row_gradient(const RowStats& st, int tail, float inv_t,
                                                    float scale) {
  RowGradient g;
  g.none = st.m == neg_inf();
  g.scale = scale * inv_t;
  g.total = st.total + st.r;
  g.top_m = st.m;
  g.top_shift = -st.ln_s * kLog2e;
  g.m = st.m;
  g.shift = g.top_shift;
  g.coef = g.scale * g.total;
  if (tail) {
    // p_i (total - r / s) = (p_i / s) (total s - r); nothing is unlisted and above -inf: all zeros
    const float s = expf((st.rest_m - st.m) * inv_t + st.ln_rest - st.ln_s);
    const bool empty = st.rest_m == neg_inf();
    g.m = empty ? 0.0f : st.rest_m;
    g.shift = empty ? neg_inf() : -st.ln_rest * kLog2e;
    g.coef = empty ? 0.0f : g.scale * (g.total * s - st.r);
    if (g.total != g.total) g.coef = g.total;
  }
  return g;
}
__device__ __forceinline__ float listed_gradient(const RowGradient& g, float z, float mass, float c) {
  return g.scale * (ex2(fmaf(z - g.top_m, c, g.top_shift)) * g.total - mass);
}
// The formula for unlisted tokens, on one element and on two.
struct Unlisted {
  RowGradient g;
  float c;
  F2 nm2, c2, shift2, coef2;
  __device__ __forceinline__ Unlisted(const RowGradient& g_, float c_)
      : g(g_), c(c_), nm2(f2(-g_.m, -g_.m)), c2(f2(c_, c_)), shift2(f2(g_.shift, g_.shift)),
        coef2(f2(g_.coef, g_.coef)) {}
  __device__ __forceinline__ float operator()(float x) const {
    return ex2(fmaf(x - g.m, c, g.shift)) * g.coef;
  }
  __device__ __forceinline__ void operator()(float x0, float x1, float& d0, float& d1) const {
    float y0, y1;
    f2_split(f2_fma(f2_add(f2(x0, x1), nm2), c2, shift2), y0, y1);
    f2_split(f2_mul(f2(ex2(y0), ex2(y1)), coef2), d0, d1);
  }
};
struct Nothing {
  __device__ __forceinline__ float operator()(float) const { return 0.0f; }
  __device__ __forceinline__ void operator()(float, float, float& a, float& b) const { a = b = 0.0f; }
};

// Loss of a row from its list (one warp; `slot(f)` calls f(ln q, q, z) for the lane's slots).
template <typename Slots>
__device__ __forceinline__ float warp_loss(const RowStats& st, float inv_t, Slots slots) {
  const bool none = st.m == neg_inf();
  float loss = 0.0f;
  slots([&](float lnq, float q, float z) {
    const float lp = none || z == neg_inf() ? neg_inf() : (z - st.m) * inv_t - st.ln_s;
    if (!(q <= 0.0f)) loss = fmaf(q, lnq - lp, loss);
  });
  loss = warp_sum(loss);
  if (st.r > 0.0f) {
    const float ls = st.rest_m == neg_inf() ? neg_inf()
                                            : (st.rest_m - st.m) * inv_t + st.ln_rest - st.ln_s;
    loss = fmaf(st.r, logf(st.r) - ls, loss);
  }
  return st.total != st.total ? quiet_nan() : loss;
}

// A slot's token: -1 for an empty one, V for one past the vocabulary.
__device__ __forceinline__ int slot_token(int64_t at, int V) {
  return at < 0 ? -1 : at < V ? static_cast<int>(at) : V;
}
// A slot's number in place of a logit, and back.
__device__ __forceinline__ void put_slot(float* p, int64_t at, int slot) {
  reinterpret_cast<int*>(p)[at] = slot;
}
__device__ __forceinline__ void put_slot(uint16_t* p, int64_t at, int slot) {
  p[at] = static_cast<uint16_t>(slot);
}
__device__ __forceinline__ int get_slot(const float* p, int64_t at) {
  return reinterpret_cast<const int*>(p)[at];
}
__device__ __forceinline__ int get_slot(const uint16_t* p, int64_t at) { return p[at]; }

template <typename T>
__device__ __forceinline__ float row_weight(const DistillTopkArgs& a, int64_t o, int64_t i) {
  return a.weight.p != nullptr ? a.weight.p[o * a.weight.strides[0] + i * a.weight.strides[1]] : 1.0f;
}
// ------------------------------------------------------------------ a warp for a short row
// Rows of at most kShort elements: the slots and the row's elements stay in the lanes' registers
// (S slots, E elements and one of the row's unaligned ends); the row passes through shared memory
// for the slots to find their logits.
constexpr int kShort = 1024;

template <typename T, int E, int S>
__global__ void __launch_bounds__(kThreads, E <= 16 && S == 1 ? 4 : 3) distill_short_kernel(DistillTopkArgs a) {
  constexpr int kV = kVec<T>, kVecs = E / kV;
  __shared__ __align__(16) T rows_held[kWarps][(kVecs * 32 + 2) * kV];
  const int lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  if (row >= a.outer * a.inner) return;
  const int64_t o = static_cast<uint32_t>(row) / static_cast<uint32_t>(a.inner), i = row - o * a.inner;
  const int V = static_cast<int>(a.V), K = static_cast<int>(a.K);
  const T* x = static_cast<const T*>(a.logits) + o * a.l_strides[0] + i * a.l_strides[1];
  T* d = a.dlogits != nullptr
             ? static_cast<T*>(a.dlogits) + o * a.d_strides[0] + i * a.d_strides[1]
             : nullptr;
  const float w = row_weight<T>(a, o, i);
  if (w == 0.0f) {
    if (d != nullptr) map_row<T, 32>(x, d, V, lane, true, Nothing(), Nothing());
    if (lane == 0) a.loss[row] = 0.0f;
    return;
  }
  // the row on its way to shared memory, the list to registers
  const RowSpan span = row_span(x, V);
  T* held = rows_held[threadIdx.x >> 5] + (kV - span.head) % kV;
  const uint4* vec = reinterpret_cast<const uint4*>(x + span.head);
  uint4* hvec = reinterpret_cast<uint4*>(held + span.head);
#pragma unroll
  for (int u = 0; u < kVecs; ++u) {
    const int v = u * 32 + lane;
    if (v < span.vecs)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(hvec + v)), "l"(vec + v)
                   : "memory");
  }
  int edge = -1;  // this lane's element of the row's ends
  if (lane < span.head) edge = lane;
  if (lane >= 8 && lane - 8 < span.tail) edge = V - span.tail + lane - 8;
  if (edge >= 0) held[edge] = x[edge];
  int at[S];
  float lnq[S], q[S], z[S], mass[S];
#pragma unroll
  for (int s = 0; s < S; ++s) {
    const int j = s * 32 + lane;
    at[s] = -1;
    lnq[s] = neg_inf();
    if (j < K) {
      at[s] = slot_token(a.index[o * a.i_strides[0] + i * a.i_strides[1] + j * a.i_strides[2]], V);
      const float t = a.teacher[o * a.t_strides[0] + i * a.t_strides[1] + j * a.t_strides[2]];
      if (at[s] >= 0) lnq[s] = t;
    }
  }
  const float inv_t = 1.0f / a.temperature, c = kLog2e * inv_t;
  RowStats st;
  st.shift = 0.0f;
  if (!a.tail) {
    float m = lnq[0], sum = 0.0f;
#pragma unroll
    for (int s = 1; s < S; ++s) m = max_nan(m, lnq[s]);
    m = warp_max(m);
    if (m != neg_inf()) {
#pragma unroll
      for (int s = 0; s < S; ++s) sum += expf(lnq[s] - m);
      st.shift = m + logf(warp_sum(sum));
    }
  }
  st.total = 0.0f;
  bool bad = false;
#pragma unroll
  for (int s = 0; s < S; ++s) {
    lnq[s] -= st.shift;
    q[s] = expf(lnq[s]);
    st.total += q[s];
    bad |= at[s] == V;
    if (at[s] == V) at[s] = -1;  // no token to find
    mass[s] = at[s] >= 0 ? q[s] : -1.0f;
  }
  st.total = warp_sum(st.total);
  st.r = a.tail ? max_nan(0.0f, 1.0f - st.total) : 0.0f;
  if (__any_sync(0xffffffffu, bad)) st.total = quiet_nan();
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncwarp();
#pragma unroll
  for (int s = 0; s < S; ++s) z[s] = at[s] >= 0 ? logit_at<T>(held, at[s]) : neg_inf();
  __syncwarp();
#pragma unroll
  for (int s = 0; s < S; ++s)
    if (at[s] >= 0) put_slot(held, at[s], s * 32 + lane);
  __syncwarp();
  bool other = false;
#pragma unroll
  for (int s = 0; s < S; ++s) other |= at[s] >= 0 && get_slot(held, at[s]) != s * 32 + lane;
  st.repeated = __any_sync(0xffffffffu, other) ? 1.0f : 0.0f;  // and all have read
#pragma unroll
  for (int s = 0; s < S; ++s)
    if (at[s] >= 0) logit_put(held, at[s], neg_inf());
  __syncwarp();
  if (st.repeated != 0.0f) {  // masses to the first slot of each token
#pragma unroll
    for (int s = 0; s < S; ++s) {
      float sum = 0.0f;
      bool first = at[s] >= 0;
#pragma unroll
      for (int t = 0; t < S; ++t)
        for (int k = 0; k < 32; ++k) {
          const int other_at = __shfl_sync(0xffffffffu, at[t], k);
          const float other_q = __shfl_sync(0xffffffffu, q[t], k);
          if (other_at != at[s]) continue;
          sum += other_q;
          if (t * 32 + k < s * 32 + lane) first = false;
        }
      mass[s] = first ? sum : -1.0f;
    }
  }
  int distinct = 0;
  float zs[S < 2 ? 2 : S];
  if (S < 2) zs[1] = neg_inf();
#pragma unroll
  for (int s = 0; s < S; ++s) {
    const bool own = !(mass[s] < 0.0f);
    zs[s] = own ? z[s] : neg_inf();
    distinct += own ? 1 : 0;
  }
  if (K >= V && a.tail) {  // where every token is listed there is no other class
    if (__reduce_add_sync(0xffffffffu, distinct) >= V) st.r = 0.0f;
  }

  float xs[E];
#pragma unroll
  for (int u = 0; u < kVecs; ++u) {
    const int v = u * 32 + lane;
    float part[kV];
    unpack(v < span.vecs ? hvec[v] : void_vec<T>(), part);
#pragma unroll
    for (int e = 0; e < kV; ++e) xs[u * kV + e] = part[e];
  }
  const float edge_x = edge >= 0 ? logit_at<T>(held, edge) : neg_inf();
  const SoftState rest = soft_of_warp<false>(xs, edge_x, c);
  const SoftState all = soft_merge(rest, soft_of_warp<false>(zs, neg_inf(), c), c);
  st.m = all.m;
  st.ln_s = all.m == neg_inf() ? neg_inf() : logf(all.s);
  st.rest_m = rest.m;
  st.ln_rest = rest.m == neg_inf() ? neg_inf() : logf(rest.s);
  const float loss = warp_loss(st, inv_t, [&](auto f) {
#pragma unroll
    for (int s = 0; s < S; ++s) f(lnq[s], q[s], z[s]);
  });
  if (lane == 0) {
    a.loss[row] = w * loss;
    if (a.stats != nullptr) *reinterpret_cast<RowStats*>(a.stats + kStats * row) = st;
  }
  if (d == nullptr) return;

  const RowGradient g = row_gradient(st, a.tail, inv_t, w);
  const Unlisted f(g, c);
  if (edge >= 0) logit_put(d, edge, g.none ? 0.0f : f(edge_x));
  T* out = d + span.head;
  const bool aligned = (reinterpret_cast<uintptr_t>(out) & 15u) == 0;
#pragma unroll
  for (int u = 0; u < kVecs; ++u) {
    const int v = u * 32 + lane;
    if (v >= span.vecs) continue;
    float ds[kV];
#pragma unroll
    for (int e = 0; e < kV; e += 2) {
      f(xs[u * kV + e], xs[u * kV + e + 1], ds[e], ds[e + 1]);
      if (g.none) ds[e] = ds[e + 1] = 0.0f;
    }
    if (aligned) {
      store_vec(out + v * kV, ds);
    } else {
#pragma unroll
      for (int e = 0; e < kV; ++e) logit_put(out, v * kV + e, ds[e]);
    }
  }
  if (g.none) return;
  __syncwarp();
#pragma unroll
  for (int s = 0; s < S; ++s)
    if (!(mass[s] < 0.0f)) logit_put(d, at[s], listed_gradient(g, z[s], mass[s], c));
}

// ------------------------------------------------------------ a CTA or a cluster for a row
struct CtaShared {
  float2 part[kMaxCluster * kWarps];  // maximum and sum of every warp of the cluster
  int repeated[kMaxCluster];          // a token is twice in the list, and in that CTA's slice
  SoftState top;                      // softmax state of the listed tokens
  float total, r, shift;
  int index[kTopMax];  // -1: empty slot; V: a token past the vocabulary
  float lnq[kTopMax], q[kTopMax], z[kTopMax];
  float mass[kTopMax];  // q summed over the slots of the same token; below 0: not its first slot
};
static_assert(sizeof(CtaShared) % 4 == 0, "the slice follows, aligned");
constexpr size_t kCtaShared = (sizeof(CtaShared) + 15) & ~size_t(15);

// Masses of repeated tokens to the first slot of each, and the listed tokens' softmax state
// (one warp).
__device__ __forceinline__ void list_state(CtaShared& sh, int K, int V, int lane, float c, bool repeated) {
  float zs[kTopMax / 32];
#pragma unroll
  for (int s = 0; s < kTopMax / 32; ++s) {
    const int j = s * 32 + lane;
    zs[s] = neg_inf();
    if (j >= K) continue;
    const int at = sh.index[j];
    const bool token = at >= 0 && at < V;
    float mass = token ? sh.q[j] : -1.0f;
    if (repeated && token) {
      mass = 0.0f;
      bool first = true;
      for (int k = 0; k < K; ++k)
        if (sh.index[k] == at) {
          mass += sh.q[k];
          if (k < j) first = false;
        }
      if (!first) mass = -1.0f;
    }
    sh.mass[j] = mass;
    if (!(mass < 0.0f)) zs[s] = sh.z[j];
  }
  const SoftState top = soft_of_warp<false>(zs, neg_inf(), c);
  if (lane == 0) sh.top = top;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) distill_topk_kernel(DistillTopkArgs a, int C) {
  extern __shared__ __align__(16) uint8_t smem[];
  constexpr int kV = kVec<T>;
  CtaShared& sh = *reinterpret_cast<CtaShared*>(smem);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int V = static_cast<int>(a.V), K = static_cast<int>(a.K);
  const uint32_t rank = C > 1 ? cta_rank() : 0;
  const int64_t row = blockIdx.x / static_cast<uint32_t>(C);
  const int64_t o = static_cast<uint32_t>(row) / static_cast<uint32_t>(a.inner), i = row - o * a.inner;
  const T* x = static_cast<const T*>(a.logits) + o * a.l_strides[0] + i * a.l_strides[1];
  T* d = a.dlogits != nullptr
             ? static_cast<T*>(a.dlogits) + o * a.d_strides[0] + i * a.d_strides[1]
             : nullptr;

  // This CTA's slice: vectors [v0, v1) between the row's 16-byte boundaries, the row's head with
  // the first slice and its tail with the last; n elements from `from`.
  const RowSpan span = row_span(x, V);
  const int per = (span.vecs + C - 1) / C;
  const int v0 = min(static_cast<int>(rank) * per, span.vecs), v1 = min(v0 + per, span.vecs);
  const int head = rank == 0 ? span.head : 0, tail = rank == C - 1 ? span.tail : 0;
  const int from = span.head + v0 * kV - head, vecs = v1 - v0, n = head + vecs * kV + tail;

  const float w = row_weight<T>(a, o, i);
  if (w == 0.0f) {  // the whole cluster
    if (d != nullptr) map_row<T, kThreads>(x + from, d + from, n, tid, true, Nothing(), Nothing());
    if (tid == 0 && rank == 0) a.loss[row] = 0.0f;
    return;
  }
  if (C > 1) cluster_arrive();  // shared memory may be written once all CTAs have started

  T* held = reinterpret_cast<T*>(smem + kCtaShared) + (kV - head) % kV;  // element from + e: held[e]
  const uint4* vec = reinterpret_cast<const uint4*>(x + span.head) + v0;
  uint4* hvec = reinterpret_cast<uint4*>(held + head);
  for (int v = tid; v < vecs; v += kThreads)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(hvec + v)), "l"(vec + v)
                 : "memory");
  const int edge = tid < head ? tid : tid - head < tail ? n - tail + tid - head : -1;
  if (edge >= 0) held[edge] = x[from + edge];
  if (tid < K) {
    const int at = slot_token(a.index[o * a.i_strides[0] + i * a.i_strides[1] + tid * a.i_strides[2]], V);
    const float t = a.teacher[o * a.t_strides[0] + i * a.t_strides[1] + tid * a.t_strides[2]];
    sh.index[tid] = at;
    sh.lnq[tid] = at >= 0 ? t : neg_inf();
    sh.z[tid] = at >= 0 && at < V ? logit_at<T>(x, at) : neg_inf();
  }
  const float inv_t = 1.0f / a.temperature, c = kLog2e * inv_t;
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();  // the slice and the list are in shared memory
  auto in_slice = [&](int at) { return at >= from && at < from + n; };
  if (warp == 0) {  // strike the listed tokens out
    for (int j = lane; j < K; j += 32)
      if (in_slice(sh.index[j])) put_slot(held, sh.index[j] - from, j);
    __syncwarp();
    bool other = false;
    for (int j = lane; j < K; j += 32)
      if (in_slice(sh.index[j])) other |= get_slot(held, sh.index[j] - from) != j;
    other = __any_sync(0xffffffffu, other);  // and all have read
    for (int j = lane; j < K; j += 32)
      if (in_slice(sh.index[j])) logit_put(held, sh.index[j] - from, neg_inf());
    if (lane == 0) sh.repeated[rank] = other ? 1 : 0;
  } else if (warp == 1) {  // the list's masses
    float m = neg_inf(), shift = 0.0f, total = 0.0f;
    if (!a.tail) {
      for (int j = lane; j < K; j += 32) m = max_nan(m, sh.lnq[j]);
      m = warp_max(m);
      if (m != neg_inf()) {
        float s = 0.0f;
        for (int j = lane; j < K; j += 32) s += expf(sh.lnq[j] - m);
        shift = m + logf(warp_sum(s));
      }
    }
    bool bad = false;
    for (int j = lane; j < K; j += 32) {
      const float l = sh.lnq[j] - shift, q = expf(l);
      sh.lnq[j] = l;
      sh.q[j] = q;
      total += q;
      bad |= sh.index[j] == V;
    }
    total = warp_sum(total);
    bad = __any_sync(0xffffffffu, bad);
    if (lane == 0) {
      sh.total = bad ? quiet_nan() : total;  // a token past the vocabulary: NaN throughout
      sh.r = a.tail ? max_nan(0.0f, 1.0f - total) : 0.0f;
      sh.shift = shift;
    }
    __syncwarp();
    list_state(sh, K, V, lane, c, false);
  }
  __syncthreads();

  SoftState rest = soft_empty();
  if (edge >= 0) soft_add(rest, logit_at<T>(held, edge), c);
  SoftSums sums(rest);
  const float slack = kBaseSlack / c;
  for (int b = 0; b < vecs; b += kThreads * kUnroll) {
    uint4 wv[kUnroll];
    if (b + kThreads * kUnroll <= vecs) {
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) wv[u] = hvec[b + u * kThreads + tid];
    } else {
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int v = b + u * kThreads + tid;
        wv[u] = v < vecs ? hvec[v] : void_vec<T>();
      }
    }
    sums.add<false, T>(wv, max_of(wv, T()), c, slack);
  }
  rest = sums.state();
  rest = soft_join(rest, c);
  if (C > 1) {  // every warp's state to every CTA of the cluster
    cluster_wait();
    if (lane < C) {
      const uint32_t to = peer_smem(&sh.part[rank * kWarps + warp], lane);
      peer_store(to, rest.m);
      peer_store(to + 4, rest.s);
      if (warp == 0) peer_store(peer_smem(&sh.repeated[rank], lane), __int_as_float(sh.repeated[rank]));
    }
    cluster_arrive();
    cluster_wait();
  } else {
    if (lane == 0) sh.part[warp] = make_float2(rest.m, rest.s);
    __syncthreads();
  }
  rest = soft_empty();
  for (int k = lane; k < C * kWarps; k += 32)
    rest = soft_merge(rest, {sh.part[k].x, sh.part[k].y, 0.0f}, c);
  rest = soft_join(rest, c);
  const bool repeated = __any_sync(0xffffffffu, lane < C && sh.repeated[lane] != 0);
  if (repeated) {  // in every CTA of the cluster
    __syncthreads();
    if (warp == 1) list_state(sh, K, V, lane, c, true);
    __syncthreads();
  }
  const SoftState all = soft_merge(rest, {sh.top.m, sh.top.s, 0.0f}, c);
  RowStats st;
  st.m = all.m;
  st.ln_s = all.m == neg_inf() ? neg_inf() : logf(all.s);
  st.rest_m = rest.m;
  st.ln_rest = rest.m == neg_inf() ? neg_inf() : logf(rest.s);
  st.total = sh.total;
  st.r = sh.r;
  st.shift = sh.shift;
  st.repeated = repeated ? 1.0f : 0.0f;
  if (rank == 0 && warp == 0) {
    const float loss = warp_loss(st, inv_t, [&](auto f) {
      for (int j = lane; j < K; j += 32) f(sh.lnq[j], sh.q[j], sh.z[j]);
    });
    if (lane == 0) {
      a.loss[row] = w * loss;
      if (a.stats != nullptr) *reinterpret_cast<RowStats*>(a.stats + kStats * row) = st;
    }
  }
  if (d == nullptr) return;

  const RowGradient g = row_gradient(st, a.tail, inv_t, w);
  const Unlisted f(g, c);
  T* out = d + from + head;
  if ((reinterpret_cast<uintptr_t>(out) & 15u) == 0) {
    if (edge >= 0) logit_put(d, from + edge, g.none ? 0.0f : f(logit_at<T>(held, edge)));
    for (int v = tid; v < vecs; v += kThreads) {
      float xs[kV], ds[kV];
      unpack(hvec[v], xs);
#pragma unroll
      for (int e = 0; e < kV; e += 2) {
        f(xs[e], xs[e + 1], ds[e], ds[e + 1]);
        if (g.none) ds[e] = ds[e + 1] = 0.0f;
      }
      store_vec(out + static_cast<int64_t>(v) * kV, ds);
    }
  } else {  // x and d lie differently in their vectors
    for (int e = tid; e < n; e += kThreads)
      logit_put(d, from + e, g.none ? 0.0f : f(logit_at<T>(held, e)));
  }
  if (g.none) return;
  __syncthreads();
  if (tid < K && in_slice(sh.index[tid]) && !(sh.mass[tid] < 0.0f))
    logit_put(d, sh.index[tid], listed_gradient(g, sh.z[tid], sh.mass[tid], c));
}

// --------------------------------------------------- the gradient from the forward's statistics
template <typename T, int G>
__global__ void __launch_bounds__(kThreads) distill_topk_bwd_kernel(DistillTopkArgs a, int pieces,
                                                                    int piece) {
  const int tid = threadIdx.x % G, group = threadIdx.x / G;
  const int V = static_cast<int>(a.V), K = static_cast<int>(a.K);
  const uint32_t unit = blockIdx.x * (kThreads / G) + group;
  const int64_t row = unit / static_cast<uint32_t>(pieces);
  if (row >= a.outer * a.inner) return;  // whole warps of the warp form
  const int64_t o = static_cast<uint32_t>(row) / static_cast<uint32_t>(a.inner), i = row - o * a.inner;
  const int from = static_cast<int>(unit - static_cast<uint32_t>(row) * pieces) * piece;
  const int n = min(piece, V - from);
  const T* x = static_cast<const T*>(a.logits) + o * a.l_strides[0] + i * a.l_strides[1];
  T* d = static_cast<T*>(a.dlogits) + o * a.d_strides[0] + i * a.d_strides[1];
  const float w = row_weight<T>(a, o, i);
  if (w == 0.0f) {
    map_row<T, G>(x + from, d + from, n, tid, true, Nothing(), Nothing());
    return;
  }
  const float inv_t = 1.0f / a.temperature, c = kLog2e * inv_t;
  const RowStats st = *reinterpret_cast<const RowStats*>(a.stats + kStats * row);
  const float up = a.g_loss.p[o * a.g_loss.strides[0] + i * a.g_loss.strides[1]];
  const RowGradient g = row_gradient(st, a.tail, inv_t, w * up);
  const Unlisted f(g, c);
  map_row<T, G>(x + from, d + from, n, tid, g.none, f, f);
  if (g.none) return;
  if (G == 32) __syncwarp();
  else __syncthreads();
  // the listed tokens of this piece, over what the formula for the others left there
  const int64_t* index = a.index + o * a.i_strides[0] + i * a.i_strides[1];
  const float* teacher = a.teacher + o * a.t_strides[0] + i * a.t_strides[1];
  for (int j = tid; j < K; j += G) {
    const int64_t at = index[j * a.i_strides[2]];
    if (at < from || at >= from + n) continue;
    float mass = expf(teacher[j * a.t_strides[2]] - st.shift);
    if (st.repeated != 0.0f) {
      bool first = true;
      mass = 0.0f;
      for (int k = 0; first && k < K; ++k)
        if (index[k * a.i_strides[2]] == at) {
          mass += expf(teacher[k * a.t_strides[2]] - st.shift);
          first = k >= j;
        }
      if (!first) continue;
    }
    logit_put(d, at, listed_gradient(g, logit_at<T>(x, at), mass, c));
  }
}

int launch_check(const char* what, cudaError_t e) {
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) {
    set_error(std::string(what) + ": " + cudaGetErrorString(e));
    return BDH_ERR_CUDA;
  }
  return BDH_OK;
}

template <typename T, int E>
int launch_short(const DistillTopkArgs& a, cudaStream_t stream) {
  const unsigned grid = static_cast<unsigned>((a.outer * a.inner + kWarps - 1) / kWarps);
  if (a.K <= 32) distill_short_kernel<T, E, 1><<<grid, kThreads, 0, stream>>>(a);
  else distill_short_kernel<T, E, kTopMax / 32><<<grid, kThreads, 0, stream>>>(a);
  return launch_check("distill_topk launch", cudaSuccess);
}

template <typename T>
int forward_by_size(const DistillTopkArgs& a, cudaStream_t stream) {
  if (a.V <= 256) return launch_short<T, 8>(a, stream);
  if (a.V <= 512) return launch_short<T, 16>(a, stream);
  if (a.V <= kShort) return launch_short<T, 32>(a, stream);
  int dev = 0;
  cudaGetDevice(&dev);
  const int64_t rows = a.outer * a.inner, bytes = a.V * static_cast<int64_t>(sizeof(T));
  int cluster = 1;
  while (cluster < kMaxCluster &&
         (bytes > static_cast<int64_t>(cluster) * kSliceBytes ||
          (rows * cluster < 4 * sm_count(dev) && bytes >= cluster * int64_t(32768))))
    cluster *= 2;
  if (rows * cluster >= int64_t(1) << 31) {
    set_error("distill_topk: too many rows for this vocabulary");
    return BDH_ERR_INVALID;
  }
  // a slice's vectors, and one more for the row's head and one for its tail
  const size_t smem = kCtaShared + (static_cast<size_t>((a.V / kVec<T> + cluster - 1) / cluster) + 2) * 16;
  auto* kern = distill_topk_kernel<T>;
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               static_cast<int>(smem));
    if (e != cudaSuccess) return launch_check("distill_topk shared memory", e);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(rows * cluster));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 1 : 0;
  return launch_check("distill_topk launch", cudaLaunchKernelEx(&cfg, kern, a, cluster));
}

template <typename T>
int backward_by_size(const DistillTopkArgs& a, cudaStream_t stream) {
  const int64_t rows = a.outer * a.inner;
  if (a.V <= kShort) {
    const unsigned grid = static_cast<unsigned>((rows + kWarps - 1) / kWarps);
    distill_topk_bwd_kernel<T, 32><<<grid, kThreads, 0, stream>>>(a, 1, static_cast<int>(a.V));
  } else {
    const int64_t pieces = (a.V + kPiece - 1) / kPiece;
    if (rows * pieces >= int64_t(1) << 31) {
      set_error("distill_topk_bwd: too many rows for this vocabulary");
      return BDH_ERR_INVALID;
    }
    distill_topk_bwd_kernel<T, kThreads><<<static_cast<unsigned>(rows * pieces), kThreads, 0, stream>>>(
        a, static_cast<int>(pieces), kPiece);
  }
  return launch_check("distill_topk_bwd launch", cudaSuccess);
}

}  // namespace

int launch_distill_topk(const DistillTopkArgs& a, cudaStream_t stream) {
  if (a.outer * a.inner == 0) return BDH_OK;
  return a.dtype == BDH_DTYPE_F32 ? forward_by_size<float>(a, stream)
                                  : forward_by_size<uint16_t>(a, stream);
}

int launch_distill_topk_bwd(const DistillTopkArgs& a, cudaStream_t stream) {
  if (a.outer * a.inner == 0) return BDH_OK;
  return a.dtype == BDH_DTYPE_F32 ? backward_by_size<float>(a, stream)
                                  : backward_by_size<uint16_t>(a, stream);
}

}  // namespace bdh
