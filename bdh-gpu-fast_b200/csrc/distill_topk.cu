// Distillation from the log probabilities that a teacher kept for its top tokens, and its
// gradient. With the student's z = x / temperature and p = softmax(z), and a row's list of K
// (token, teacher value) slots:
//
//   q_j   : tail = 0: softmax of the list's values; tail = 1: exp(value_j), and the class "every
//           other token" with r = max(0, 1 - sum_j q_j) against s = sum of p over unlisted tokens
//   loss  = w [ sum_j q_j (ln q_j - ln p[token_j]) + r (ln r - ln s) ]
//   dx_i  = w/temperature [ p_i (sum_j q_j + r) - r (p_i / s) [i unlisted] - sum_j q_j [i = token_j] ]
//
// A slot with token < 0 is empty; a repeated token's masses add; a row of weight 0 counts for nothing,
// whatever it holds.
// The unlisted tokens are summed by themselves, so that s keeps its digits when the list holds
// nearly everything. Where the student masks all of them there is no class beside the list as long as r may
// be the list's rounding.
//
// A row that a warp takes passes through shared memory: the listed tokens are struck out there (-inf),
// the rest is summed from it and turned into the gradient from it. Repeated tokens are found on the
// way: every slot writes its number in place of its token's logit and reads it back.
// A longer row is streamed by a CTA of 128 or 256 threads, or by a cluster whose CTAs take a slice each and
// exchange their sums through distributed shared memory; a bit per element in shared memory says what is
// listed (and was set twice for a repeated token); a row whose bits have no room in one CTA is split over
// more. For the gradient the slice is streamed again, from L2.
// Where a token is repeated its masses are added up by a search (K^2 comparisons, seldom needed).
// The backward from stored statistics has nothing to sum.
//
// What bounds it: of long rows with a gradient neither memory nor the issue slots alone (66% and 0.63 of
// them in use): 2048 rows of 131072 in bf16 with K = 64 take 213 us, 5.0 TB/s of the 1.07 GB that must be
// read and written (DRAM moves 1.14: nearly all of the second pass comes from L2); warps wait for loads,
// and between the passes for one another. The loss alone of 600 rows of 100003 takes 26 us, 4.6 TB/s: 592
// CTAs run at a time, and the last 8 rows by themselves (592 rows: 24). Short rows with their lists are
// latency: 16384 rows of 256 with K = 16 take 9 us with their gradient.
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
// The backward from stored statistics: elements of a row per CTA, and the longest of many rows that are
// a warp's each. The bytes that it moves bound it, as the log probabilities' (measured there): 89 us for
// 1024 rows of 131072 in bf16, 6.0 TB/s; 6.3 us for 16384 rows of 256 by 8 lanes each.
constexpr int kPiece = 16384, kWarpGradBytes = 8 * 1024;
// A warp takes rows up to kWarpRowBytes where there are kWarpRows for every SM (kWarpsHeld a CTA, each
// held in shared memory). Loss and gradient of 8192 rows in bf16, by warps against by CTAs: 2048 long 19
// and 83 us, 8192 long 73 and 96, 16384 long 259 and 132 (four such rows fill more than half of an SM's
// shared memory); of 592 rows of 8192 11.9 and 8.7 us.
constexpr int kWarpRowBytes = 24 * 1024, kWarpRows = 8, kWarpsHeld = 4;
// With a gradient, a row longer than this is split over a cluster: the slices of some 600 CTAs in flight
// are read again from L2, with policies that keep them there until then. 2048 rows of 131072 in bf16:
// 128 KB slices 213 us, 64 KB 228 us (two CTAs more to wait for), whole rows of 256 KB 249 us (they no
// longer fit L2). Without the L2 policies 232, 224 and 255 us: the DRAM reads of 128 KB slices are then
// 0.98 GB, of 64 KB slices 0.54 GB. Few rows are split further, to three CTAs for every SM and 16 KB (one
// row of 131072 with its gradient: 20 us whole, 7.0 in eight; 128 rows 22 whole, 18 in two).
constexpr int kSliceBytes = 136 * 1024;
// Rows of up to this size that are not split are streamed by 128 threads instead of 256: more rows' lists
// and waits pass at a time, until the slices in flight outgrow L2. 8192 rows in bf16 by 128 and by 256
// threads: the loss of 16384 long ones 66 and 85 us, of 50021 141 and 160, of 65536 174 and 183 (1184
// rows 38 and 31); loss and gradient of 16384 long ones 115 and 130, of 20000 136 and 154, of 32768 204 and
// 205 (1184 rows 40 and 33).
constexpr int kHalfBytes = 112 * 1024, kHalfGradBytes = 48 * 1024;

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

// What the gradient needs of a row. Unlisted tokens: the map below, with a tail relative to their own
// sum s, however small it is: p_i (total - r / s) = (p_i / s) (total s - r).
struct RowGradient {
  float top_m, top_l2;   // listed: p = 2^(c (z - top_m) - top_l2), scale (p total - mass)
  float scale, total;
  float m, l2, coef;     // unlisted
  bool none;             // no logit above -inf in the row
  __device__ __forceinline__ RowMap unlisted(float c) const { return RowMap(c, m, l2, coef, 0.0f); }
  __device__ __forceinline__ float listed(float z, float mass, float c) const {
    return scale * (ex2(fmaf(z - top_m, c, -top_l2)) * total - mass);
  }
};
__device__ __forceinline__ RowGradient row_gradient(const RowStats& st, int tail, float inv_t,
                                                    float scale) {
  RowGradient g;
  g.none = st.m == neg_inf();
  g.scale = scale * inv_t;
  g.total = st.total + st.r;
  g.top_m = g.m = st.m;
  g.top_l2 = g.l2 = st.ln_s * kLog2e;
  g.coef = g.scale * g.total;
  if (tail) {
    const float s = expf((st.rest_m - st.m) * inv_t + st.ln_rest - st.ln_s);
    const bool empty = st.rest_m == neg_inf();  // nothing unlisted above -inf: zeros
    g.m = empty ? 0.0f : st.rest_m;
    g.l2 = empty ? 0.0f : st.ln_rest * kLog2e;
    g.coef = empty ? 0.0f : g.scale * (g.total * s - st.r);
    if (g.total != g.total) g.coef = g.total;
  }
  if (g.none) g.m = g.l2 = 0.0f;
  return g;
}
// ln of the student's probability outside the list.
__device__ __forceinline__ float ln_rest_mass(const RowStats& st, float inv_t) {
  return st.rest_m == neg_inf() ? neg_inf() : (st.rest_m - st.m) * inv_t + st.ln_rest - st.ln_s;
}
// A list of all that a teacher allows has a mass of 1 up to its rounding: r is then noise (K 2^-23, or a log
// softmax's 2^-24 of logits up to 256), which a student that masks everything else (-inf, or so low that no
// model's logits go there) would pay for with an infinite loss, or one of the mask's size.
constexpr float kListRounding = 1.0f / 65536.0f, kMaskedMass = -1000.0f;
__device__ __forceinline__ void settle_rest(RowStats& st, float inv_t) {
  if (st.r <= kListRounding && ln_rest_mass(st, inv_t) < kMaskedMass) st.r = 0.0f;
}
// Loss of a row from its list (L lanes; `slots(f)` calls f(ln q, q, z) for the lane's slots).
template <int L, typename Slots>
__device__ __forceinline__ float row_loss(const RowStats& st, float inv_t, Slots slots) {
  const bool none = st.m == neg_inf();
  float loss = 0.0f;
  slots([&](float lnq, float q, float z) {
    const float lp = none || z == neg_inf() ? neg_inf() : (z - st.m) * inv_t - st.ln_s;
    if (!(q <= 0.0f)) loss = fmaf(q, lnq - lp, loss);
  });
  loss = warp_sum<L>(loss);
  if (st.r > 0.0f) loss = fmaf(st.r, logf(st.r) - ln_rest_mass(st, inv_t), loss);
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

struct Nothing {
  __device__ __forceinline__ float operator()(float) const { return 0.0f; }
};

template <typename T>
__device__ __forceinline__ float row_weight(const DistillTopkArgs& a, int64_t o, int64_t i) {
  return a.weight.p != nullptr ? a.weight.p[o * a.weight.strides[0] + i * a.weight.strides[1]] : 1.0f;
}
// ------------------------------------------------------------------ lanes for a short row
// Rows of at most kShort elements: the slots and the row's elements stay in registers, S slots and E
// elements (and up to two of its unaligned ends) in each of the L lanes that have a row; the row passes
// through shared memory for the slots to find their logits. With few lanes a row the shuffles and the
// row's own figures serve several rows at once (a byte model's 256: 4 rows a warp; 16384 such rows with
// their gradient 9.0 us, 14.8 with a warp each).
constexpr int kShort = 1024;
static_assert(kTopMax <= kShort, "a list that holds a whole row is a short row's");

template <typename T, int L, int E, int S>
__global__ void __launch_bounds__(kThreads) distill_short_kernel(DistillTopkArgs a, FastDiv inner) {
  constexpr int kV = kVec<T>, kVecs = E / kV, kEnds = L < 16 ? 2 : 1, kN = E + kEnds;
  __shared__ __align__(16) T rows_held[kThreads / L][(kVecs * L + 2) * kV];
  const int lane = threadIdx.x % L, rows = static_cast<int>(a.outer * a.inner);
  int row = static_cast<int>(blockIdx.x * (kThreads / L) + threadIdx.x / L);
  const bool live = row < rows;
  if (!__any_sync(0xffffffffu, live)) return;
  if (!live) row = rows - 1;  // (the warp's other rows need these lanes)
  int o, i;
  inner.divmod(row, o, i);
  const int V = static_cast<int>(a.V), K = static_cast<int>(a.K);
  const T* x = static_cast<const T*>(a.logits) + o * a.l_strides[0] + i * a.l_strides[1];
  const float w = row_weight<T>(a, o, i);
  // the row on its way to shared memory, the list to registers
  const RowSpan span = row_span(x, V);
  T* held = rows_held[threadIdx.x / L] + (kV - span.head) % kV;
  const uint4* vec = reinterpret_cast<const uint4*>(x + span.head);
  uint4* hvec = reinterpret_cast<uint4*>(held + span.head);
#pragma unroll
  for (int u = 0; u < kVecs; ++u) {
    const int v = u * L + lane;
    if (v < span.vecs)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(hvec + v)), "l"(vec + v)
                   : "memory");
  }
  int end[kEnds];  // elements of the row's ends, or -1
  if (kEnds == 2) {
    end[0] = lane < span.head ? lane : -1;
    end[kEnds - 1] = lane < span.tail ? V - span.tail + lane : -1;
  } else {
    end[0] = lane < span.head ? lane : lane - span.head < span.tail ? V - span.tail + lane - span.head : -1;
  }
#pragma unroll
  for (int e = 0; e < kEnds; ++e)
    if (end[e] >= 0) held[end[e]] = x[end[e]];
  int at[S];
  float lnq[S], q[S], z[S], mass[S];
#pragma unroll
  for (int s = 0; s < S; ++s) {
    const int j = s * L + lane;
    at[s] = -1;
    lnq[s] = neg_inf();
    if (j < K) {
      at[s] = slot_token(a.index[o * a.i_strides[0] + i * a.i_strides[1] + j * a.i_strides[2]], V);
      const float t = a.teacher[o * a.t_strides[0] + i * a.t_strides[1] + j * a.t_strides[2]];
      if (at[s] >= 0) lnq[s] = t;
    }
  }
  const float inv_t = a.inv_t, c = a.c;
  RowStats st;
  st.shift = 0.0f;
  if (!a.tail) {
    float m = lnq[0], sum = 0.0f;
#pragma unroll
    for (int s = 1; s < S; ++s) m = max_nan(m, lnq[s]);
    m = warp_max<L>(m);
    const float from = m == neg_inf() ? 0.0f : m;
#pragma unroll
    for (int s = 0; s < S; ++s) sum += expf(lnq[s] - from);
    sum = warp_sum<L>(sum);
    if (m != neg_inf()) st.shift = m + logf(sum);
  }
  st.total = 0.0f;
  float bad = 0.0f;
#pragma unroll
  for (int s = 0; s < S; ++s) {
    lnq[s] -= st.shift;
    q[s] = expf(lnq[s]);
    st.total += q[s];
    if (at[s] == V) {  // no token to find
      bad = quiet_nan();
      at[s] = -1;
    }
    mass[s] = at[s] >= 0 ? q[s] : -1.0f;
  }
  st.total = warp_sum<L>(st.total);
  st.r = a.tail ? max_nan(0.0f, 1.0f - st.total) : 0.0f;
  st.total += warp_sum<L>(bad);
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncwarp();
#pragma unroll
  for (int s = 0; s < S; ++s) z[s] = at[s] >= 0 ? logit_at<T>(held, at[s]) : neg_inf();
  __syncwarp();
#pragma unroll
  for (int s = 0; s < S; ++s)
    if (at[s] >= 0) put_slot(held, at[s], s * L + lane);
  __syncwarp();
  bool other = false;
#pragma unroll
  for (int s = 0; s < S; ++s) other |= at[s] >= 0 && get_slot(held, at[s]) != s * L + lane;
  const unsigned others = __ballot_sync(0xffffffffu, other);  // and all have read
  const unsigned mine = (L == 32 ? 0xffffffffu : (1u << L) - 1) << (threadIdx.x & 31) / L * L;
  st.repeated = others & mine ? 1.0f : 0.0f;
#pragma unroll
  for (int s = 0; s < S; ++s)
    if (at[s] >= 0) logit_put(held, at[s], neg_inf());
  __syncwarp();
  if (others != 0) {  // in a row of the warp: masses to the first slot of each token
    float sums[S];
#pragma unroll
    for (int s = 0; s < S; ++s) {
      sums[s] = 0.0f;
      bool first = at[s] >= 0;
#pragma unroll
      for (int t = 0; t < S; ++t)
#pragma unroll 1
        for (int k = 0; k < L; ++k) {
          const int other_at = __shfl_sync(0xffffffffu, at[t], k, L);
          const float other_q = __shfl_sync(0xffffffffu, q[t], k, L);
          if (other_at != at[s]) continue;
          sums[s] += other_q;
          if (t * L + k < s * L + lane) first = false;
        }
      if (!first) sums[s] = -1.0f;
    }
#pragma unroll
    for (int s = 0; s < S; ++s) mass[s] = sums[s];
  }
  float zs[S];
  int distinct = 0;
#pragma unroll
  for (int s = 0; s < S; ++s) {
    const bool own = !(mass[s] < 0.0f);
    zs[s] = own ? z[s] : neg_inf();
    distinct += own ? 1 : 0;
  }
  if (K >= V && a.tail) {  // where every token is listed there is no other class
    if (warp_sum<L>(static_cast<float>(distinct)) >= static_cast<float>(V)) st.r = 0.0f;
  }

  float xs[kN];
#pragma unroll
  for (int u = 0; u < kVecs; ++u) {
    const int v = u * L + lane;
    float part[kV];
    unpack(v < span.vecs ? hvec[v] : void_vec<T>(), part);
#pragma unroll
    for (int e = 0; e < kV; ++e) xs[u * kV + e] = part[e];
  }
#pragma unroll
  for (int e = 0; e < kEnds; ++e) xs[E + e] = end[e] >= 0 ? logit_at<T>(held, end[e]) : neg_inf();
  SoftState rest = soft_of_lanes<false, L>(xs, c), top = soft_of_lanes<false, L>(zs, c);
  const SoftState all = soft_merge(rest, top, c);
  st.m = all.m;
  st.ln_s = all.m == neg_inf() ? neg_inf() : logf(all.s);
  st.rest_m = rest.m;
  st.ln_rest = rest.m == neg_inf() ? neg_inf() : logf(rest.s);
  settle_rest(st, inv_t);
  const float loss = row_loss<L>(st, inv_t, [&](auto f) {
#pragma unroll
    for (int s = 0; s < S; ++s) f(lnq[s], q[s], z[s]);
  });
  const bool counts = w != 0.0f;  // a row of weight 0: zeros, whatever it holds
  if (lane == 0 && live) {
    a.loss[row] = counts ? w * loss : 0.0f;
    if (a.stats != nullptr)
      *reinterpret_cast<RowStats*>(a.stats + kStats * static_cast<int64_t>(row)) = st;
  }
  if (a.dlogits == nullptr) return;

  T* d = static_cast<T*>(a.dlogits) + o * a.d_strides[0] + i * a.d_strides[1];
  const RowGradient g = row_gradient(st, a.tail, inv_t, w);
  const bool zero = g.none || !counts;
  const RowMap f = g.unlisted(c);
  T* out = d + span.head;
  const bool aligned = (reinterpret_cast<uintptr_t>(out) & 15u) == 0;
  if (live) {
#pragma unroll
    for (int e = 0; e < kEnds; ++e)
      if (end[e] >= 0) logit_put(d, end[e], zero ? 0.0f : f.plain(xs[E + e]));
#pragma unroll
    for (int u = 0; u < kVecs; ++u) {
      const int v = u * L + lane;
      if (v >= span.vecs) continue;
      float ds[kV];
#pragma unroll
      for (int e = 0; e < kV; ++e) ds[e] = zero ? 0.0f : f.plain(xs[u * kV + e]);
      if (aligned) {
        store_vec(out + v * kV, ds);
      } else {
#pragma unroll
        for (int e = 0; e < kV; ++e) logit_put(out, v * kV + e, ds[e]);
      }
    }
  }
  __syncwarp();
  if (!live || zero) return;
#pragma unroll
  for (int s = 0; s < S; ++s)
    if (!(mass[s] < 0.0f)) logit_put(d, at[s], g.listed(z[s], mass[s], c));
}

// ------------------------------------------------------------------ the list of a longer row
struct RowShared {
  SoftState top;  // softmax state of the listed tokens
  float total, r, shift;
  int pad[2];
};
struct List {   // arrays of list_room(K)
  int* index;   // -1: empty slot; V: a token past the vocabulary
  float* lnq;
  float* q;
  float* z;     // the student's logit
  float* mass;  // q summed over the slots of the same token; below 0: not its first slot
};
__host__ __device__ constexpr int list_room(int K) { return (K + 31) / 32 * 32; }
__host__ __device__ constexpr size_t list_bytes(int K) {
  return 5 * sizeof(float) * static_cast<size_t>(list_room(K));
}
__device__ __forceinline__ List list_at(uint8_t* p, int K) {
  float* f = reinterpret_cast<float*>(p);
  const int room = list_room(K);
  return {reinterpret_cast<int*>(f), f + room, f + 2 * room, f + 3 * room, f + 4 * room};
}

// q, the masses and the totals of the list in shared memory (one warp).
__device__ __forceinline__ void list_masses(RowShared& sh, const List& l, int K, int V, int tail, int lane) {
  float m = neg_inf(), shift = 0.0f, total = 0.0f;
  if (!tail) {
    for (int j = lane; j < K; j += 32) m = max_nan(m, l.lnq[j]);
    m = warp_max(m);
    if (m != neg_inf()) {
      float s = 0.0f;
      for (int j = lane; j < K; j += 32) s += expf(l.lnq[j] - m);
      shift = m + logf(warp_sum(s));
    }
  }
  bool bad = false;
  for (int j = lane; j < K; j += 32) {
    const int at = l.index[j];
    const float lq = l.lnq[j] - shift, q = expf(lq);
    l.lnq[j] = lq;
    l.q[j] = q;
    l.mass[j] = at >= 0 && at < V ? q : -1.0f;
    total += q;
    bad |= at == V;
  }
  total = warp_sum(total);
  bad = __any_sync(0xffffffffu, bad);
  if (lane == 0) {
    sh.total = bad ? quiet_nan() : total;  // a token past the vocabulary: NaN throughout
    sh.r = tail ? max_nan(0.0f, 1.0f - total) : 0.0f;
    sh.shift = shift;
  }
}
// The listed tokens' softmax state (one warp); with `repeated`, of each token's first slot, to which
// the masses of the others go.
__device__ __forceinline__ void list_state(RowShared& sh, const List& l, int K, int V, int lane, float c,
                                           bool repeated) {
  float zs[kTopMax / 32];
#pragma unroll
  for (int s = 0; s < kTopMax / 32; ++s) {
    const int j = s * 32 + lane;
    zs[s] = neg_inf();
    if (j >= K) continue;
    const int at = l.index[j];
    bool first = at >= 0 && at < V;
    if (repeated && first) {
      float mass = 0.0f;
      for (int k = 0; k < K; ++k)
        if (l.index[k] == at) {
          mass += l.q[k];
          if (k < j) first = false;
        }
      l.mass[j] = first ? mass : -1.0f;
    }
    if (first) zs[s] = l.z[j];
  }
  const SoftState top = soft_of_lanes<false, 32>(zs, c);
  if (lane == 0) sh.top = top;
}
// The row's statistics from the unlisted tokens' state.
__device__ __forceinline__ RowStats row_stats(const RowShared& sh, const SoftState& rest, bool repeated,
                                              float inv_t, float c) {
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
  settle_rest(st, inv_t);
  return st;
}
__device__ __forceinline__ void write_loss(const DistillTopkArgs& a, const RowStats& st, const List& l,
                                           int64_t row, float w, float inv_t, int lane) {
  const int K = static_cast<int>(a.K);
  const float loss = row_loss<32>(st, inv_t, [&](auto f) {
    for (int j = lane; j < K; j += 32) f(l.lnq[j], l.q[j], l.z[j]);
  });
  if (lane == 0) {
    a.loss[row] = w * loss;
    if (a.stats != nullptr) *reinterpret_cast<RowStats*>(a.stats + kStats * row) = st;
  }
}

// ------------------------------------------------------------------ a warp for a middling row
// Bytes of the row: its vectors, and one more each for the row's head and tail.
template <typename T>
__host__ __device__ constexpr size_t held_bytes(int64_t V) {
  return (static_cast<size_t>(V / kVec<T>) + 2) * 16;
}
__host__ __device__ constexpr size_t held_at(int K) {
  return (sizeof(RowShared) + list_bytes(K) + 15) & ~size_t(15);
}

template <typename T>
__global__ void __launch_bounds__(32 * kWarpsHeld, 10) distill_warp_kernel(DistillTopkArgs a, FastDiv inner) {
  extern __shared__ __align__(16) uint8_t smem[];
  constexpr int kV = kVec<T>;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int V = static_cast<int>(a.V), K = static_cast<int>(a.K);
  const uint32_t row32 = blockIdx.x * kWarpsHeld + warp;
  const int64_t row = row32;
  if (row >= a.outer * a.inner) return;
  int o, i;
  inner.divmod(static_cast<int>(row32), o, i);
  const T* x = static_cast<const T*>(a.logits) + o * a.l_strides[0] + i * a.l_strides[1];
  T* d = a.dlogits != nullptr
             ? static_cast<T*>(a.dlogits) + o * a.d_strides[0] + i * a.d_strides[1]
             : nullptr;
  uint8_t* base = smem + warp * (held_at(K) + held_bytes<T>(V));
  RowShared& sh = *reinterpret_cast<RowShared*>(base);
  const List l = list_at(base + sizeof(RowShared), K);
  const RowSpan span = row_span(x, V);
  const float w = row_weight<T>(a, o, i);
  T* held = reinterpret_cast<T*>(base + held_at(K)) + (kV - span.head) % kV;
  const uint4* vec = reinterpret_cast<const uint4*>(x + span.head);
  uint4* hvec = reinterpret_cast<uint4*>(held + span.head);
  for (int v = lane; v < span.vecs; v += 32)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(hvec + v)), "l"(vec + v)
                 : "memory");
  const int edge = lane < span.head               ? lane
                   : lane - span.head < span.tail ? V - span.tail + lane - span.head
                                                  : -1;
  if (edge >= 0) held[edge] = x[edge];
  for (int j = lane; j < K; j += 32) {
    const int at = slot_token(a.index[o * a.i_strides[0] + i * a.i_strides[1] + j * a.i_strides[2]], V);
    const float t = a.teacher[o * a.t_strides[0] + i * a.t_strides[1] + j * a.t_strides[2]];
    l.index[j] = at;
    l.lnq[j] = at >= 0 ? t : neg_inf();
  }
  const float inv_t = a.inv_t, c = a.c;
  asm volatile("cp.async.wait_all;" ::: "memory");
  if (w == 0.0f) {  // (the row was on its way before its weight was there)
    if (d != nullptr) map_row<T, 32>(x, d, V, lane, true, Nothing());
    if (lane == 0) a.loss[row] = 0.0f;
    return;
  }
  __syncwarp();
  auto is_token = [&](int at) { return at >= 0 && at < V; };
  for (int j = lane; j < K; j += 32) l.z[j] = is_token(l.index[j]) ? logit_at<T>(held, l.index[j]) : neg_inf();
  __syncwarp();
  for (int j = lane; j < K; j += 32)
    if (is_token(l.index[j])) put_slot(held, l.index[j], j);
  __syncwarp();
  bool repeated = false;
  for (int j = lane; j < K; j += 32)
    if (is_token(l.index[j])) repeated |= get_slot(held, l.index[j]) != j;
  repeated = __any_sync(0xffffffffu, repeated);  // and all have read
  for (int j = lane; j < K; j += 32)
    if (is_token(l.index[j])) logit_put(held, l.index[j], neg_inf());
  list_masses(sh, l, K, V, a.tail, lane);
  __syncwarp();
  list_state(sh, l, K, V, lane, c, repeated);
  __syncwarp();

  SoftSums<false> sums;
  const float slack = kBaseSlack / c;
  for (int b = 0; b < span.vecs; b += 32 * kUnroll) {
    uint4 wv[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int v = b + u * 32 + lane;
      wv[u] = v < span.vecs ? hvec[v] : void_vec<T>();
    }
    sums.template add<T>(wv, max_of(wv, T()), c, slack, 0u, batch_fill<32>(b, span.vecs, lane), [](int) {});
  }
  SoftState rest = sums.wide ? soft_slowly<T, 32>(hvec, 0, span.vecs, lane, c) : sums.state(c);
  if (edge >= 0) soft_add(rest, logit_at<T>(held, edge), c);
  rest = soft_join(rest, c);
  const RowStats st = row_stats(sh, rest, repeated, inv_t, c);
  write_loss(a, st, l, row, w, inv_t, lane);
  if (d == nullptr) return;

  const RowGradient g = row_gradient(st, a.tail, inv_t, w);
  const RowMap f = g.unlisted(c);
  T* out = d + span.head;
  if ((reinterpret_cast<uintptr_t>(out) & 15u) == 0 && !f.wide) {
    if (edge >= 0) logit_put(d, edge, g.none ? 0.0f : f(logit_at<T>(held, edge)));
    for (int v = lane; v < span.vecs; v += 32) {
      float xs[kV], ds[kV];
      unpack(hvec[v], xs);
#pragma unroll
      for (int e = 0; e < kV; ++e) ds[e] = g.none ? 0.0f : f(xs[e]);
      store_vec(out + static_cast<int64_t>(v) * kV, ds);
    }
  } else {  // x and d lie differently in their vectors
    for (int e = lane; e < V; e += 32) logit_put(d, e, g.none ? 0.0f : f.of(logit_at<T>(held, e)));
  }
  if (g.none) return;
  __syncwarp();
  for (int j = lane; j < K; j += 32)
    if (is_token(l.index[j]) && !(l.mass[j] < 0.0f))
      logit_put(d, l.index[j], g.listed(l.z[j], l.mass[j], c));
}

// ------------------------------------------------------------------ a CTA or a cluster for a long row
struct CtaShared {
  float2 part[kMaxCluster * kWarps];  // base and sum of every warp of the cluster
  int repeated[kMaxCluster];          // a token is twice in the list, and in that CTA's slice
  uint32_t edge_bits;                 // which of the row's ends are listed, a bit per element
  RowShared row;
  RowGradient gradient;
};
// The slice's bits: a byte per vector, the vectors of a thread's batch in one word.
__host__ __device__ constexpr size_t bits_at(int K) {
  return (sizeof(CtaShared) + list_bytes(K) + 15) & ~size_t(15);
}
template <typename T, int G>
__host__ __device__ constexpr int slice_batches(int64_t V, int cluster) {
  return static_cast<int>(((V / kVec<T> + cluster - 1) / cluster + G * kUnroll - 1) / (G * kUnroll));
}
static_assert(kUnroll == 4, "a batch's bytes make a word");
template <typename T, int G>
__host__ __device__ constexpr size_t cta_smem(int K, int64_t V, int cluster) {
  return bits_at(K) + static_cast<size_t>(slice_batches<T, G>(V, cluster)) * G * kUnroll;
}
static_assert(cta_smem<float, kThreads>(kTopMax, BDH_DISTILL_VOCAB_MAX, kMaxCluster) <= 128 * 1024,
              "the widest row's bits have room in the largest cluster");

// -inf in the places of a vector that the bits name.
__device__ __forceinline__ void strike(uint4& w, uint32_t bits, float) {
  if (bits & 1) w.x = 0xff800000u;
  if (bits & 2) w.y = 0xff800000u;
  if (bits & 4) w.z = 0xff800000u;
  if (bits & 8) w.w = 0xff800000u;
}
__device__ __forceinline__ uint32_t strike_pair(uint32_t w, uint32_t bits) {
  if (bits & 1) w = (w & 0xffff0000u) | 0xff80u;
  if (bits & 2) w = (w & 0xffffu) | 0xff800000u;
  return w;
}
__device__ __forceinline__ void strike(uint4& w, uint32_t bits, uint16_t) {
  w.x = strike_pair(w.x, bits);
  w.y = strike_pair(w.y, bits >> 2);
  w.z = strike_pair(w.z, bits >> 4);
  w.w = strike_pair(w.w, bits >> 6);
}

// soft_slowly with the bits' elements left out.
template <typename T, int G>
__device__ __forceinline__ SoftState soft_slowly_struck(const uint4* vec, int v0, int v1, int tid, float c,
                                                        const uint32_t* bits) {
  SoftState st = soft_empty();
  const T* x = reinterpret_cast<const T*>(vec);
#pragma unroll 1
  for (int v = v0 + tid, at = 0; v < v1; v += G, ++at)
#pragma unroll 1
    for (int e = 0; e < kVec<T>; ++e)
      if ((bits[at / kUnroll * G + tid] >> (at % kUnroll * 8 + e) & 1) == 0)
        soft_add(st, logit_at<T>(x, static_cast<int64_t>(v) * kVec<T> + e), c);
  return st;
}
// The unlisted tokens' gradients for the vectors [v0, v1), whose first batch is in `next` (not for a
// wide row).
template <typename T, int G>
__device__ __forceinline__ void write_slice(uint4 (&next)[kUnroll], const uint4* vec, T* out, int v0, int v1,
                                            int tid, uint64_t drop, const RowMap& f) {
  constexpr int kV = kVec<T>;
  const bool aligned = (reinterpret_cast<uintptr_t>(out) & 15u) == 0;
  stream_early<T, G>(next, vec, v0, v1, tid, drop, [&](const uint4 (&wv)[kUnroll], int b, auto fill,
                                                       auto refill) {
    constexpr bool kWhole = !std::is_same<decltype(fill), int>::value;
    T* to = out + static_cast<int64_t>(b + tid) * kV;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int v = b + u * G + tid;
      float xs[kV], ds[kV];
      unpack(wv[u], xs);
      refill(u);
      if (!kWhole && v >= v1) continue;
#pragma unroll
      for (int e = 0; e < kV; ++e) ds[e] = ex2(fmaf(xs[e], f.c, -f.b)) * f.k0;
      if (aligned) {
        st_global_v4_hint(to + u * G * kV, pack(ds), drop);
      } else {
#pragma unroll
        for (int e = 0; e < kV; ++e) logit_put(to, u * G * kV + e, ds[e]);
      }
    }
  });
}

// G threads stream; one warp more has the list.
template <typename T, int G>
__global__ void __launch_bounds__(G + 32, G == kThreads ? 4 : 7)
    distill_cta_kernel(DistillTopkArgs a, int C, FastDiv inner) {
  extern __shared__ __align__(16) uint8_t smem[];
  constexpr int kV = kVec<T>, kStep = G * kUnroll;
  CtaShared& sh = *reinterpret_cast<CtaShared*>(smem);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const bool lister = warp == G / 32;
  const int V = static_cast<int>(a.V), K = static_cast<int>(a.K);
  const List l = list_at(smem + sizeof(CtaShared), K);
  uint32_t* bits = reinterpret_cast<uint32_t*>(smem + bits_at(K));
  const uint32_t rank = C > 1 ? cta_rank() : 0;
  const uint32_t row32 = blockIdx.x / static_cast<uint32_t>(C);
  const int64_t row = row32;
  int o, i;
  inner.divmod(static_cast<int>(row32), o, i);
  const T* x = static_cast<const T*>(a.logits) + o * a.l_strides[0] + i * a.l_strides[1];
  T* d = a.dlogits != nullptr
             ? static_cast<T*>(a.dlogits) + o * a.d_strides[0] + i * a.d_strides[1]
             : nullptr;
  if (C > 1) cluster_arrive();  // shared memory may be written once all CTAs have started
  // This CTA's slice: vectors [v0, v1) between the row's 16-byte boundaries, the row's head with
  // the first slice and its tail with the last; n elements from `from`.
  const float w = row_weight<T>(a, o, i);
  const RowSpan span = row_span(x, V);
  const uint4* vec = reinterpret_cast<const uint4*>(x + span.head);
  const int per = (span.vecs + C - 1) / C;
  const int v0 = min(static_cast<int>(rank) * per, span.vecs), v1 = min(v0 + per, span.vecs);
  const int head = rank == 0 ? span.head : 0, tail = rank == C - 1 ? span.tail : 0;
  const int from = span.head + v0 * kV - head, n = head + (v1 - v0) * kV + tail;
  const float inv_t = a.inv_t, c = a.c;

  // The first pass's lines stay in L2 for the second, which lets go of them, as the gradient's do.
  const uint64_t drop = l2_policy_evict_first();
  const uint64_t keep = d != nullptr ? l2_policy_evict_last() : drop;

  uint4 next[kUnroll];
  int edge = -1;
  float edge_x = neg_inf();
  int slot_at[kTopMax / 32];  // the lister's slots
  if (!lister) {
    load_batch<G>(next, vec, v0, v1, tid, keep);
    edge = tid < head ? from + tid : tid - head < tail ? V - tail + tid - head : -1;
    if (edge >= 0) edge_x = logit_at<T>(x, edge);
    for (int k = tid; k < slice_batches<T, G>(V, C) * G; k += G) bits[k] = 0;
    if (tid == 0) sh.edge_bits = 0;
  } else {
#pragma unroll
    for (int s = 0; s < kTopMax / 32; ++s) {
      const int j = s * 32 + lane;
      slot_at[s] = -1;
      if (j >= K) continue;
      slot_at[s] = slot_token(a.index[o * a.i_strides[0] + i * a.i_strides[1] + j * a.i_strides[2]], V);
      const float t = a.teacher[o * a.t_strides[0] + i * a.t_strides[1] + j * a.t_strides[2]];
      l.index[j] = slot_at[s];
      l.lnq[j] = slot_at[s] >= 0 ? t : neg_inf();
    }
  }
  if (w == 0.0f) {  // the whole cluster; a batch of the row was on its way
    if (!lister && d != nullptr)
      map_row<T, G>(x + from, d + from, n, tid, true, Nothing());
    if (tid == 0 && rank == 0) a.loss[row] = 0.0f;
    if (C > 1) cluster_wait();
    return;
  }
  __syncthreads();
  auto in_slice = [&](int at) { return at >= from && at < from + n; };  // (and below V)
  if (lister) {
    bool repeated = false;
#pragma unroll
    for (int s = 0; s < kTopMax / 32; ++s) {
      const int at = slot_at[s];
      if (!in_slice(at)) continue;
      const int e = at - from - head, v = e >= 0 ? e / kV : -1;
      uint32_t bit, before;
      if (e < 0 || v >= v1 - v0) {  // an end: bits as the threads that hold them
        bit = 1u << (e < 0 ? at - from : head + at - (V - tail));
        before = atomicOr(&sh.edge_bits, bit);
      } else {
        const int in_batch = v % kStep;
        bit = 1u << (in_batch / G * 8 + e % kV);
        before = atomicOr(&bits[v / kStep * G + in_batch % G], bit);
      }
      repeated |= (before & bit) != 0;
    }
    __syncthreads();  // the bits are set
    // While the others stream: the list; then, of all, the row's statistics and what the gradient needs.
#pragma unroll
    for (int s = 0; s < kTopMax / 32; ++s) {
      const int at = slot_at[s];
      if (s * 32 + lane < K) l.z[s * 32 + lane] = at >= 0 && at < V ? logit_at<T>(x, at) : neg_inf();
    }
    repeated = __any_sync(0xffffffffu, repeated);
    list_masses(sh.row, l, K, V, a.tail, lane);
    __syncwarp();
    list_state(sh.row, l, K, V, lane, c, false);
    if (C > 1) {
      cluster_wait();
      if (lane < C) peer_store(peer_smem(&sh.repeated[rank], lane), __int_as_float(repeated ? 1 : 0));
      cluster_arrive();
      cluster_wait();
    } else {
      if (lane == 0) sh.repeated[0] = repeated ? 1 : 0;
      __syncthreads();
    }
    repeated = __any_sync(0xffffffffu, lane < C && sh.repeated[lane] != 0);
    if (repeated) list_state(sh.row, l, K, V, lane, c, true);  // in every CTA of the cluster
    SoftState rest = soft_empty();
    for (int k = lane; k < C * (G / 32); k += 32)
      rest = soft_merge(rest, {sh.part[k].x, sh.part[k].y, 0.0f}, c);
    rest = soft_join(rest, c);
    __syncwarp();
    const RowStats st = row_stats(sh.row, rest, repeated, inv_t, c);
    const RowGradient g = row_gradient(st, a.tail, inv_t, w);
    if (d != nullptr) {
      if (lane == 0) sh.gradient = g;
      __syncthreads();
    }
    if (rank == 0) write_loss(a, st, l, row, w, inv_t, lane);
    if (d == nullptr || g.none) return;
    __syncthreads();  // the unlisted tokens' gradients are written
    for (int j = lane; j < K; j += 32)
      if (in_slice(l.index[j]) && !(l.mass[j] < 0.0f))
        logit_put(d, l.index[j], g.listed(l.z[j], l.mass[j], c));
    return;
  }

  __syncthreads();  // the bits are set
  SoftSums<false> sums;
  const float slack = kBaseSlack / c;
  const uint32_t* my_bits = bits + tid;
  stream_early<T, G>(next, vec, v0, v1, tid, keep, [&](uint4 (&wv)[kUnroll], int, auto fill,
                                                              auto refill) {
    const uint32_t struck = *my_bits;
    my_bits += G;
    if (struck != 0) {
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (struck >> 8 * u & 0xff) strike(wv[u], struck >> 8 * u, T());
    }
    sums.template add<T>(wv, max_of(wv, T()), c, slack, 0u, fill, refill);
  });
  if (d != nullptr) load_batch<G>(next, vec, v0, v1, tid, drop);  // again, for the gradient
  SoftState rest = soft_empty();
  if (!sums.wide) rest = sums.state(c);
  else rest = soft_slowly_struck<T, G>(vec, v0, v1, tid, c, bits);
  if (edge >= 0 && (sh.edge_bits >> tid & 1) == 0) soft_add(rest, edge_x, c);
  {
    const float m = warp_max(rest.m);
    if (m != neg_inf()) soft_raise(rest, m, c);
    rest.s = warp_sum(rest.s);
  }
  if (C > 1) {  // every warp's state to every CTA of the cluster
    cluster_wait();
    if (lane < C) {
      const uint32_t to = peer_smem(&sh.part[rank * (G / 32) + warp], lane);
      peer_store(to, rest.m);
      peer_store(to + 4, rest.s);
    }
    cluster_arrive();
    cluster_wait();
  } else {
    if (lane == 0) sh.part[warp] = make_float2(rest.m, rest.s);
    __syncthreads();
  }
  if (d == nullptr) return;
  __syncthreads();
  const RowGradient& g = sh.gradient;
  const bool none = g.none;
  const RowMap f = g.unlisted(c);
  if (edge >= 0) logit_put(d, edge, none ? 0.0f : f.of(edge_x));
  if (f.wide || none) {
    map_row<T, G>(x + from + head, d + from + head, n - head - tail, tid, none, f);
  } else {
    write_slice<T, G>(next, vec, d + span.head, v0, v1, tid, drop, f);
  }
  if (!none) __syncthreads();
}

// --------------------------------------------------- the gradient from the forward's statistics
template <typename T, int G>
__global__ void __launch_bounds__(kThreads) distill_topk_bwd_kernel(DistillTopkArgs a, FastDiv pieces,
                                                                    int piece, FastDiv inner) {
  const int tid = threadIdx.x % G, group = threadIdx.x / G;
  const int V = static_cast<int>(a.V), K = static_cast<int>(a.K);
  int row32, nth, o, i;
  pieces.divmod(static_cast<int>(blockIdx.x * (kThreads / G) + group), row32, nth);
  const int64_t row = row32;
  if (row >= a.outer * a.inner) return;  // whole warps of the warp form
  inner.divmod(row32, o, i);
  const int from = nth * piece;
  const int n = min(piece, V - from);
  const T* x = static_cast<const T*>(a.logits) + o * a.l_strides[0] + i * a.l_strides[1];
  T* d = static_cast<T*>(a.dlogits) + o * a.d_strides[0] + i * a.d_strides[1];
  const float w = row_weight<T>(a, o, i);
  if (w == 0.0f) {
    map_row<T, G>(x + from, d + from, n, tid, true, Nothing());
    return;
  }
  const float inv_t = a.inv_t, c = a.c;
  const RowStats st = *reinterpret_cast<const RowStats*>(a.stats + kStats * row);
  const float up = a.g_loss.p[o * a.g_loss.strides[0] + i * a.g_loss.strides[1]];
  const RowGradient g = row_gradient(st, a.tail, inv_t, w * up);
  map_row<T, G>(x + from, d + from, n, tid, g.none, g.unlisted(c));
  if (g.none) return;
  if (G <= 32) __syncwarp();
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
    logit_put(d, at, g.listed(logit_at<T>(x, at), mass, c));
  }
}

template <typename T, int L, int E, int S>
int launch_short(const DistillTopkArgs& a, const FastDiv& inner, cudaStream_t stream) {
  constexpr int kRows = kThreads / L;
  const unsigned grid = static_cast<unsigned>((a.outer * a.inner + kRows - 1) / kRows);
  distill_short_kernel<T, L, E, S><<<grid, kThreads, 0, stream>>>(a, inner);
  return cuda_status("distill_topk launch");
}

int allow_smem(const void* kern, size_t smem) {
  return allow_shared_memory("distill_topk shared memory", kern, smem);
}

template <typename T, int G>
int launch_cta(const DistillTopkArgs& a, int cluster, const FastDiv& inner, cudaStream_t stream) {
  const int64_t rows = a.outer * a.inner;
  const size_t smem = cta_smem<T, G>(static_cast<int>(a.K), a.V, cluster);
  auto* kern = distill_cta_kernel<T, G>;
  if (int rc = allow_smem(reinterpret_cast<const void*>(kern), smem)) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(rows * cluster));
  cfg.blockDim = dim3(G + 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 1 : 0;
  return cuda_status("distill_topk launch", cudaLaunchKernelEx(&cfg, kern, a, cluster, inner));
}

template <typename T>
int forward_by_size(const DistillTopkArgs& a, cudaStream_t stream) {
  const FastDiv inner(static_cast<uint32_t>(a.inner));
  if (a.V <= 256 && a.K <= 16) return launch_short<T, 8, 32, 2>(a, inner, stream);
  if (a.V <= 512 && a.K <= 32) return launch_short<T, 16, 32, 2>(a, inner, stream);
  if (a.V <= kShort && a.K <= 32) return launch_short<T, 32, 32, 1>(a, inner, stream);
  // (16384 rows of 256 with K = 64: 16 us, held in shared memory as a longer row 22; 64 rows 3.3 and 4.7)
  if (a.V <= kShort && a.K <= 64) return launch_short<T, 32, 32, 2>(a, inner, stream);
  if (a.V <= kShort) return launch_short<T, 32, 32, 4>(a, inner, stream);
  int dev = 0;
  cudaGetDevice(&dev);
  const int K = static_cast<int>(a.K);
  const int64_t rows = a.outer * a.inner, bytes = a.V * static_cast<int64_t>(sizeof(T));
  if (bytes <= kWarpRowBytes && rows >= kWarpRows * sm_count(dev)) {
    const size_t smem = kWarpsHeld * (held_at(K) + held_bytes<T>(a.V));
    if (int rc = allow_smem(reinterpret_cast<const void*>(distill_warp_kernel<T>), smem)) return rc;
    distill_warp_kernel<T><<<static_cast<unsigned>((rows + kWarpsHeld - 1) / kWarpsHeld), 32 * kWarpsHeld, smem,
                             stream>>>(a, inner);
    return cuda_status("distill_topk launch");
  }
  int cluster = 1;
  // (a loss alone is split for its bits' room from some 900 thousand tokens in fp32 or 1.8 million in bf16)
  const size_t most = static_cast<size_t>(shared_memory_limit(dev));
  while (cluster < kMaxCluster &&
         (cta_smem<T, kThreads>(K, a.V, cluster) > most ||
          (a.dlogits != nullptr && bytes > static_cast<int64_t>(cluster) * kSliceBytes) ||
          (2 * rows * cluster <= 3 * sm_count(dev) && bytes >= cluster * int64_t(32768))))
    cluster *= 2;
  if (rows * cluster >= int64_t(1) << 31) {
    set_error("distill_topk: too many rows for this vocabulary");
    return BDH_ERR_INVALID;
  }
  if (cluster == 1 && bytes <= (a.dlogits != nullptr ? kHalfGradBytes : kHalfBytes))
    return launch_cta<T, kThreads / 2>(a, 1, inner, stream);
  return launch_cta<T, kThreads>(a, cluster, inner, stream);
}

template <typename T, int G>
int launch_backward(const DistillTopkArgs& a, int64_t pieces, int piece, cudaStream_t stream) {
  constexpr int kGroups = kThreads / G;
  const int64_t grid = (a.outer * a.inner * pieces + kGroups - 1) / kGroups;
  if (grid * kGroups >= int64_t(1) << 31) {
    set_error("distill_topk_bwd: too many rows for this vocabulary");
    return BDH_ERR_INVALID;
  }
  distill_topk_bwd_kernel<T, G><<<static_cast<unsigned>(grid), kThreads, 0, stream>>>(
      a, FastDiv(static_cast<uint32_t>(pieces)), piece, FastDiv(static_cast<uint32_t>(a.inner)));
  return cuda_status("distill_topk_bwd launch");
}

template <typename T>
int backward_by_size(const DistillTopkArgs& a, cudaStream_t stream) {
  const int64_t rows = a.outer * a.inner, bytes = a.V * static_cast<int64_t>(sizeof(T));
  int dev = 0;
  cudaGetDevice(&dev);
  if (a.V <= 256) return launch_backward<T, 8>(a, 1, 256, stream);
  if (a.V <= 512) return launch_backward<T, 16>(a, 1, 512, stream);
  if (a.V <= kShort) return launch_backward<T, 32>(a, 1, kShort, stream);
  if (bytes <= kWarpGradBytes && rows >= kWarpRows * sm_count(dev))
    return launch_backward<T, 32>(a, 1, static_cast<int>(a.V), stream);
  return launch_backward<T, kThreads>(a, (a.V + kPiece - 1) / kPiece, kPiece, stream);
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
