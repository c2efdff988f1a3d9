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
// nearly everything.
#include <string>

#include "bdh_sm100.h"
#include "internal.h"
#include "logits.cuh"
#include "tma_host.h"

namespace bdh {

namespace {

constexpr int kThreads = 256;
static_assert(kThreads >= kTopMax, "one thread per slot");

struct Shared {
  SoftState part[kThreads / 32];
  int index[kTopMax];  // -1: empty slot
  float lnq[kTopMax], q[kTopMax], z[kTopMax];
  float mass[kTopMax];  // q summed over the slots of the same token
  int owner[kTopMax];   // 1: the first slot of its token
  float row[4];         // total mass, r, list covers the vocabulary, bad index
};

// The row's list into shared memory: q, the total mass, r. All threads; ends in a barrier.
template <typename T>
__device__ void load_list(const DistillTopkArgs& a, const T* x, int64_t o, int64_t i, Shared& sh) {
  const int K = static_cast<int>(a.K), V = static_cast<int>(a.V), j = threadIdx.x;
  if (j < K) {
    const int64_t at = a.index[o * a.i_strides[0] + i * a.i_strides[1] + j * a.i_strides[2]];
    const float t = a.teacher[o * a.t_strides[0] + i * a.t_strides[1] + j * a.t_strides[2]];
    // a slot of probability 0 still names a listed token; past the vocabulary: V, and a bad row
    sh.index[j] = at < 0 ? -1 : at < V ? static_cast<int>(at) : V;
    sh.lnq[j] = at < 0 ? neg_inf() : t;
    sh.z[j] = at >= 0 && at < V ? logit_at<T>(x, at) : neg_inf();
  }
  __syncthreads();
  if (threadIdx.x < 32) {  // the list's softmax by the first warp
    float m = neg_inf();
    for (int k = threadIdx.x; k < K; k += 32) m = max_nan(m, sh.lnq[k]);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, d));
    float shift = 0.0f;
    if (!a.tail && m != neg_inf()) {
      float s = 0.0f;
      for (int k = threadIdx.x; k < K; k += 32) s += expf(sh.lnq[k] - m);
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
      shift = m + logf(s);
    }
    float total = 0.0f, bad = 0.0f;
    for (int k = threadIdx.x; k < K; k += 32) {
      const float l = sh.lnq[k] - shift, q = expf(l);
      sh.lnq[k] = l;
      sh.q[k] = q;
      total += q;
      if (sh.index[k] == V) bad = 1.0f;
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
      total += __shfl_xor_sync(0xffffffffu, total, d);
      bad += __shfl_xor_sync(0xffffffffu, bad, d);
    }
    if (threadIdx.x == 0) {
      sh.row[0] = total;
      sh.row[1] = a.tail ? max_nan(0.0f, 1.0f - total) : 0.0f;
      sh.row[3] = bad;
    }
  }
  __syncthreads();
  bool first = false;
  if (j < K && sh.index[j] >= 0) {
    first = true;
    float mass = 0.0f;
    for (int k = 0; k < K; ++k)
      if (sh.index[k] == sh.index[j]) {
        if (k < j) first = false;
        mass += sh.q[k];
      }
    sh.mass[j] = mass;
  }
  if (j < K) sh.owner[j] = first ? 1 : 0;
  const int distinct = __syncthreads_count(first ? 1 : 0);
  if (threadIdx.x == 0) {
    if (distinct >= V) sh.row[1] = 0.0f;  // every token is listed: there is no other class
    if (sh.row[3] > 0.0f) sh.row[0] = quiet_nan();  // a token past the vocabulary: NaN throughout
  }
  __syncthreads();
}

// dx of the row from its four stored figures: m, ln s of all tokens and of the unlisted ones.
template <typename T>
__device__ void write_grad(const DistillTopkArgs& a, const T* x, T* d, Shared& sh, float m,
                           float ln_s, float m_rest, float ln_rest, float scale) {
  const int V = static_cast<int>(a.V), K = static_cast<int>(a.K);
  const float inv_t = 1.0f / a.temperature;
  const float total = sh.row[0] + sh.row[1], r = sh.row[1];
  // unlisted tokens: p_i (total - r / s) = (p_i / s) (total s - r), with s as small as it comes
  const float s = a.tail ? expf((m_rest - m) * inv_t + ln_rest - ln_s) : 1.0f;
  const float base_m = a.tail ? m_rest : m, base_l = a.tail ? ln_rest : ln_s;
  const float coef = scale * inv_t * (a.tail ? total * s - r : total);
  const bool none = m == neg_inf(), rest_none = base_m == neg_inf();
  for (int v = threadIdx.x; v < V; v += kThreads) {
    const float p = rest_none ? 0.0f : ex2(((logit_at<T>(x, v) - base_m) * inv_t - base_l) * kLog2e);
    logit_put(d, v, none ? 0.0f : p * coef);
  }
  __syncthreads();
  const int j = threadIdx.x;
  if (j < K && sh.owner[j] && sh.index[j] < V && !none) {
    const float p = ex2(((sh.z[j] - m) * inv_t - ln_s) * kLog2e);
    logit_put(d, sh.index[j], scale * inv_t * (p * total - sh.mass[j]));
  }
}

template <typename T>
__device__ void zero_row(T* d, int V) {
  for (int v = threadIdx.x; v < V; v += kThreads) logit_put(d, v, 0.0f);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) distill_topk_kernel(DistillTopkArgs a) {
  __shared__ Shared sh;
  const int64_t row = blockIdx.x;
  const int64_t o = row / a.inner, i = row - o * a.inner;
  const T* x = static_cast<const T*>(a.logits) + o * a.l_strides[0] + i * a.l_strides[1];
  T* d = a.dlogits != nullptr
             ? static_cast<T*>(a.dlogits) + o * a.d_strides[0] + i * a.d_strides[1]
             : nullptr;
  const int V = static_cast<int>(a.V), K = static_cast<int>(a.K);
  const float w = a.weight.p != nullptr
                      ? a.weight.p[o * a.weight.strides[0] + i * a.weight.strides[1]]
                      : 1.0f;
  if (w == 0.0f) {
    if (d != nullptr) zero_row(d, V);
    if (threadIdx.x == 0) a.loss[row] = 0.0f;
    return;
  }
  load_list(a, x, o, i, sh);
  const float inv_t = 1.0f / a.temperature, c = kLog2e * inv_t;
  SoftState rest = soft_empty();
  for (int v = threadIdx.x; v < V; v += kThreads) {
    bool in = false;
    for (int k = 0; k < K; ++k) in |= sh.index[k] == v;
    if (!in) soft_add(rest, logit_at<T>(x, v), c);
  }
  rest = soft_warp(rest, c);
  if ((threadIdx.x & 31) == 0) sh.part[threadIdx.x >> 5] = rest;
  __syncthreads();
  rest = sh.part[0];
  for (int k = 1; k < kThreads / 32; ++k) rest = soft_merge(rest, sh.part[k], c);
  SoftState all = rest;
  for (int k = 0; k < K; ++k)
    if (sh.owner[k]) soft_add(all, sh.z[k], c);
  const bool none = all.m == neg_inf();
  const float ln_s = none ? neg_inf() : logf(all.s);
  const float ln_rest = rest.m == neg_inf() ? neg_inf() : logf(rest.s);
  if (threadIdx.x == 0) {
    float loss = 0.0f;
    for (int k = 0; k < K; ++k)
      if (sh.q[k] > 0.0f || sh.q[k] != sh.q[k]) {
        const float lp = none || sh.z[k] == neg_inf() ? neg_inf() : (sh.z[k] - all.m) * inv_t - ln_s;
        loss = fmaf(sh.q[k], sh.lnq[k] - lp, loss);
      }
    const float r = sh.row[1];
    if (r > 0.0f) {
      const float ls = rest.m == neg_inf() ? neg_inf() : (rest.m - all.m) * inv_t + ln_rest - ln_s;
      loss = fmaf(r, logf(r) - ls, loss);
    }
    a.loss[row] = w * (loss + 0.0f * sh.row[0]);
    if (a.stats != nullptr) {
      a.stats[4 * row] = all.m;
      a.stats[4 * row + 1] = ln_s;
      a.stats[4 * row + 2] = rest.m;
      a.stats[4 * row + 3] = ln_rest;
    }
  }
  if (d != nullptr) write_grad(a, x, d, sh, all.m, ln_s, rest.m, ln_rest, w);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) distill_topk_bwd_kernel(DistillTopkArgs a) {
  __shared__ Shared sh;
  const int64_t row = blockIdx.x;
  const int64_t o = row / a.inner, i = row - o * a.inner;
  const T* x = static_cast<const T*>(a.logits) + o * a.l_strides[0] + i * a.l_strides[1];
  T* d = static_cast<T*>(a.dlogits) + o * a.d_strides[0] + i * a.d_strides[1];
  const float w = a.weight.p != nullptr
                      ? a.weight.p[o * a.weight.strides[0] + i * a.weight.strides[1]]
                      : 1.0f;
  if (w == 0.0f) {
    zero_row(d, static_cast<int>(a.V));
    return;
  }
  load_list(a, x, o, i, sh);
  const float g = a.g_loss.p[o * a.g_loss.strides[0] + i * a.g_loss.strides[1]];
  const float* st = a.stats + 4 * row;
  write_grad(a, x, d, sh, st[0], st[1], st[2], st[3], w * g);
}

int launch_check(const char* what) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    set_error(std::string(what) + ": " + cudaGetErrorString(e));
    return BDH_ERR_CUDA;
  }
  return BDH_OK;
}

}  // namespace

int launch_distill_topk(const DistillTopkArgs& a, cudaStream_t stream) {
  const unsigned rows = static_cast<unsigned>(a.outer * a.inner);
  if (rows == 0) return BDH_OK;
  if (a.dtype == BDH_DTYPE_F32)
    distill_topk_kernel<float><<<rows, kThreads, 0, stream>>>(a);
  else
    distill_topk_kernel<uint16_t><<<rows, kThreads, 0, stream>>>(a);
  return launch_check("distill_topk launch");
}

int launch_distill_topk_bwd(const DistillTopkArgs& a, cudaStream_t stream) {
  const unsigned rows = static_cast<unsigned>(a.outer * a.inner);
  if (rows == 0) return BDH_OK;
  if (a.dtype == BDH_DTYPE_F32)
    distill_topk_bwd_kernel<float><<<rows, kThreads, 0, stream>>>(a);
  else
    distill_topk_bwd_kernel<uint16_t><<<rows, kThreads, 0, stream>>>(a);
  return launch_check("distill_topk_bwd launch");
}

}  // namespace bdh
