// Log probabilities of given tokens with entropy and top alternatives, and their gradient:
//
//   z = x / temperature, lse = ln sum_i exp(z_i), logprob = z[token] - lse,
//   entropy = - sum_i p_i ln p_i, and the K largest logits' (z_i - lse, i)
//   dx_i = 1/temperature [ p_i (g_lse - g_logprob - sum_j g_top_j - g_entropy (ln p_i + entropy))
//                          + [i = token] g_logprob + sum_j [i = top_j] g_top_j ]
//
// One CTA per row; the row's softmax state in one pass (logits.cuh), the top list by K rounds of
// "the largest below the last one" over the row.
#include <string>

#include "bdh_sm100.h"
#include "internal.h"
#include "logits.cuh"
#include "tma_host.h"

namespace bdh {

namespace {

constexpr int kThreads = 256;

struct Shared {
  SoftState part[kThreads / 32];
  uint64_t key[kThreads / 32];
};

__device__ __forceinline__ uint64_t warp_max_key(uint64_t k) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const uint64_t other = __shfl_xor_sync(0xffffffffu, k, o);
    k = other > k ? other : k;
  }
  return k;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) token_logprobs_kernel(TokenLogprobsArgs a, RowLayout ll,
                                                                  RowLayout tl) {
  __shared__ Shared sh;
  const int64_t row = blockIdx.x;
  const int64_t o = row / a.inner, i = row - o * a.inner;
  const T* x = static_cast<const T*>(a.logits) + ll.at(o, i);
  const int V = static_cast<int>(a.V);
  const float inv_t = 1.0f / a.temperature, c = kLog2e * inv_t;
  SoftState st = soft_empty();
  for (int v = threadIdx.x; v < V; v += kThreads) soft_add(st, logit_at<T>(x, v), c);
  st = soft_warp(st, c);
  if ((threadIdx.x & 31) == 0) sh.part[threadIdx.x >> 5] = st;
  __syncthreads();
  st = sh.part[0];
  for (int w = 1; w < kThreads / 32; ++w) st = soft_merge(st, sh.part[w], c);
  const bool none = st.m == neg_inf();  // nothing finite in the row
  const float ln_s = none ? neg_inf() : logf(st.s);
  if (threadIdx.x == 0) {
    if (a.lse != nullptr) a.lse[row] = none ? neg_inf() : fmaf(st.m, inv_t, ln_s);
    if (a.entropy != nullptr) a.entropy[row] = none ? 0.0f : ln_s - kLn2 * st.a / st.s;
    if (a.stats != nullptr) {
      a.stats[2 * row] = st.m;
      a.stats[2 * row + 1] = ln_s;
    }
    if (a.tokens != nullptr && a.logprob != nullptr) {
      const int64_t tok = a.tokens[tl.at(o, i)];
      float lp = quiet_nan();
      if (tok == a.ignore_index) lp = 0.0f;
      else if (tok >= 0 && tok < V) lp = none ? neg_inf() : (logit_at<T>(x, tok) - st.m) * inv_t - ln_s;
      a.logprob[row] = lp;
    }
  }
  uint64_t last = ~0ull;
  for (int k = 0; k < a.K; ++k) {
    uint64_t best = 0;
    for (int v = threadIdx.x; v < V; v += kThreads) {
      const uint64_t key = top_key(logit_at<T>(x, v), v);
      if (key < last && key > best) best = key;
    }
    best = warp_max_key(best);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh.key[threadIdx.x >> 5] = best;
    __syncthreads();
    for (int w = 0; w < kThreads / 32; ++w) best = sh.key[w] > best ? sh.key[w] : best;
    last = best;
    if (threadIdx.x == 0) {
      const uint32_t at = key_index(best);
      if (a.top_index != nullptr) a.top_index[row * a.K + k] = at;
      if (a.top_logprob != nullptr)
        a.top_logprob[row * a.K + k] =
            none ? neg_inf() : (logit_at<T>(x, at) - st.m) * inv_t - ln_s;
    }
  }
}

struct GradShared {
  int index[kTopMax + 1];
  float add[kTopMax + 1];
};

template <typename T>
__global__ void __launch_bounds__(kThreads) token_logprobs_bwd_kernel(TokenLogprobsBwdArgs a) {
  __shared__ GradShared sh;
  const int64_t row = blockIdx.x;
  const int64_t o = row / a.f.inner, i = row - o * a.f.inner;
  const RowLayout ll = {a.f.l_strides[0], a.f.l_strides[1]}, dl = {a.d_strides[0], a.d_strides[1]};
  const T* x = static_cast<const T*>(a.f.logits) + ll.at(o, i);
  T* d = static_cast<T*>(a.dlogits) + dl.at(o, i);
  const int V = static_cast<int>(a.f.V), K = a.g_top != nullptr ? static_cast<int>(a.f.K) : 0;
  const float inv_t = 1.0f / a.f.temperature;
  const float m = a.f.stats[2 * row], ln_s = a.f.stats[2 * row + 1];
  auto up = [&](const RowGrad& g) {
    return g.p != nullptr ? g.p[o * g.strides[0] + i * g.strides[1]] : 0.0f;
  };
  float g_tok = up(a.g_logprob);
  const float g_ent = up(a.g_entropy);
  const float ent = a.g_entropy.p != nullptr ? a.f.entropy[row] : 0.0f;
  float sum = up(a.g_lse);
  int64_t tok = -1;
  if (a.g_logprob.p != nullptr && a.f.tokens != nullptr) {
    tok = a.f.tokens[o * a.f.t_strides[0] + i * a.f.t_strides[1]];
    if (tok == a.f.ignore_index) {
      tok = -1;
      g_tok = 0.0f;
    } else if (tok < 0 || tok >= V) {  // no such token: its log probability is NaN, and so is this
      tok = -1;
      sum = quiet_nan();
    }
  } else {
    g_tok = 0.0f;
  }
  sum -= g_tok;
  for (int k = 0; k < K; ++k) sum -= a.g_top[row * K + k];
  for (int k = threadIdx.x; k <= K; k += kThreads) {
    sh.index[k] = k == 0 ? static_cast<int>(tok) : static_cast<int>(a.f.top_index[row * K + k - 1]);
    sh.add[k] = k == 0 ? g_tok : a.g_top[row * K + k - 1];
  }
  __syncthreads();
  const bool none = m == neg_inf();
  auto dense = [&](float v) {
    const float t = (v - m) * inv_t - ln_s;
    const float p = ex2(t * kLog2e);
    return p * (sum - g_ent * (max_nan(t, kExpFloor) + ent));
  };
  for (int v = threadIdx.x; v < V; v += kThreads)
    logit_put(d, v, none ? 0.0f : dense(logit_at<T>(x, v)) * inv_t);
  __syncthreads();
  for (int k = threadIdx.x; k <= K; k += kThreads) {
    const int at = sh.index[k];
    bool mine = at >= 0 && at < V && !none;
    float add = sh.add[k];
    for (int j = 0; mine && j <= K; ++j)
      if (j != k && sh.index[j] == at) {
        mine = j > k;
        add += sh.add[j];
      }
    if (mine) logit_put(d, at, (dense(logit_at<T>(x, at)) + add) * inv_t);
  }
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

int launch_token_logprobs(const TokenLogprobsArgs& a, cudaStream_t stream) {
  const unsigned rows = static_cast<unsigned>(a.outer * a.inner);
  if (rows == 0) return BDH_OK;
  const RowLayout ll = {a.l_strides[0], a.l_strides[1]}, tl = {a.t_strides[0], a.t_strides[1]};
  if (a.dtype == BDH_DTYPE_F32)
    token_logprobs_kernel<float><<<rows, kThreads, 0, stream>>>(a, ll, tl);
  else
    token_logprobs_kernel<uint16_t><<<rows, kThreads, 0, stream>>>(a, ll, tl);
  return launch_check("token_logprobs launch");
}

int launch_token_logprobs_bwd(const TokenLogprobsBwdArgs& a, cudaStream_t stream) {
  const unsigned rows = static_cast<unsigned>(a.f.outer * a.f.inner);
  if (rows == 0) return BDH_OK;
  if (a.f.dtype == BDH_DTYPE_F32)
    token_logprobs_bwd_kernel<float><<<rows, kThreads, 0, stream>>>(a);
  else
    token_logprobs_bwd_kernel<uint16_t><<<rows, kThreads, 0, stream>>>(a);
  return launch_check("token_logprobs_bwd launch");
}

}  // namespace bdh
