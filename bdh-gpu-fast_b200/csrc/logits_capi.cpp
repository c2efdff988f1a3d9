// extern "C" entries of the operators on logits: argument checks and the launches of
// token_logprobs.cu and distill_topk.cu. Nothing here allocates; every call is stream-ordered
// and graph-capturable.
#include <cstring>
#include <string>

#include "bdh_sm100.h"
#include "internal.h"
#include "tma_host.h"

namespace bdh {

namespace {

constexpr float kLog2eHost = 1.4426950408889634f;

int refuse(const char* what, const char* why) {
  set_error(std::string(what) + ": " + why);
  return BDH_ERR_INVALID;
}

// The checks that every entry makes; 0 when the call may go on.
int check_rows(const char* what, int dtype, int64_t outer, int64_t inner, int64_t V, int64_t K,
               float temperature) {
  if (dtype != BDH_DTYPE_F32 && dtype != BDH_DTYPE_BF16)
    return refuse(what, "dtype must be f32 or bf16");
  if (outer < 0 || inner < 0 || V < 0 || K < 0) return refuse(what, "negative size");
  const int64_t most = (int64_t(1) << 31) - 1024;  // (rows are rounded up to whole CTAs in 32 bits)
  if (V < 1 || V > (int64_t(1) << 30)) return refuse(what, "vocabulary must be 1 to 2^30 wide");
  if (outer > most || inner > most || (inner > 0 && outer > most / inner))
    return refuse(what, "at most 2^31 - 1024 rows");
  if (K > BDH_TOP_MAX) return refuse(what, "at most BDH_TOP_MAX entries in a row's list");
  if (!(temperature > 1e-30f && temperature < 1e30f))  // so that 1 / temperature has room as well
    return refuse(what, "temperature must be positive and finite");
  return BDH_OK;
}

// The bits of -2 kWide / c, cut to bf16 (twice) where the logits are: within the range of both types for
// every temperature that check_rows lets through.
uint32_t least_logit(float c, int dtype) {
  const float least = -2.0f * kWide / c;
  uint32_t bits;
  std::memcpy(&bits, &least, sizeof(bits));
  return dtype == BDH_DTYPE_F32 ? bits : (bits & 0xffff0000u) | bits >> 16;
}

RowGrad row_grad(const float* p, const int64_t strides[2]) {
  RowGrad g;
  g.p = p;
  if (p != nullptr) std::memcpy(g.strides, strides, sizeof(g.strides));
  return g;
}

}  // namespace

}  // namespace bdh

using namespace bdh;

extern "C" {

int bdh_token_logprobs(const void* logits, int dtype, const int64_t l_strides[2],
                       const int64_t* tokens, const int64_t t_strides[2], int64_t ignore_index,
                       float* logprob, float* lse, float* entropy, float* stats,
                       float* top_logprob, int64_t* top_index, int64_t outer, int64_t inner,
                       int64_t V, int64_t K, float temperature, void* stream) {
  if (int rc = check_rows("token_logprobs", dtype, outer, inner, V, K, temperature)) return rc;
  if (K > V) return refuse("token_logprobs", "the list is longer than the vocabulary");
  if (outer * inner == 0) return BDH_OK;
  if (logits == nullptr) return refuse("token_logprobs", "logits is null");
  if ((logprob == nullptr) != (tokens == nullptr))
    return refuse("token_logprobs", "tokens and logprob come together");
  if (K > 0 && (top_logprob == nullptr || top_index == nullptr))
    return refuse("token_logprobs", "the list needs top_logprob and top_index");
  TokenLogprobsArgs a;
  a.logits = logits; a.dtype = dtype;
  std::memcpy(a.l_strides, l_strides, sizeof(a.l_strides));
  a.tokens = tokens;
  if (tokens != nullptr) std::memcpy(a.t_strides, t_strides, sizeof(a.t_strides));
  a.ignore_index = ignore_index;
  a.outer = outer; a.inner = inner; a.V = V; a.K = K;
  a.inv_t = 1.0f / temperature; a.c = kLog2eHost * a.inv_t;
  a.least = least_logit(a.c, dtype);
  a.logprob = logprob; a.lse = lse; a.entropy = entropy; a.stats = stats;
  a.top_logprob = top_logprob; a.top_index = top_index;
  return launch_token_logprobs(a, static_cast<cudaStream_t>(stream));
}

int bdh_token_logprobs_bwd(const void* logits, int dtype, const int64_t l_strides[2],
                           const int64_t* tokens, const int64_t t_strides[2], int64_t ignore_index,
                           const float* stats, const float* entropy, const int64_t* top_index,
                           const float* g_logprob, const int64_t glp_strides[2],
                           const float* g_lse, const int64_t gls_strides[2],
                           const float* g_entropy, const int64_t gen_strides[2],
                           const float* g_top, void* dlogits, const int64_t d_strides[2],
                           int64_t outer, int64_t inner, int64_t V, int64_t K, float temperature,
                           void* stream) {
  if (int rc = check_rows("token_logprobs_bwd", dtype, outer, inner, V, K, temperature)) return rc;
  if (K > V) return refuse("token_logprobs_bwd", "the list is longer than the vocabulary");
  if (outer * inner == 0) return BDH_OK;
  if (logits == nullptr || dlogits == nullptr || stats == nullptr)
    return refuse("token_logprobs_bwd", "logits, stats or dlogits is null");
  if (g_entropy != nullptr && entropy == nullptr)
    return refuse("token_logprobs_bwd", "g_entropy needs the forward's entropy");
  if (g_logprob != nullptr && tokens == nullptr)
    return refuse("token_logprobs_bwd", "g_logprob needs tokens");
  if (g_top != nullptr && K > 0 && top_index == nullptr)
    return refuse("token_logprobs_bwd", "g_top needs top_index");
  TokenLogprobsBwdArgs a;
  a.f.logits = logits; a.f.dtype = dtype;
  std::memcpy(a.f.l_strides, l_strides, sizeof(a.f.l_strides));
  a.f.tokens = tokens;
  if (tokens != nullptr) std::memcpy(a.f.t_strides, t_strides, sizeof(a.f.t_strides));
  a.f.ignore_index = ignore_index;
  a.f.outer = outer; a.f.inner = inner; a.f.V = V; a.f.K = K;
  a.f.inv_t = 1.0f / temperature; a.f.c = kLog2eHost * a.f.inv_t;
  a.f.stats = const_cast<float*>(stats);
  a.f.entropy = const_cast<float*>(entropy);
  a.f.top_index = const_cast<int64_t*>(top_index);
  a.g_logprob = row_grad(g_logprob, glp_strides);
  a.g_lse = row_grad(g_lse, gls_strides);
  a.g_entropy = row_grad(g_entropy, gen_strides);
  a.g_top = g_top;
  a.dlogits = dlogits;
  std::memcpy(a.d_strides, d_strides, sizeof(a.d_strides));
  return launch_token_logprobs_bwd(a, static_cast<cudaStream_t>(stream));
}

int bdh_distill_topk(const void* logits, int dtype, const int64_t l_strides[2],
                     const int64_t* index, const int64_t i_strides[3], const float* teacher,
                     const int64_t t_strides[3], const float* weight, const int64_t w_strides[2],
                     float* loss, float* stats, void* dlogits, const int64_t d_strides[2],
                     int64_t outer, int64_t inner, int64_t V, int64_t K, float temperature,
                     int tail, void* stream) {
  if (int rc = check_rows("distill_topk", dtype, outer, inner, V, K, temperature)) return rc;
  if (K < 1) return refuse("distill_topk", "the list needs at least one slot");
  if (V > BDH_DISTILL_VOCAB_MAX)
    return refuse("distill_topk", "the vocabulary is wider than BDH_DISTILL_VOCAB_MAX");
  if (outer * inner == 0) return BDH_OK;
  if (logits == nullptr || index == nullptr || teacher == nullptr || loss == nullptr)
    return refuse("distill_topk", "logits, index, teacher or loss is null");
  DistillTopkArgs a;
  a.logits = logits; a.dtype = dtype;
  std::memcpy(a.l_strides, l_strides, sizeof(a.l_strides));
  a.index = index;
  std::memcpy(a.i_strides, i_strides, sizeof(a.i_strides));
  a.teacher = teacher;
  std::memcpy(a.t_strides, t_strides, sizeof(a.t_strides));
  a.weight = row_grad(weight, w_strides);
  a.outer = outer; a.inner = inner; a.V = V; a.K = K;
  a.inv_t = 1.0f / temperature; a.c = kLog2eHost * a.inv_t;
  a.tail = tail ? 1 : 0;
  a.loss = loss; a.stats = stats;
  a.dlogits = dlogits;
  if (dlogits != nullptr) std::memcpy(a.d_strides, d_strides, sizeof(a.d_strides));
  return launch_distill_topk(a, static_cast<cudaStream_t>(stream));
}

int bdh_distill_topk_bwd(const void* logits, int dtype, const int64_t l_strides[2],
                         const int64_t* index, const int64_t i_strides[3], const float* teacher,
                         const int64_t t_strides[3], const float* weight,
                         const int64_t w_strides[2], const float* stats, const float* g_loss,
                         const int64_t g_strides[2], void* dlogits, const int64_t d_strides[2],
                         int64_t outer, int64_t inner, int64_t V, int64_t K, float temperature,
                         int tail, void* stream) {
  if (int rc = check_rows("distill_topk_bwd", dtype, outer, inner, V, K, temperature)) return rc;
  if (K < 1) return refuse("distill_topk_bwd", "the list needs at least one slot");
  if (V > BDH_DISTILL_VOCAB_MAX)
    return refuse("distill_topk_bwd", "the vocabulary is wider than BDH_DISTILL_VOCAB_MAX");
  if (outer * inner == 0) return BDH_OK;
  if (logits == nullptr || index == nullptr || teacher == nullptr || stats == nullptr ||
      g_loss == nullptr || dlogits == nullptr)
    return refuse("distill_topk_bwd", "logits, index, teacher, stats, g_loss or dlogits is null");
  DistillTopkArgs a;
  a.logits = logits; a.dtype = dtype;
  std::memcpy(a.l_strides, l_strides, sizeof(a.l_strides));
  a.index = index;
  std::memcpy(a.i_strides, i_strides, sizeof(a.i_strides));
  a.teacher = teacher;
  std::memcpy(a.t_strides, t_strides, sizeof(a.t_strides));
  a.weight = row_grad(weight, w_strides);
  a.outer = outer; a.inner = inner; a.V = V; a.K = K;
  a.inv_t = 1.0f / temperature; a.c = kLog2eHost * a.inv_t;
  a.tail = tail ? 1 : 0;
  a.stats = const_cast<float*>(stats);
  a.g_loss = row_grad(g_loss, g_strides);
  a.dlogits = dlogits;
  std::memcpy(a.d_strides, d_strides, sizeof(a.d_strides));
  return launch_distill_topk_bwd(a, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
