// bdh_sm100_ext: the reference's native attention module for the sm_100a library.
//
// The reference binds its CUDA / CPU kernels as the PyTorch extension `bdh_cuda_ext`
// (csrc/tril_attn_bind.cpp:25-40: tril_score_v(q, k, v), tril_decode(q, k_past, v_past),
// attribute has_cuda; declarations csrc/tril_attn.h:14-23) and kernels/cuda_attn.py calls it
// (:391-414, :490-502). This module exports the same names with the same arguments, results
// and error type (RuntimeError from TORCH_CHECK) on top of the C-ABI of libbdh_sm100.so
// (include/bdh_sm100.h), plus the ops of the fused path: the analytic backward, RoPE and the
// RoPE-fused forms of the forward and the decode step.
//
// Semantics kept from the reference module: inputs are borrowed (any strides with a contiguous
// last dimension; no .contiguous() copies of the operands), outputs are fresh tensors in q's
// dtype, the launch goes to the current CUDA stream of q's device with no host sync (so the ops
// can be captured in CUDA graphs). Differences on purpose: CUDA tensors only (no CPU path: a CPU
// tensor raises), fp32 and bf16 only, and scratch memory comes from the PyTorch caching
// allocator (the library itself never allocates).
#include <ATen/EmptyTensor.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <pybind11/stl.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <cstdint>
#include <cstdlib>
#include <cstring>
#include <mutex>
#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include "bdh_sm100.h"

namespace {

// Messages are put together as std::string: streaming integers through TORCH_CHECK's message
// builder crashed this build (torch 2.11 headers, the image's g++), strings do not.
void check_rc(int rc, const char* what) {
  TORCH_CHECK(rc == 0, std::string("cuda_sm100 ") + what + " failed (code " + std::to_string(rc) +
                           "): " + bdh_last_error());
}

int dtype_code(const at::Tensor& t) {
  if (t.scalar_type() == at::kFloat) return BDH_DTYPE_F32;
  if (t.scalar_type() == at::kBFloat16) return BDH_DTYPE_BF16;
  TORCH_CHECK(false, std::string("cuda_sm100 supports float32 and bfloat16 tensors, got ") +
                         c10::toString(t.scalar_type()));
  return -1;
}

struct Strides4 {
  int64_t s[4];
  explicit Strides4(const at::Tensor& t) {
    for (int i = 0; i < 4; ++i) s[i] = t.stride(i);
  }
};

void require_cuda(std::initializer_list<const at::Tensor*> ts) {
  const at::Device dev = (*ts.begin())->device();
  for (const at::Tensor* t : ts) {
    TORCH_CHECK(t->is_cuda(), "cuda_sm100 requires CUDA tensors (no CPU fallback)");
    TORCH_CHECK(t->device() == dev, "cuda_sm100: all tensors must be on the same device");
  }
}

void* stream_of(const at::Tensor& t) {
  return reinterpret_cast<void*>(at::cuda::getCurrentCUDAStream(t.device().index()).stream());
}

// The operand itself when TMA can read it in place (16-byte aligned base, 16-byte multiple
// strides, contiguous last dimension), else a contiguous copy zero-padded on the last dimension
// to a 16-byte multiple (zeros change no dot product over that dimension).
at::Tensor tma_ready(const at::Tensor& x) {
  const int64_t esz = x.element_size();
  bool ok = x.stride(-1) == 1 && reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0;
  for (int64_t d = 0; ok && d + 1 < x.dim(); ++d)
    if (x.size(d) > 1 && (x.stride(d) * esz) % 16 != 0) ok = false;
  if (ok) return x;
  const int64_t mult = 16 / esz;
  const int64_t n = x.size(-1);
  const int64_t npad = (n + mult - 1) / mult * mult;
  std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = npad;
  at::Tensor y = at::zeros(shape, x.options());
  y.narrow(-1, 0, n).copy_(x);
  return y;
}

// "(d0, d1, ...)" of a tensor's shape, for error messages.
std::string shape_str(const at::Tensor& t) {
  std::string s = "(";
  for (int64_t d = 0; d < t.dim(); ++d) s += (d ? ", " : "") + std::to_string(t.size(d));
  return s + ")";
}

bool same_operand(const at::Tensor& a, const at::Tensor& b) {
  return a.data_ptr() == b.data_ptr() && a.sizes() == b.sizes() && a.strides() == b.strides() &&
         a.scalar_type() == b.scalar_type();
}

void check_cold_shapes(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v) {
  TORCH_CHECK(q.dim() == 4 && k.dim() == 4 && v.dim() == 4, "q, k, v must be 4D (B, H, T, D)");
  TORCH_CHECK(q.sizes() == k.sizes(), "q and k shapes must match, got ", shape_str(q), " vs ", shape_str(k));
  TORCH_CHECK(v.size(0) == q.size(0) && v.size(2) == q.size(2), "v batch/seq must match q");
  TORCH_CHECK(v.size(1) == 1 || v.size(1) == q.size(1), "v heads must equal q heads or 1");
  TORCH_CHECK(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(),
              "cuda_sm100: q, k, v dtypes must match");
}

at::Tensor freqs_vector(const at::Tensor& freqs, int64_t n) {
  at::Tensor f = freqs.reshape({-1});
  TORCH_CHECK(f.scalar_type() == at::kFloat && f.numel() == n,
              "freqs must be float32 with one entry per latent dimension");
  return f.contiguous();
}

// ------------------------------------------------------------------------ forward
// ln_eps >= 0: each output row LayerNormed over D (bdh_tril_score_v_layernorm).
at::Tensor score_v(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, double ln_eps) {
  check_cold_shapes(q, k, v);
  require_cuda({&q, &k, &v});
  const c10::cuda::CUDAGuard guard(q.device());
  const int dt = dtype_code(q);
  const int64_t B = q.size(0), H = q.size(1), T = q.size(2), Hv = v.size(1), D = v.size(3);
  at::Tensor out = at::empty({B, H, T, D}, q.options());
  if (out.numel() == 0) return out;
  const bool same = same_operand(q, k);
  at::Tensor qq = tma_ready(q);
  at::Tensor kk = same ? qq : tma_ready(k);
  at::Tensor vv = tma_ready(v);
  const int64_t Np = qq.size(3), Dp = vv.size(3);
  at::Tensor out_full = Dp != D ? at::empty({B, H, T, Dp}, q.options()) : out;
  const int k_is_q = same_operand(qq, kk) ? 1 : 0;
  const size_t wsz = bdh_tril_score_v_workspace_size(dt, B, H, Hv, T, Np, Dp, k_is_q);
  at::Tensor ws = at::empty({static_cast<int64_t>(std::max<size_t>(wsz, 1))},
                            q.options().dtype(at::kByte));
  const Strides4 sq(qq), sk(kk), sv(vv), so(out_full);
  if (ln_eps < 0) {
    check_rc(bdh_tril_score_v(qq.data_ptr(), sq.s, kk.data_ptr(), sk.s, vv.data_ptr(), sv.s, dt,
                              out_full.data_ptr(), so.s, dt, B, H, Hv, T, Np, Dp, ws.data_ptr(),
                              wsz, stream_of(q)),
             "tril_score_v");
  } else {
    TORCH_CHECK(Dp == D, "tril_score_v: the fused LayerNorm needs D a multiple of 16 bytes");
    check_rc(bdh_tril_score_v_layernorm(qq.data_ptr(), sq.s, kk.data_ptr(), sk.s, vv.data_ptr(),
                                        sv.s, dt, out_full.data_ptr(), so.s, dt, B, H, Hv, T, Np,
                                        Dp, static_cast<float>(ln_eps), ws.data_ptr(), wsz,
                                        stream_of(q)),
             "tril_score_v_layernorm");
  }
  if (Dp != D) out.copy_(out_full.narrow(3, 0, D));
  return out;
}

at::Tensor tril_score_v(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                        std::optional<double> ln_eps) {
  if (ln_eps.has_value()) TORCH_CHECK(*ln_eps >= 0.0, "ln_eps must be >= 0");
  return score_v(q, k, v, ln_eps.has_value() ? *ln_eps : -1.0);
}

// RoPE of x (B,H,T,N) at positions pos0 .. pos0 + T - 1 (phases from freqs in registers);
// relu_input rotates relu(x). out may be a strided view of another dtype (e.g. a cache slot).
at::Tensor rope_rotate(const at::Tensor& x_in, const at::Tensor& freqs, int64_t pos0,
                       std::optional<at::Tensor> out_opt, bool relu_input) {
  TORCH_CHECK(x_in.dim() == 4, "rope_rotate expects a 4-D (B, H, T, N) tensor");
  TORCH_CHECK(x_in.size(3) % 2 == 0, "RoPE last dim must be even, got " + std::to_string(x_in.size(3)));
  require_cuda({&x_in, &freqs});
  const c10::cuda::CUDAGuard guard(x_in.device());
  const at::Tensor f = freqs_vector(freqs, x_in.size(3));
  at::Tensor out;
  if (out_opt.has_value()) {
    out = *out_opt;
    TORCH_CHECK(out.sizes() == x_in.sizes() && out.device() == x_in.device(),
                "rope out= must match x shape/device");
    const at::MemOverlapStatus ov = at::get_overlap_status(out, x_in);
    TORCH_CHECK(ov != at::MemOverlapStatus::Full && ov != at::MemOverlapStatus::Partial,
                "rope out= must not alias x");
    TORCH_CHECK(out.stride(3) == 1, "rope out= must have a contiguous last dimension");
  } else {
    out = at::empty(x_in.sizes(), x_in.options());
  }
  const at::Tensor x = x_in.stride(3) == 1 ? x_in : x_in.contiguous();
  if (x.numel() == 0) return out;
  const Strides4 sx(x), so(out);
  check_rc(bdh_rope_rotate(x.data_ptr(), dtype_code(x), sx.s, out.data_ptr(), dtype_code(out), so.s,
                           nullptr, f.data_ptr<float>(), x.size(0), x.size(1), x.size(2), x.size(3),
                           pos0, relu_input ? 1 : 0, stream_of(x)),
           "rope_rotate");
  return out;
}

// RoPE then the forward, as the attention module runs them (bdh.py:396-412 with the
// reference's RoPE, kernels/rope.py:108-126): QR = R(q) at positions rope_start.. (one pass),
// out = tril(QR QR^T, -1) v. Returns (out, QR); QR goes to qr_out when given (e.g. the cache
// slot of a prefill).
std::tuple<at::Tensor, at::Tensor> rope_tril_score_v(const at::Tensor& q, const at::Tensor& v,
                                                     const at::Tensor& freqs, int64_t rope_start,
                                                     std::optional<at::Tensor> qr_out) {
  at::Tensor qr = rope_rotate(q, freqs, rope_start, qr_out, false);
  at::Tensor qq = qr.scalar_type() == q.scalar_type() ? qr : qr.to(q.scalar_type());
  return {score_v(qq, qq, v, -1.0), qr};
}

// ------------------------------------------------------------------------- decode
at::Tensor decode_impl(const at::Tensor& q_in, const at::Tensor& k_past, const at::Tensor& v_past,
                       const at::Tensor* freqs, int64_t pos, std::optional<at::Tensor> kr_slot) {
  TORCH_CHECK(q_in.dim() == 4 && k_past.dim() == 4 && v_past.dim() == 4,
              "q, k_past, v_past must be 4D");
  const int64_t B = q_in.size(0), H = q_in.size(1), Tq = q_in.size(2), N = q_in.size(3);
  const int64_t S = k_past.size(2), Hv = v_past.size(1), D = v_past.size(3);
  TORCH_CHECK(k_past.size(0) == B && k_past.size(1) == H && k_past.size(3) == N,
              "k_past shape ", shape_str(k_past), " incompatible with q ", shape_str(q_in));
  TORCH_CHECK(v_past.size(0) == B && v_past.size(2) == S, "v_past shape ", shape_str(v_past),
              " incompatible with k_past S=" + std::to_string(S));
  TORCH_CHECK(Hv == 1 || Hv == H, "v_past heads must equal q heads or 1");
  require_cuda({&q_in, &k_past, &v_past});
  TORCH_CHECK(k_past.scalar_type() == v_past.scalar_type(),
              "k_past and v_past must share the cache storage dtype");
  const c10::cuda::CUDAGuard guard(q_in.device());
  const int qd = dtype_code(q_in), kd = dtype_code(k_past);
  at::Tensor out = at::empty({B, H, Tq, D}, q_in.options());
  if (out.numel() == 0) {
    if (kr_slot.has_value() && freqs != nullptr && Tq > 0) rope_rotate(q_in, *freqs, pos, kr_slot, false);
    return out;
  }
  const at::Tensor q = q_in.stride(3) == 1 ? q_in : q_in.contiguous();
  TORCH_CHECK(k_past.stride(3) == 1 && v_past.stride(3) == 1,
              "cache views must have a contiguous last dimension");
  at::Tensor f;
  const float* fptr = nullptr;
  if (freqs != nullptr) {
    f = freqs_vector(*freqs, N);
    fptr = f.data_ptr<float>();
  }
  void* slot_ptr = nullptr;
  int64_t slot_strides[4] = {0, 0, 0, 1};
  if (kr_slot.has_value()) {
    TORCH_CHECK(freqs != nullptr, "kr_slot requires freqs (the slot receives the rotated query)");
    const at::Tensor& s = *kr_slot;
    TORCH_CHECK(s.sizes() == q.sizes() && s.scalar_type() == k_past.scalar_type() && s.stride(3) == 1,
                "kr_slot must match q's shape, the cache dtype and have unit last stride");
    slot_ptr = s.data_ptr();
    for (int i = 0; i < 4; ++i) slot_strides[i] = s.stride(i);
  }
  const size_t wsz = bdh_tril_decode_workspace_size(B, H, Tq, S, N, D);
  at::Tensor ws = at::empty({static_cast<int64_t>(std::max<size_t>(wsz, 4))},
                            q.options().dtype(at::kByte));
  const Strides4 sq(q), sk(k_past), sv(v_past), so(out);
  check_rc(bdh_tril_decode(q.data_ptr(), sq.s, qd, k_past.data_ptr(), sk.s, v_past.data_ptr(), sv.s,
                           kd, out.data_ptr(), so.s, B, H, Hv, Tq, S, N, D, fptr, pos, slot_ptr,
                           slot_ptr != nullptr ? slot_strides : nullptr, ws.data_ptr(), wsz,
                           stream_of(q)),
           "tril_decode");
  return out;
}

// out = (q k_past^T) v_past over the packed past only (no self term); S = 0 gives zeros.
at::Tensor tril_decode(const at::Tensor& q, const at::Tensor& k_past, const at::Tensor& v_past) {
  return decode_impl(q, k_past, v_past, nullptr, 0, std::nullopt);
}

// The decode step with the new query rotated to positions pos.. inside the kernel and, with
// kr_slot, the rotated rows written there (the cache append of this step).
at::Tensor rope_tril_decode(const at::Tensor& q_new, const at::Tensor& freqs, int64_t pos,
                            const at::Tensor& kr_past, const at::Tensor& v_past,
                            std::optional<at::Tensor> kr_slot) {
  return decode_impl(q_new, kr_past, v_past, &freqs, pos, kr_slot);
}

// ----------------------------------------------------------------------- backward
// Analytic gradients of tril(q k^T, -1) v (kernels/attention_bwd.py:45-83): (dq, dk, dv).
// When k is q the returned dq holds dq + dk and dk is None (StrictTrilSelfAttnFn's form); with
// freqs (self form only) q is the rotated QR and dq is the gradient of the unrotated latent.
std::tuple<at::Tensor, std::optional<at::Tensor>, at::Tensor> tril_score_v_bwd(
    const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& dout,
    std::optional<at::Tensor> freqs, int64_t pos0) {
  check_cold_shapes(q, k, v);
  require_cuda({&q, &k, &v, &dout});
  const c10::cuda::CUDAGuard guard(q.device());
  const int64_t B = q.size(0), H = q.size(1), T = q.size(2), N = q.size(3);
  const int64_t Hv = v.size(1), D = v.size(3);
  TORCH_CHECK(dout.dim() == 4 && dout.size(0) == B && dout.size(1) == H && dout.size(2) == T &&
                  dout.size(3) == D,
              "dout shape " + shape_str(dout) + " must be (" + std::to_string(B) + ", " +
                  std::to_string(H) + ", " + std::to_string(T) + ", " + std::to_string(D) + ")");
  const int dt = dtype_code(q);
  const bool same = same_operand(q, k);
  TORCH_CHECK(!freqs.has_value() || same,
              "the fused RoPE adjoint needs the self-attention form (k is q)");
  at::Tensor qq = tma_ready(q);
  at::Tensor kk = same ? qq : tma_ready(k);
  at::Tensor vv = tma_ready(v);
  at::Tensor dd = tma_ready(dout.to(q.scalar_type()));
  const int64_t Np = qq.size(3), Dp = vv.size(3);
  if (dd.size(3) != Dp) dd = at::constant_pad_nd(dd, {0, Dp - dd.size(3)});
  at::Tensor dq = at::empty({B, H, T, Np}, q.options());
  std::optional<at::Tensor> dk;
  if (!same) dk = at::empty({B, H, T, Np}, q.options());
  at::Tensor dv = at::empty({B, Hv, T, Dp}, q.options());
  at::Tensor f;
  const float* fptr = nullptr;
  if (freqs.has_value()) {
    f = freqs_vector(*freqs, N);
    TORCH_CHECK(Np == N, "the fused RoPE adjoint needs an aligned latent width");
    fptr = f.data_ptr<float>();
  }
  const size_t wsz = bdh_tril_score_v_bwd_workspace_size(dt, B, H, Hv, T, Np, Dp, same ? 1 : 0);
  at::Tensor ws = at::empty({static_cast<int64_t>(std::max<size_t>(wsz, 1))},
                            q.options().dtype(at::kByte));
  const Strides4 sq(qq), sk(kk), sv(vv), sd(dd), sdq(dq), sdv(dv);
  const Strides4 sdk(dk.has_value() ? *dk : dq);
  if (B * H * T > 0)
    check_rc(bdh_tril_score_v_bwd(qq.data_ptr(), sq.s, kk.data_ptr(), sk.s, vv.data_ptr(), sv.s,
                                  dd.data_ptr(), sd.s, dt, dq.data_ptr(), sdq.s,
                                  dk.has_value() ? dk->data_ptr() : nullptr, sdk.s, dv.data_ptr(),
                                  sdv.s, B, H, Hv, T, Np, Dp, fptr, pos0, ws.data_ptr(), wsz,
                                  stream_of(q)),
             "tril_score_v_bwd");
  if (Np != N) {
    dq = dq.narrow(3, 0, N).contiguous();
    if (dk.has_value()) dk = dk->narrow(3, 0, N).contiguous();
  }
  if (Dp != D) dv = dv.narrow(3, 0, D).contiguous();
  return {dq, dk, dv};
}

// ------------------------------------------------------------ fused layer (model path)
// The same checks and C-ABI calls as kernels/sm100_attn.py's latent_encode, latent_gate_dec,
// layer_norm and residual_layer_norm (bf16 latents with a contiguous last dimension, 16-byte
// aligned bases, strides in multiples of 8 elements; weights d-contiguous or n-contiguous).
void check_latent(const char* name, std::initializer_list<const at::Tensor*> ts) {
  for (const at::Tensor* t : ts) {
    TORCH_CHECK(t->scalar_type() == at::kBFloat16,
                std::string(name) + ": bf16 tensors required, got " + c10::toString(t->scalar_type()));
    bool ok = t->stride(-1) == 1 && reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0;
    for (int64_t d = 0; ok && d + 1 < t->dim(); ++d)
      if (t->size(d) > 1 && t->stride(d) % 8 != 0) ok = false;
    TORCH_CHECK(ok, std::string(name) +
                        ": tensors need a contiguous last dim, 16-byte aligned base and strides "
                        "that are multiples of 8 elements");
  }
}

void check_weight(const char* name, const at::Tensor& w) {
  TORCH_CHECK(w.scalar_type() == at::kBFloat16,
              std::string(name) + ": bf16 weights required, got " + c10::toString(w.scalar_type()));
  const bool k_major = w.stride(1) == 1 && w.stride(2) != 1 && w.stride(0) % 8 == 0 && w.stride(2) % 8 == 0;
  if (!k_major) {
    check_latent(name, {&w});
  } else {
    TORCH_CHECK(reinterpret_cast<uintptr_t>(w.data_ptr()) % 16 == 0,
                std::string(name) + ": weights need a 16-byte aligned base");
  }
}

// Element strides for the C-ABI: a size-1 dimension is never stepped, so an odd stride there
// becomes a legal 8.
template <int R>
struct StridesN {
  int64_t s[R];
  explicit StridesN(const at::Tensor& t) {
    for (int i = 0; i < R; ++i) {
      const int64_t st = t.stride(i);
      s[i] = (t.size(i) > 1 || st % 8 == 0 || st == 1) ? st : 8;
    }
    s[R - 1] = t.stride(R - 1);
  }
};

// freqs[2p] == freqs[2p + 1] (BDH's get_freqs): the fused encode shares one (cos, sin) per
// pair. Checked once per freqs tensor version (the check reads the tensor back).
bool paired_freqs(const at::Tensor& f) {
  static std::mutex mu;
  static std::vector<std::tuple<const void*, int64_t, int64_t, bool>> seen;
  const auto key = std::make_tuple(f.data_ptr(), static_cast<int64_t>(f._version()), f.numel());
  {
    std::lock_guard<std::mutex> g(mu);
    for (const auto& e : seen)
      if (std::get<0>(e) == std::get<0>(key) && std::get<1>(e) == std::get<1>(key) &&
          std::get<2>(e) == std::get<2>(key))
        return std::get<3>(e);
  }
  const bool ok = at::equal(f.slice(0, 0, f.numel(), 2), f.slice(0, 1, f.numel(), 2));
  std::lock_guard<std::mutex> g(mu);
  if (seen.size() > 64) seen.clear();
  seen.emplace_back(std::get<0>(key), std::get<1>(key), std::get<2>(key), ok);
  return ok;
}

// xs = relu(x enc) (B,T,H,N) and qr = RoPE(xs) (B,H,T,N) at positions pos0.., bf16.
std::tuple<std::optional<at::Tensor>, at::Tensor> latent_encode(
    const at::Tensor& x, const at::Tensor& enc, const at::Tensor& freqs, int64_t pos0,
    std::optional<at::Tensor> xs_out, std::optional<at::Tensor> qr_out, bool want_xs) {
  TORCH_CHECK(x.dim() == 3 && enc.dim() == 3 && x.size(2) == enc.size(1),
              "latent_encode expects x (B,T,D) and enc (H,D,N)");
  require_cuda({&x, &enc, &freqs});
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t B = x.size(0), T = x.size(1), D = x.size(2), H = enc.size(0), N = enc.size(2);
  const at::Tensor f = freqs_vector(freqs, N);
  TORCH_CHECK(paired_freqs(f), "latent_encode requires paired frequencies (freqs[2p] == freqs[2p+1])");
  std::optional<at::Tensor> xs = xs_out;
  if (!xs.has_value() && want_xs) xs = at::empty({B, T, H, N}, x.options().dtype(at::kBFloat16));
  at::Tensor qr = qr_out.has_value() ? *qr_out : at::empty({B, H, T, N}, x.options().dtype(at::kBFloat16));
  TORCH_CHECK((!xs.has_value() || xs->sizes() == at::IntArrayRef({B, T, H, N})) &&
                  qr.sizes() == at::IntArrayRef({B, H, T, N}),
              "latent_encode: xs_out must be (B,T,H,N) and qr_out (B,H,T,N)");
  if (xs.has_value())
    check_latent("latent_encode", {&x, &*xs, &qr});
  else
    check_latent("latent_encode", {&x, &qr});
  check_weight("latent_encode", enc);
  const StridesN<3> sx(x), se(enc);
  const StridesN<4> sq(qr);
  std::optional<StridesN<4>> sxs;
  if (xs.has_value()) sxs.emplace(*xs);
  check_rc(bdh_latent_encode(x.data_ptr(), sx.s, enc.data_ptr(), se.s,
                             xs.has_value() ? xs->data_ptr() : nullptr, sxs ? sxs->s : nullptr,
                             qr.data_ptr(), sq.s, f.data_ptr<float>(), B, T, H, D, N, pos0,
                             stream_of(x)),
           "latent_encode");
  return {xs, qr};
}

// (xs * relu(y encv)) dec in one kernel: y (B,H,T,D), encv (H,D,N) d-contiguous, xs (B,T,H,N),
// dec (H*N, D) latent-contiguous; D = 256, N a multiple of 128. Returns (B,T,D) bf16.
at::Tensor latent_gate_dec(const at::Tensor& y, const at::Tensor& encv, const at::Tensor& xs,
                           const at::Tensor& dec, std::optional<at::Tensor> out_opt) {
  TORCH_CHECK(y.dim() == 4 && encv.dim() == 3 && xs.dim() == 4 && dec.dim() == 2,
              "latent_gate_dec expects y (B,H,T,D), encv (H,D,N), xs (B,T,H,N), dec (H*N,D)");
  require_cuda({&y, &encv, &xs, &dec});
  const c10::cuda::CUDAGuard guard(y.device());
  const int64_t B = y.size(0), H = y.size(1), T = y.size(2), D = y.size(3), N = encv.size(2);
  TORCH_CHECK(xs.sizes() == at::IntArrayRef({B, T, H, N}) && encv.sizes() == at::IntArrayRef({H, D, N}) &&
                  dec.sizes() == at::IntArrayRef({H * N, D}),
              "latent_gate_dec: shapes of y, encv, xs and dec disagree");
  TORCH_CHECK(D == 256 && N % 128 == 0, "latent_gate_dec: needs D = 256 and N a multiple of 128");
  TORCH_CHECK(dec.scalar_type() == at::kBFloat16 && encv.scalar_type() == at::kBFloat16,
              "latent_gate_dec: bf16 weights required");
  at::Tensor out = out_opt.has_value() ? *out_opt : at::empty({B, T, D}, y.options().dtype(at::kBFloat16));
  TORCH_CHECK(out.sizes() == at::IntArrayRef({B, T, D}), "latent_gate_dec: out must be (B,T,D)");
  check_latent("latent_gate_dec", {&y, &xs, &out});
  check_weight("latent_gate_dec", encv);
  const size_t wsz = bdh_latent_gate_dec_workspace_size(B, T, H, D, N);
  at::Tensor ws;
  if (wsz > 0) ws = at::empty({static_cast<int64_t>(wsz)}, y.options().dtype(at::kByte));
  const StridesN<4> sy(y), sxs(xs);
  const StridesN<3> sev(encv), so(out);
  const StridesN<2> sd(dec);
  check_rc(bdh_latent_gate_dec_ws(y.data_ptr(), sy.s, encv.data_ptr(), sev.s, xs.data_ptr(), sxs.s,
                                  dec.data_ptr(), sd.s, out.data_ptr(), so.s, B, T, H, D, N,
                                  wsz > 0 ? ws.data_ptr() : nullptr, wsz, stream_of(y)),
           "latent_gate_dec");
  return out;
}

// (rows, D) with one row stride for the LayerNorm entries: a view when the leading dimensions
// flatten to one, else nullopt.
std::optional<at::Tensor> rows_view(const at::Tensor& t) {
  if (t.stride(-1) != 1) return std::nullopt;
  try {
    return t.view({-1, t.size(-1)});
  } catch (const c10::Error&) {
    return std::nullopt;
  }
}

int64_t row_stride(const at::Tensor& v) { return v.size(0) > 1 ? v.stride(0) : v.size(1); }

// Affine-free LayerNorm over the last dim, fp32 math, stored in out_dtype (default x's dtype).
at::Tensor layer_norm(const at::Tensor& x, double eps, std::optional<at::ScalarType> out_dtype,
                      std::optional<at::Tensor> out_opt) {
  require_cuda({&x});
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t D = x.size(-1);
  std::optional<at::Tensor> xv = rows_view(x);
  if (!xv.has_value()) xv = x.contiguous().view({-1, D});
  at::Tensor out = out_opt.has_value() ? *out_opt
                                       : at::empty(x.sizes(), x.options().dtype(out_dtype.value_or(x.scalar_type())));
  std::optional<at::Tensor> ov = rows_view(out);
  TORCH_CHECK(ov.has_value() && ov->size(0) == xv->size(0),
              "layer_norm: out must be row-contiguous with x's shape");
  check_rc(bdh_layernorm(xv->data_ptr(), dtype_code(*xv), row_stride(*xv), ov->data_ptr(),
                         dtype_code(*ov), row_stride(*ov), xv->size(0), D, static_cast<float>(eps),
                         stream_of(x)),
           "layer_norm");
  return out;
}

// LN(x + LN(y)) over the last dim (BDH._residual_ln): x fp32, y fp32 or bf16. Returns the
// fp32 result and, with want_bf16, its bf16 copy.
std::tuple<at::Tensor, std::optional<at::Tensor>> residual_layer_norm(const at::Tensor& x,
                                                                      const at::Tensor& y,
                                                                      double eps, bool want_bf16) {
  TORCH_CHECK(x.scalar_type() == at::kFloat && x.sizes() == y.sizes(),
              "residual_layer_norm: x must be fp32 and y of x's shape");
  require_cuda({&x, &y});
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t D = x.size(-1);
  std::optional<at::Tensor> xv = rows_view(x);
  if (!xv.has_value()) xv = x.contiguous().view({-1, D});
  std::optional<at::Tensor> yv = rows_view(y);
  if (!yv.has_value()) yv = y.contiguous().view({-1, D});
  at::Tensor out = at::empty(x.sizes(), x.options());
  std::optional<at::Tensor> out16;
  if (want_bf16) out16 = at::empty(x.sizes(), x.options().dtype(at::kBFloat16));
  check_rc(bdh_residual_layernorm(xv->data_ptr<float>(), row_stride(*xv), yv->data_ptr(),
                                  dtype_code(*yv), row_stride(*yv), out.data_ptr<float>(), D,
                                  out16.has_value() ? out16->data_ptr() : nullptr, D, xv->size(0), D,
                                  static_cast<float>(eps), stream_of(x)),
           "residual_layer_norm");
  return {out, out16};
}

// ------------------------------------------------------------------ operators on logits ----
// The operators have no forward-mode form: a tangent is refused where it would otherwise be dropped.
void check_no_tangent(const at::Tensor& t, const char* what) {
  if (t._fw_grad(0).defined())
    TORCH_CHECK_NOT_IMPLEMENTED(false, std::string(what) +
                                           ": forward-mode derivatives are not implemented");
}

// Logits (..., V) as (outer, inner) rows of V with unit stride: the last leading dimension is
// the inner one and the rest the outer, in place for up to two leading dimensions (and for more
// where they flatten), else a copy.
struct LogitRows {
  at::Tensor t;
  int64_t outer = 1, inner = 1, V = 0;
  int64_t strides[2] = {0, 0};
  at::DimVector lead;  // the caller's leading shape

  LogitRows(const at::Tensor& x, const char* what) : t(x) {
    if (x.dim() < 1) TORCH_CHECK_VALUE(false, std::string(what) + ": logits must be (..., V)");
    require_cuda({&x});
    check_no_tangent(x, what);
    if (x.scalar_type() != at::kFloat && x.scalar_type() != at::kBFloat16)
      TORCH_CHECK_TYPE(false, std::string(what) + ": logits must be float32 or bfloat16, got " +
                                  c10::toString(x.scalar_type()));
    V = x.size(-1);
    if (V < 1) TORCH_CHECK_VALUE(false, std::string(what) + ": the vocabulary is empty");
    lead.assign(x.sizes().begin(), x.sizes().end() - 1);
    for (size_t d = 0; d + 1 < lead.size(); ++d) outer *= lead[d];
    if (!lead.empty()) inner = lead.back();
    if (V > 1 && t.stride(-1) != 1) t = t.contiguous();
    if (t.dim() > 3) t = t.numel() == 0 ? t : t.reshape({outer, inner, V});
    if (t.dim() == 3) strides[0] = t.stride(0);
    if (t.dim() >= 2) strides[1] = t.stride(-2);
  }
  int64_t rows() const { return outer * inner; }
};

// A tensor of one value per row (or, with entries, `extra` values per row) beside the logits'
// leading shape, as its {outer, inner[, entry]} strides.
struct BesideRows {
  at::Tensor t;
  int64_t strides[3] = {0, 0, 0};

  BesideRows(const LogitRows& x, const at::Tensor& v, at::ScalarType dtype, int64_t extra,
             const char* what)
      : t(v) {
    if (!t.is_cuda() || t.device() != x.t.device())
      TORCH_CHECK(false, std::string(what) + " must be on the logits' device");
    check_no_tangent(t, what);
    const int64_t lists = extra >= 0 ? 1 : 0;
    const int64_t n = static_cast<int64_t>(x.lead.size());
    bool ok = t.dim() == n + lists && (lists == 0 || t.size(-1) == extra);
    for (int64_t d = 0; ok && d < n; ++d) ok = t.size(d) == x.lead[d];
    if (!ok)
      TORCH_CHECK_VALUE(false, std::string(what) + " has shape " + shape_str(t) +
                                   ", which does not go with logits of " + shape_str(x.t));
    if (t.scalar_type() != dtype) t = t.to(dtype);
    if (n > 2 && t.numel() > 0)
      t = lists ? t.reshape({x.outer, x.inner, extra}) : t.reshape({x.outer, x.inner});
    const int64_t r = t.dim() - lists;
    if (r >= 2) strides[0] = t.stride(r - 2);
    if (r >= 1) strides[1] = t.stride(r - 1);
    if (lists) strides[2] = t.stride(-1);
  }
};

bool whole(const at::Tensor& t) { return t.scalar_type() == at::kLong || t.scalar_type() == at::kInt; }

// One upstream gradient or weight per row; a 0-dimensional or broadcast one is read in place.
std::optional<BesideRows> per_row(const LogitRows& x, const std::optional<at::Tensor>& v,
                                  const char* what) {
  if (!v.has_value()) return std::nullopt;
  if (!v->is_floating_point())
    TORCH_CHECK_TYPE(false, std::string(what) + " must be a floating point tensor");
  at::Tensor t = *v;
  if (t.dim() == 0) t = t.expand(x.lead);
  return BesideRows(x, t, at::kFloat, -1, what);
}
const float* data_of(const std::optional<BesideRows>& v) {
  return v.has_value() ? v->t.data_ptr<float>() : nullptr;
}
const int64_t* strides_of(const std::optional<BesideRows>& v) {
  static const int64_t none[2] = {0, 0};
  return v.has_value() ? v->strides : none;
}

std::optional<BesideRows> token_rows(const LogitRows& x, const std::optional<at::Tensor>& tokens,
                                     const char* what) {
  if (!tokens.has_value()) return std::nullopt;
  if (!whole(*tokens)) TORCH_CHECK_TYPE(false, std::string(what) + ": tokens must be int64 or int32");
  return BesideRows(x, *tokens, at::kLong, -1, "tokens");
}

// A new tensor on the logits' device from the caching allocator (of the current device and stream), without
// at::empty's dispatch: a small call spends most of its host time on its outputs.
at::Tensor fresh(at::IntArrayRef shape, at::ScalarType dtype) {
  at::globalContext().lazyInitDevice(c10::DeviceType::CUDA);
  return at::detail::empty_generic(shape, c10::cuda::CUDACachingAllocator::get(),
                                   c10::DispatchKeySet(c10::DispatchKey::CUDA), dtype, std::nullopt);
}

// The fp32 figures of a call, one a row and of one shape, in one allocation (three would be a tenth of a
// small call). Each is a tensor of its own (not a view of another) at a 16-byte boundary of the shared
// storage. Nothing else shares one: lists outlive the figures and are saved, which a storage of two types
// cannot be.
void fresh_figures(std::initializer_list<at::Tensor*> figures, at::IntArrayRef shape) {
  int64_t each = 1;
  for (int64_t d : shape) each *= d;
  each = (each + 3) / 4 * 4;
  const at::Tensor slab = fresh({each * static_cast<int64_t>(figures.size())}, at::kFloat);
  int64_t at = 0;
  for (at::Tensor* figure : figures) {
    *figure = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(slab.storage()), slab.key_set(),
                                                       slab.dtype());
    figure->unsafeGetTensorImpl()->set_sizes_contiguous(shape);
    figure->unsafeGetTensorImpl()->set_storage_offset(at);
    at += each;
  }
}

void check_temperature(double temperature, const char* what) {
  if (!(temperature > 0.0) || !(temperature < 1e30) || !(temperature > 1e-30))
    TORCH_CHECK_VALUE(false, std::string(what) + ": temperature must be positive and finite, got " +
                                 std::to_string(temperature));
}

at::DimVector with_entries(const LogitRows& x, int64_t k) {
  at::DimVector s = x.lead;
  s.push_back(k);
  return s;
}

using MaybeTensor = std::optional<at::Tensor>;
MaybeTensor maybe(const at::Tensor& t) { return t.defined() ? MaybeTensor(t) : std::nullopt; }

// (logprob, entropy, lse, top_logprob, top_index, stats) per row; None where not asked for.
std::tuple<MaybeTensor, at::Tensor, at::Tensor, MaybeTensor, MaybeTensor, MaybeTensor>
token_logprobs(const at::Tensor& logits, const MaybeTensor& tokens, int64_t top_k,
               double temperature, int64_t ignore_index, bool want_stats) {
  const LogitRows x(logits, "token_logprobs");
  if (top_k < 0 || top_k > BDH_TOP_MAX || top_k > x.V)
    TORCH_CHECK_VALUE(false, "token_logprobs: top_k must be 0 to min(V, " +
                                 std::to_string(BDH_TOP_MAX) + "), got " + std::to_string(top_k));
  check_temperature(temperature, "token_logprobs");
  const std::optional<BesideRows> tok = token_rows(x, tokens, "token_logprobs");
  const c10::cuda::CUDAGuard guard(x.t.device());
  at::Tensor logprob, entropy, lse, top_logprob, top_index, stats;
  if (tok.has_value()) fresh_figures({&logprob, &entropy, &lse}, x.lead);
  else fresh_figures({&entropy, &lse}, x.lead);
  if (top_k > 0) {
    const at::DimVector entries = with_entries(x, top_k);
    top_logprob = fresh(entries, at::kFloat);
    top_index = fresh(entries, at::kLong);
  }
  if (want_stats) stats = fresh({x.rows(), 2}, at::kFloat);
  auto fp = [](const at::Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; };
  check_rc(bdh_token_logprobs(
               x.t.data_ptr(), dtype_code(x.t), x.strides,
               tok.has_value() ? tok->t.data_ptr<int64_t>() : nullptr, strides_of(tok),
               ignore_index, fp(logprob), lse.data_ptr<float>(), entropy.data_ptr<float>(),
               fp(stats), fp(top_logprob),
               top_index.defined() ? top_index.data_ptr<int64_t>() : nullptr, x.outer, x.inner,
               x.V, top_k, static_cast<float>(temperature), stream_of(x.t)),
           "token_logprobs");
  return {maybe(logprob), entropy, lse, maybe(top_logprob), maybe(top_index), maybe(stats)};
}

at::Tensor token_logprobs_bwd(const at::Tensor& logits, const MaybeTensor& tokens,
                              const at::Tensor& stats, const MaybeTensor& entropy,
                              const MaybeTensor& top_index, const MaybeTensor& g_logprob,
                              const MaybeTensor& g_entropy, const MaybeTensor& g_lse,
                              const MaybeTensor& g_top, double temperature, int64_t ignore_index) {
  const LogitRows x(logits, "token_logprobs_bwd");
  check_temperature(temperature, "token_logprobs_bwd");
  const std::optional<BesideRows> tok = token_rows(x, tokens, "token_logprobs_bwd"),
                                  glp = per_row(x, g_logprob, "g_logprob"),
                                  gen = per_row(x, g_entropy, "g_entropy"),
                                  gls = per_row(x, g_lse, "g_lse");
  const int64_t k = g_top.has_value() && top_index.has_value() ? top_index->size(-1) : 0;
  if (k > BDH_TOP_MAX || k > x.V)
    TORCH_CHECK_VALUE(false, "token_logprobs_bwd: a list of " + std::to_string(k) + " is too long");
  const c10::cuda::CUDAGuard guard(x.t.device());
  auto rowmajor = [&](const MaybeTensor& v, at::ScalarType dtype, int64_t n, const char* what) {
    if (!v->is_cuda() || v->device() != x.t.device() || v->scalar_type() != dtype || v->numel() != n)
      TORCH_CHECK_VALUE(false, std::string("token_logprobs_bwd: bad ") + what);
    check_no_tangent(*v, what);
    return v->contiguous();
  };
  const at::Tensor st = rowmajor(stats, at::kFloat, 2 * x.rows(), "stats");
  at::Tensor en, ti, gt;
  if (gen.has_value()) {
    if (!entropy.has_value()) TORCH_CHECK_VALUE(false, "token_logprobs_bwd: g_entropy needs entropy");
    en = rowmajor(entropy, at::kFloat, x.rows(), "entropy");
  }
  if (k > 0) {
    ti = rowmajor(top_index, at::kLong, k * x.rows(), "top_index");
    gt = rowmajor(g_top, at::kFloat, k * x.rows(), "g_top");
  }
  at::Tensor d = fresh(logits.sizes(), x.t.scalar_type());
  const int64_t ds[2] = {x.inner * x.V, x.V};
  check_rc(bdh_token_logprobs_bwd(
               x.t.data_ptr(), dtype_code(x.t), x.strides,
               tok.has_value() ? tok->t.data_ptr<int64_t>() : nullptr, strides_of(tok),
               ignore_index, st.data_ptr<float>(), gen.has_value() ? en.data_ptr<float>() : nullptr,
               k > 0 ? ti.data_ptr<int64_t>() : nullptr, data_of(glp), strides_of(glp),
               data_of(gls), strides_of(gls), data_of(gen), strides_of(gen),
               k > 0 ? gt.data_ptr<float>() : nullptr, d.data_ptr(), ds, x.outer, x.inner, x.V, k,
               static_cast<float>(temperature), stream_of(x.t)),
           "token_logprobs_bwd");
  return d;
}

struct DistillList {
  BesideRows index, teacher;
  std::optional<BesideRows> weight;
  int64_t k;
};
DistillList distill_list(const LogitRows& x, const at::Tensor& index, const at::Tensor& teacher,
                         const MaybeTensor& weight, double temperature) {
  if (!whole(index)) TORCH_CHECK_TYPE(false, "distill_topk: teacher_index must be int64 or int32");
  if (!teacher.is_floating_point())
    TORCH_CHECK_TYPE(false, "distill_topk: teacher_logprob must be a floating point tensor");
  const int64_t k = index.dim() > 0 ? index.size(-1) : 0;
  if (k < 1 || k > BDH_TOP_MAX)
    TORCH_CHECK_VALUE(false, "distill_topk: the list must have 1 to " + std::to_string(BDH_TOP_MAX) +
                                 " slots, got " + std::to_string(k));
  check_temperature(temperature, "distill_topk");
  return {BesideRows(x, index, at::kLong, k, "teacher_index"),
          BesideRows(x, teacher, at::kFloat, k, "teacher_logprob"), per_row(x, weight, "weight"), k};
}

// (loss per row, dlogits or None, stats or None)
std::tuple<at::Tensor, MaybeTensor, MaybeTensor> distill_topk(
    const at::Tensor& logits, const at::Tensor& index, const at::Tensor& teacher,
    const MaybeTensor& weight, double temperature, bool tail, bool want_grad, bool want_stats) {
  const LogitRows x(logits, "distill_topk");
  const c10::cuda::CUDAGuard guard(x.t.device());
  const DistillList l = distill_list(x, index, teacher, weight, temperature);
  at::Tensor loss = fresh(x.lead, at::kFloat);
  MaybeTensor d, stats;
  if (want_grad) d = fresh(logits.sizes(), x.t.scalar_type());
  if (want_stats) stats = fresh({x.rows(), 8}, at::kFloat);
  const int64_t ds[2] = {x.inner * x.V, x.V};
  check_rc(bdh_distill_topk(x.t.data_ptr(), dtype_code(x.t), x.strides,
                            l.index.t.data_ptr<int64_t>(), l.index.strides,
                            l.teacher.t.data_ptr<float>(), l.teacher.strides, data_of(l.weight),
                            strides_of(l.weight), loss.data_ptr<float>(),
                            want_stats ? stats->data_ptr<float>() : nullptr,
                            want_grad ? d->data_ptr() : nullptr, ds, x.outer, x.inner, x.V, l.k,
                            static_cast<float>(temperature), tail ? 1 : 0, stream_of(x.t)),
           "distill_topk");
  return {loss, d, stats};
}

at::Tensor distill_topk_bwd(const at::Tensor& logits, const at::Tensor& index,
                            const at::Tensor& teacher, const MaybeTensor& weight,
                            const at::Tensor& stats, const at::Tensor& g_loss, double temperature,
                            bool tail) {
  const LogitRows x(logits, "distill_topk_bwd");
  const c10::cuda::CUDAGuard guard(x.t.device());
  const DistillList l = distill_list(x, index, teacher, weight, temperature);
  const std::optional<BesideRows> g = per_row(x, g_loss, "g_loss");
  if (!stats.is_cuda() || stats.device() != x.t.device() || stats.scalar_type() != at::kFloat ||
      stats.numel() != 8 * x.rows())
    TORCH_CHECK_VALUE(false, "distill_topk_bwd: bad stats");
  const at::Tensor st = stats.contiguous();
  at::Tensor d = fresh(logits.sizes(), x.t.scalar_type());
  const int64_t ds[2] = {x.inner * x.V, x.V};
  check_rc(bdh_distill_topk_bwd(x.t.data_ptr(), dtype_code(x.t), x.strides,
                                l.index.t.data_ptr<int64_t>(), l.index.strides,
                                l.teacher.t.data_ptr<float>(), l.teacher.strides, data_of(l.weight),
                                strides_of(l.weight), st.data_ptr<float>(), data_of(g),
                                strides_of(g), d.data_ptr(), ds, x.outer, x.inner, x.V, l.k,
                                static_cast<float>(temperature), tail ? 1 : 0, stream_of(x.t)),
           "distill_topk_bwd");
  return d;
}

// The operators as autograd nodes (kernels/logits.py has the same in Python for the ctypes
// binding). Each is differentiable once: a second derivative raises, as once_differentiable's does.
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

at::Tensor defined_or_not(const MaybeTensor& t) { return t.value_or(at::Tensor()); }

// What backward needs of a constant input: saved as a variable (so that a later change in place is
// noticed), or, where it was made in inference mode, which cannot be, beside the variables.
at::Tensor constant(AutogradContext* ctx, const char* name, const at::Tensor& t) {
  if (!t.defined() || !t.is_inference()) return t;
  ctx->saved_data[name] = t;
  return at::Tensor();
}
at::Tensor constant_back(AutogradContext* ctx, const char* name, const at::Tensor& saved) {
  const auto it = ctx->saved_data.find(name);
  return it == ctx->saved_data.end() ? saved : it->second.toTensor();
}

variable_list once(variable_list grads, const at::Tensor& logits) {
  if (!at::GradMode::is_enabled()) return grads;
  // beside the logits, so that a second derivative by anything they come from finds the error
  auto error = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice an operator on logits, which is differentiable once", 2);
  grads[0] = (*error)({grads[0], logits})[0];
  return grads;
}

struct TokenLogprobsFn : torch::autograd::Function<TokenLogprobsFn> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& logits,
                               const MaybeTensor& tokens, int64_t top_k, double temperature,
                               int64_t ignore_index) {
    auto [logprob, entropy, lse, top_logprob, top_index, stats] =
        token_logprobs(logits, tokens, top_k, temperature, ignore_index, true);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({logits, constant(ctx, "tokens", defined_or_not(tokens)), *stats, entropy,
                            defined_or_not(top_index)});
    ctx->saved_data["temperature"] = temperature;
    ctx->saved_data["ignore_index"] = ignore_index;
    variable_list out = {entropy, lse};  // the figures asked for: a node has no undefined outputs
    if (logprob.has_value()) out.push_back(*logprob);
    if (top_index.has_value()) {
      ctx->mark_non_differentiable({*top_index});
      out.push_back(*top_logprob);
      out.push_back(*top_index);
    }
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    variable_list out(5);
    variable_list saved = ctx->get_saved_variables();
    saved[1] = constant_back(ctx, "tokens", saved[1]);
    const size_t top = saved[1].defined() ? 3 : 2;
    const at::Tensor g_logprob = saved[1].defined() ? g[2] : at::Tensor(),
                     g_top = saved[4].defined() ? g[top] : at::Tensor();
    if (!g[0].defined() && !g[1].defined() && !g_logprob.defined() && !g_top.defined()) return out;
    out[0] = token_logprobs_bwd(saved[0], maybe(saved[1]), saved[2], saved[3], maybe(saved[4]),
                                maybe(g_logprob), maybe(g[0]), maybe(g[1]), maybe(g_top),
                                ctx->saved_data["temperature"].toDouble(),
                                ctx->saved_data["ignore_index"].toInt());
    return once(out, saved[0]);
  }
};

std::tuple<MaybeTensor, at::Tensor, at::Tensor, MaybeTensor, MaybeTensor> token_logprobs_autograd(
    const at::Tensor& logits, const MaybeTensor& tokens, int64_t top_k, double temperature,
    int64_t ignore_index) {
  if (!at::GradMode::is_enabled() || !logits.requires_grad()) {
    auto r = token_logprobs(logits, tokens, top_k, temperature, ignore_index, false);
    return {std::get<0>(r), std::get<1>(r), std::get<2>(r), std::get<3>(r), std::get<4>(r)};
  }
  const variable_list r = TokenLogprobsFn::apply(logits, tokens, top_k, temperature, ignore_index);
  const size_t top = tokens.has_value() ? 3 : 2;
  return {tokens.has_value() ? MaybeTensor(r[2]) : std::nullopt, r[0], r[1],
          top_k > 0 ? MaybeTensor(r[top]) : std::nullopt,
          top_k > 0 ? MaybeTensor(r[top + 1]) : std::nullopt};
}

struct DistillTopkFn : torch::autograd::Function<DistillTopkFn> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& logits, const at::Tensor& index,
                            const at::Tensor& teacher, const MaybeTensor& weight,
                            double temperature, bool tail) {
    auto [loss, d, stats] = distill_topk(logits, index, teacher, weight, temperature, tail, false, true);
    ctx->save_for_backward({logits, constant(ctx, "index", index), constant(ctx, "teacher", teacher),
                            constant(ctx, "weight", defined_or_not(weight)), *stats});
    ctx->saved_data["temperature"] = temperature;
    ctx->saved_data["tail"] = tail;
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const variable_list saved = ctx->get_saved_variables();
    variable_list out(6);
    out[0] = distill_topk_bwd(saved[0], constant_back(ctx, "index", saved[1]),
                              constant_back(ctx, "teacher", saved[2]),
                              maybe(constant_back(ctx, "weight", saved[3])), saved[4], g[0],
                              ctx->saved_data["temperature"].toDouble(),
                              ctx->saved_data["tail"].toBool());
    return once(out, saved[0]);
  }
};

at::Tensor distill_topk_autograd(const at::Tensor& logits, const at::Tensor& index,
                                 const at::Tensor& teacher, const MaybeTensor& weight,
                                 double temperature, bool tail) {
  if (!at::GradMode::is_enabled() || !logits.requires_grad())
    return std::get<0>(distill_topk(logits, index, teacher, weight, temperature, tail, false, false));
  return DistillTopkFn::apply(logits, index, teacher, weight, temperature, tail);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "BDH strict lower-triangular score x V, decode and backward on sm_100a (no softmax)";
  m.def("tril_score_v", &tril_score_v,
        "out = tril(Q@K.T, diagonal=-1) @ V  (no softmax, no scale); with ln_eps each output row "
        "is LayerNormed over D before the store",
        py::arg("q"), py::arg("k"), py::arg("v"), py::arg("ln_eps") = py::none());
  m.def("tril_decode", &tril_decode,
        "out = (Q @ K_past.T) @ V_past  (packed past; no self-attend)", py::arg("q"),
        py::arg("k_past"), py::arg("v_past"));
  m.def("tril_score_v_bwd", &tril_score_v_bwd,
        "(dq, dk, dv) of tril(Q@K.T, -1) @ V; dq = dq + dk and dk = None when k is q; with freqs "
        "q is the rotated QR and dq the gradient of the unrotated latent",
        py::arg("q"), py::arg("k"), py::arg("v"), py::arg("dout"), py::arg("freqs") = py::none(),
        py::arg("pos0") = 0);
  m.def("rope_rotate", &rope_rotate, "BDH RoPE at positions pos0.. (phases in registers)",
        py::arg("x"), py::arg("freqs"), py::arg("pos0") = 0, py::arg("out") = py::none(),
        py::arg("relu_input") = false);
  m.def("rope_tril_score_v", &rope_tril_score_v,
        "(out, QR): QR = RoPE(q) at positions rope_start.., out = tril(QR@QR.T, -1) @ V",
        py::arg("q"), py::arg("v"), py::arg("freqs"), py::arg("rope_start") = 0,
        py::arg("qr_out") = py::none());
  m.def("rope_tril_decode", &rope_tril_decode,
        "decode step with the new query RoPE-rotated to positions pos.. (and written to kr_slot)",
        py::arg("q_new"), py::arg("freqs"), py::arg("pos"), py::arg("kr_past"), py::arg("v_past"),
        py::arg("kr_slot") = py::none());
  m.def("latent_encode", &latent_encode,
        "(xs, qr): xs = relu(x @ enc) (B,T,H,N), qr = RoPE(xs) (B,H,T,N) at positions pos0.., bf16",
        py::arg("x"), py::arg("enc"), py::arg("freqs"), py::arg("pos0") = 0,
        py::arg("xs_out") = py::none(), py::arg("qr_out") = py::none(), py::arg("want_xs") = true);
  m.def("latent_gate_dec", &latent_gate_dec, "(xs * relu(y @ encv)) @ dec in one kernel, (B,T,D) bf16",
        py::arg("y"), py::arg("encv"), py::arg("xs"), py::arg("dec"), py::arg("out") = py::none());
  m.def("layer_norm", &layer_norm, "affine-free LayerNorm over the last dim (fp32 math)",
        py::arg("x"), py::arg("eps") = 1e-5, py::arg("out_dtype") = py::none(),
        py::arg("out") = py::none());
  m.def("residual_layer_norm", &residual_layer_norm,
        "(LN(x + LN(y)), its bf16 copy or None): the BDH layer's residual double LayerNorm",
        py::arg("x"), py::arg("y"), py::arg("eps") = 1e-5, py::arg("want_bf16") = false);
  m.def("token_logprobs", &token_logprobs,
        "(logprob, entropy, lse, top_logprob, top_index, stats) of every row of logits",
        py::arg("logits"), py::arg("tokens") = py::none(), py::arg("top_k") = 0,
        py::arg("temperature") = 1.0, py::arg("ignore_index") = -100, py::arg("want_stats") = false);
  m.def("token_logprobs_bwd", &token_logprobs_bwd, "gradient of token_logprobs by the logits",
        py::arg("logits"), py::arg("tokens"), py::arg("stats"), py::arg("entropy") = py::none(),
        py::arg("top_index") = py::none(), py::arg("g_logprob") = py::none(),
        py::arg("g_entropy") = py::none(), py::arg("g_lse") = py::none(),
        py::arg("g_top") = py::none(), py::arg("temperature") = 1.0, py::arg("ignore_index") = -100);
  m.def("distill_topk", &distill_topk,
        "(loss, dlogits or None, stats or None) against a teacher's list of top tokens",
        py::arg("logits"), py::arg("teacher_index"), py::arg("teacher_logprob"),
        py::arg("weight") = py::none(), py::arg("temperature") = 1.0, py::arg("tail") = false,
        py::arg("want_grad") = false, py::arg("want_stats") = false);
  m.def("distill_topk_bwd", &distill_topk_bwd, "gradient of distill_topk's loss by the logits",
        py::arg("logits"), py::arg("teacher_index"), py::arg("teacher_logprob"), py::arg("weight"),
        py::arg("stats"), py::arg("g_loss"), py::arg("temperature") = 1.0, py::arg("tail") = false);
  m.def("token_logprobs_autograd", &token_logprobs_autograd,
        "(logprob, entropy, lse, top_logprob, top_index), differentiable by the logits",
        py::arg("logits"), py::arg("tokens"), py::arg("top_k"), py::arg("temperature"),
        py::arg("ignore_index"));
  m.def("distill_topk_autograd", &distill_topk_autograd,
        "loss against a teacher's list of top tokens, differentiable by the logits",
        py::arg("logits"), py::arg("teacher_index"), py::arg("teacher_logprob"), py::arg("weight"),
        py::arg("temperature"), py::arg("tail"));
  m.def("abi_version", &bdh_abi_version, "ABI version of the loaded libbdh_sm100.so");
  m.def("in_use", [] {
    const char* v = std::getenv("BDH_SM100_EXT");
    return v == nullptr || std::strcmp(v, "0") != 0;
  }, "False where BDH_SM100_EXT is 0 (os.environ takes ten times as long to say so)");
  m.attr("has_cuda") = true;
}
