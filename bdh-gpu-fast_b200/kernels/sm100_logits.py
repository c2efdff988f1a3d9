"""ctypes binding of the library's operators on logits (``bdh_token_logprobs``,
``bdh_distill_topk`` and their backward forms, include/bdh_sm100.h), with the names, arguments and
checks of the same functions of ``bdh_sm100_ext``. ``kernels.logits`` is the public face of both.
"""

from __future__ import annotations

import ctypes
from typing import Optional

import torch
from torch.autograd import forward_ad

from .sm100_attn import _check, _code, _require_cuda, _require_lib, _stream

TOP_MAX = 128  # BDH_TOP_MAX

_vp, _i64, _f32, _int = ctypes.c_void_p, ctypes.c_int64, ctypes.c_float, ctypes.c_int
_P = ctypes.POINTER(ctypes.c_int64)
_declared = False


def _lib() -> ctypes.CDLL:
    global _declared
    lib = _require_lib()
    if not _declared:
        sizes = [_i64, _i64, _i64, _i64, _f32]
        lib.bdh_token_logprobs.argtypes = [_vp, _int, _P, _vp, _P, _i64, _vp, _vp, _vp, _vp, _vp,
                                           _vp, *sizes, _vp]
        lib.bdh_token_logprobs_bwd.argtypes = [_vp, _int, _P, _vp, _P, _i64, _vp, _vp, _vp, _vp, _P,
                                               _vp, _P, _vp, _P, _vp, _vp, _P, *sizes, _vp]
        lib.bdh_distill_topk.argtypes = [_vp, _int, _P, _vp, _P, _vp, _P, _vp, _P, _vp, _vp, _vp,
                                         _P, *sizes, _int, _vp]
        lib.bdh_distill_topk_bwd.argtypes = [_vp, _int, _P, _vp, _P, _vp, _P, _vp, _P, _vp, _vp, _P,
                                             _vp, _P, *sizes, _int, _vp]
        for name in ("bdh_token_logprobs", "bdh_token_logprobs_bwd", "bdh_distill_topk",
                     "bdh_distill_topk_bwd"):
            getattr(lib, name).restype = ctypes.c_int
        _declared = True
    return lib


def check_no_tangent(t: torch.Tensor, what: str) -> None:
    """The operators have no forward-mode form: a tangent is refused where it would otherwise be
    dropped."""
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
        raise NotImplementedError(f"{what}: forward-mode derivatives are not implemented")


class _Rows:
    """Logits (..., V) as (outer, inner) rows of V with unit stride, in place for up to two
    leading dimensions (and for more where they flatten)."""

    def __init__(self, x: torch.Tensor, what: str):
        if x.dim() < 1:
            raise ValueError(f"{what}: logits must be (..., V)")
        _require_cuda(x)
        check_no_tangent(x, what)
        if x.dtype not in (torch.float32, torch.bfloat16):
            raise TypeError(f"{what}: logits must be float32 or bfloat16, got {x.dtype}")
        self.lead, self.V = tuple(x.shape[:-1]), x.size(-1)
        if self.V < 1:
            raise ValueError(f"{what}: the vocabulary is empty")
        self.outer, self.inner = 1, 1
        for n in self.lead[:-1]:
            self.outer *= n
        if self.lead:
            self.inner = self.lead[-1]
        if self.V > 1 and x.stride(-1) != 1:
            x = x.contiguous()
        if x.dim() > 3 and x.numel() > 0:
            x = x.reshape(self.outer, self.inner, self.V)
        self.t = x
        self.rows = self.outer * self.inner
        self.strides = (_i64 * 2)(x.stride(0) if x.dim() == 3 else 0,
                                  x.stride(-2) if x.dim() >= 2 else 0)

    def beside(self, v: torch.Tensor, dtype: torch.dtype, what: str, extra: Optional[int] = None):
        """(tensor, strides) of one value (or ``extra`` values) per row."""
        if v.device != self.t.device:
            raise RuntimeError(f"{what} must be on the logits' device")
        check_no_tangent(v, what)
        want = self.lead + (() if extra is None else (extra,))
        if tuple(v.shape) != want:
            raise ValueError(f"{what} has shape {tuple(v.shape)}, which does not go with logits of "
                             f"{tuple(self.t.shape)}")
        v = v.to(dtype)
        if len(self.lead) > 2 and v.numel() > 0:
            v = v.reshape((self.outer, self.inner) + (() if extra is None else (extra,)))
        st = list(v.stride())
        entry = [st.pop()] if extra is not None else []
        lead = [0] * (2 - len(st[-2:])) + st[-2:]
        return v, (_i64 * 3)(*(lead + entry + [0])[:3])

    def per_row(self, v: Optional[torch.Tensor], what: str):
        if v is None:
            return None, (_i64 * 3)(0, 0, 0)
        if not v.is_floating_point():
            raise TypeError(f"{what} must be a floating point tensor")
        return self.beside(v.expand(self.lead) if v.dim() == 0 else v, torch.float32, what)

    def tokens(self, tokens: Optional[torch.Tensor], what: str):
        if tokens is None:
            return None, (_i64 * 3)(0, 0, 0)
        if tokens.dtype not in (torch.int64, torch.int32):
            raise TypeError(f"{what}: tokens must be int64 or int32")
        return self.beside(tokens, torch.int64, "tokens")

    def grad(self) -> tuple[torch.Tensor, ctypes.Array]:
        d = torch.empty(self.lead + (self.V,), dtype=self.t.dtype, device=self.t.device)
        return d, (_i64 * 2)(self.inner * self.V, self.V)


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _check_temperature(temperature: float, what: str) -> None:
    if not 1e-30 < temperature < 1e30:
        raise ValueError(f"{what}: temperature must be positive and finite, got {temperature}")


def token_logprobs(logits, tokens=None, top_k=0, temperature=1.0, ignore_index=-100,
                   want_stats=False):
    """(logprob, entropy, lse, top_logprob, top_index, stats) per row; None where not asked for."""
    x = _Rows(logits, "token_logprobs")
    if not 0 <= top_k <= min(x.V, TOP_MAX):
        raise ValueError(f"token_logprobs: top_k must be 0 to min(V, {TOP_MAX}), got {top_k}")
    _check_temperature(temperature, "token_logprobs")
    tok, ts = x.tokens(tokens, "token_logprobs")
    lib, dev = _lib(), x.t.device
    f32 = lambda *s: torch.empty(s, dtype=torch.float32, device=dev)  # noqa: E731
    logprob = f32(*x.lead) if tok is not None else None
    entropy, lse = f32(*x.lead), f32(*x.lead)
    top = f32(*x.lead, top_k) if top_k else None
    index = torch.empty(*x.lead, top_k, dtype=torch.int64, device=dev) if top_k else None
    stats = f32(x.rows, 2) if want_stats else None
    with torch.cuda.device(dev):
        rc = lib.bdh_token_logprobs(
            x.t.data_ptr(), _code(x.t.dtype), x.strides, _ptr(tok), ts, int(ignore_index),
            _ptr(logprob), lse.data_ptr(), entropy.data_ptr(), _ptr(stats), _ptr(top), _ptr(index),
            x.outer, x.inner, x.V, int(top_k), float(temperature), _stream(dev))
    _check(rc, "token_logprobs")
    return logprob, entropy, lse, top, index, stats


def token_logprobs_bwd(logits, tokens, stats, entropy=None, top_index=None, g_logprob=None,
                       g_entropy=None, g_lse=None, g_top=None, temperature=1.0, ignore_index=-100):
    """The gradient of ``token_logprobs`` with respect to the logits."""
    what = "token_logprobs_bwd"
    x = _Rows(logits, what)
    _check_temperature(temperature, what)
    tok, ts = x.tokens(tokens, what)
    (glp, s1), (gls, s2), (gen, s3) = (x.per_row(g_logprob, "g_logprob"), x.per_row(g_lse, "g_lse"),
                                       x.per_row(g_entropy, "g_entropy"))
    k = top_index.size(-1) if g_top is not None and top_index is not None else 0
    if k > min(TOP_MAX, x.V):
        raise ValueError(f"{what}: a list of {k} is too long")

    def rowmajor(v, dtype, n, name):
        if v is None or v.device != x.t.device or v.dtype != dtype or v.numel() != n:
            raise ValueError(f"{what}: bad {name}")
        check_no_tangent(v, name)
        return v.contiguous()

    stats = rowmajor(stats, torch.float32, 2 * x.rows, "stats")
    entropy = rowmajor(entropy, torch.float32, x.rows, "entropy") if gen is not None else None
    top_index = rowmajor(top_index, torch.int64, k * x.rows, "top_index") if k else None
    g_top = rowmajor(g_top, torch.float32, k * x.rows, "g_top") if k else None
    d, ds = x.grad()
    lib, dev = _lib(), x.t.device
    with torch.cuda.device(dev):
        rc = lib.bdh_token_logprobs_bwd(
            x.t.data_ptr(), _code(x.t.dtype), x.strides, _ptr(tok), ts, int(ignore_index),
            stats.data_ptr(), _ptr(entropy), _ptr(top_index), _ptr(glp), s1, _ptr(gls), s2,
            _ptr(gen), s3, _ptr(g_top), d.data_ptr(), ds, x.outer, x.inner, x.V, k,
            float(temperature), _stream(dev))
    _check(rc, what)
    return d


def _list(x: _Rows, index, teacher, weight, temperature):
    if index.dtype not in (torch.int64, torch.int32):
        raise TypeError("distill_topk: teacher_index must be int64 or int32")
    if not teacher.is_floating_point():
        raise TypeError("distill_topk: teacher_logprob must be a floating point tensor")
    k = index.size(-1) if index.dim() else 0
    if not 1 <= k <= TOP_MAX:
        raise ValueError(f"distill_topk: the list must have 1 to {TOP_MAX} slots, got {k}")
    _check_temperature(temperature, "distill_topk")
    return (k, x.beside(index, torch.int64, "teacher_index", k),
            x.beside(teacher, torch.float32, "teacher_logprob", k), x.per_row(weight, "weight"))


def distill_topk(logits, teacher_index, teacher_logprob, weight=None, temperature=1.0, tail=False,
                 want_grad=False, want_stats=False):
    """(loss per row, dlogits or None, stats or None) against a teacher's list of top tokens."""
    x = _Rows(logits, "distill_topk")
    k, (idx, si), (val, sv), (w, sw) = _list(x, teacher_index, teacher_logprob, weight, temperature)
    lib, dev = _lib(), x.t.device
    loss = torch.empty(x.lead, dtype=torch.float32, device=dev)
    stats = torch.empty(x.rows, 8, dtype=torch.float32, device=dev) if want_stats else None
    d, ds = x.grad() if want_grad else (None, (_i64 * 2)(0, 0))
    with torch.cuda.device(dev):
        rc = lib.bdh_distill_topk(
            x.t.data_ptr(), _code(x.t.dtype), x.strides, idx.data_ptr(), si, val.data_ptr(), sv,
            _ptr(w), sw, loss.data_ptr(), _ptr(stats), _ptr(d), ds, x.outer, x.inner, x.V, k,
            float(temperature), 1 if tail else 0, _stream(dev))
    _check(rc, "distill_topk")
    return loss, d, stats


def distill_topk_bwd(logits, teacher_index, teacher_logprob, weight, stats, g_loss, temperature=1.0,
                     tail=False):
    """The gradient of ``distill_topk``'s loss with respect to the logits."""
    x = _Rows(logits, "distill_topk_bwd")
    k, (idx, si), (val, sv), (w, sw) = _list(x, teacher_index, teacher_logprob, weight, temperature)
    g, sg = x.per_row(g_loss, "g_loss")
    if stats.device != x.t.device or stats.dtype != torch.float32 or stats.numel() != 8 * x.rows:
        raise ValueError("distill_topk_bwd: bad stats")
    stats = stats.contiguous()
    d, ds = x.grad()
    lib, dev = _lib(), x.t.device
    with torch.cuda.device(dev):
        rc = lib.bdh_distill_topk_bwd(
            x.t.data_ptr(), _code(x.t.dtype), x.strides, idx.data_ptr(), si, val.data_ptr(), sv,
            _ptr(w), sw, stats.data_ptr(), g.data_ptr(), sg, d.data_ptr(), ds, x.outer, x.inner,
            x.V, k, float(temperature), 1 if tail else 0, _stream(dev))
    _check(rc, "distill_topk_bwd")
    return d
