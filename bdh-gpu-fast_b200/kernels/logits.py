"""Operators on a language model's logits, on the sm_100a kernels of the library:

* ``token_logprobs``: the log probabilities of given tokens, the entropy and the most probable
  alternatives of every position (scoring, decoding, policy gradients, a teacher's lists);
* ``distill_topk_loss`` / ``distill_topk_loss_grad``: a student's loss against the lists that a
  teacher kept, and its gradient.

The reference computes its loss and its sampling with torch (bdh.py:680-728, :1066-1072); these
have no counterpart there. Logits are ``(..., V)`` float32 or bfloat16 with any leading shape and
strides (a shifted view ``[:, :-1]`` is read in place, the vocabulary needs no particular size);
statistics are float32. CUDA tensors only (no CPU fallback). Work is queued on the current stream
and can be captured in a CUDA graph. Both operators are differentiable with respect to the logits
(once, in reverse mode; a tangent raises); a gradient comes in the logits' dtype.
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import sm100_attn, sm100_ext, sm100_logits


class TokenLogprobs(NamedTuple):
    """Per position; ``logprob`` is None without tokens, the two lists without ``top_k``. The lists
    have a storage each; the three figures may share one."""

    logprob: Optional[torch.Tensor]      # (...,) fp32: log p[token]
    entropy: torch.Tensor                # (...,) fp32: -sum p log p
    lse: torch.Tensor                    # (...,) fp32: log sum exp(logits / temperature)
    top_logprob: Optional[torch.Tensor]  # (..., top_k) fp32, falling
    top_index: Optional[torch.Tensor]    # (..., top_k) int64


def _ops():
    """The extension's functions when it is built, else the ctypes binding of the same library."""
    ext = sm100_ext._ext
    if ext is not None and ext.in_use():
        return ext
    ops = sm100_ext.model_ops()
    return sm100_logits if ops is sm100_attn else ops


def _once(d: torch.Tensor, logits: torch.Tensor) -> torch.Tensor:
    """A gradient that raises where it is itself differentiated. (torch's once_differentiable lets
    it pass as a constant when the upstream gradient needs none; this one depends on the logits.)"""
    if not torch.is_grad_enabled():
        return d
    error = torch._C._functions.DelayedError(
        "trying to differentiate twice an operator on logits, which is differentiable once", 2)
    return error(d, logits)[0]


# The autograd nodes of the ctypes binding; the extension has its own (a tenth of the host time).
def _save(ctx, constants: dict, **variables) -> None:
    """save_for_backward, with constant inputs that were made in inference mode (and so cannot be
    saved) kept beside it."""
    ctx.beside = {k: t for k, t in constants.items() if t is not None and t.is_inference()}
    ctx.names = list(constants) + list(variables)
    ctx.save_for_backward(*(None if k in ctx.beside else t for k, t in constants.items()),
                          *variables.values())


def _saved(ctx) -> dict:
    return {**dict(zip(ctx.names, ctx.saved_tensors)), **ctx.beside}


class _TokenLogprobsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, top_k, temperature, ignore_index):
        logprob, entropy, lse, top, index, stats = _ops().token_logprobs(
            logits, tokens, top_k, temperature, ignore_index, True)
        ctx.set_materialize_grads(False)
        _save(ctx, {"tokens": tokens}, logits=logits, stats=stats, entropy=entropy, top_index=index)
        ctx.opts = (temperature, ignore_index)
        if index is not None:
            ctx.mark_non_differentiable(index)
        return logprob, entropy, lse, top, index

    @staticmethod
    def backward(ctx, g_logprob, g_entropy, g_lse, g_top, _):
        if g_logprob is None and g_entropy is None and g_lse is None and g_top is None:
            return (None,) * 5
        temperature, ignore_index = ctx.opts
        saved = _saved(ctx)
        d = _ops().token_logprobs_bwd(**saved, g_logprob=g_logprob, g_entropy=g_entropy, g_lse=g_lse,
                                      g_top=g_top, temperature=temperature,
                                      ignore_index=ignore_index)
        return _once(d, saved["logits"]), None, None, None, None


def token_logprobs(logits: torch.Tensor, tokens: Optional[torch.Tensor] = None, *, top_k: int = 0,
                   temperature: float = 1.0, ignore_index: int = -100) -> TokenLogprobs:
    """Log probabilities of ``tokens`` (int64 or int32, the logits' leading shape) under
    ``softmax(logits / temperature)``, with entropy and the ``top_k`` (at most 128) largest logits
    of every position, in one pass over the logits.

    ``top_index`` is in falling order of the logits, an equal value's lower index first, NaN before
    everything. A token equal to ``ignore_index`` has log probability 0 and passes no gradient; any
    other token outside ``[0, V)`` has NaN. A position with no logit above -inf (a mask that leaves
    nothing) has ``lse`` and log probabilities -inf, entropy 0 and a zero gradient. A NaN or +inf
    logit makes its position's figures NaN. ``logprob``, ``entropy``, ``lse`` and ``top_logprob``
    carry gradients to the logits.
    """
    ops = _ops()
    if ops is not sm100_logits:
        return tuple.__new__(TokenLogprobs, ops.token_logprobs_autograd(
            logits, tokens, top_k, temperature, ignore_index))
    if torch.is_grad_enabled() and logits.requires_grad:
        return TokenLogprobs(*_TokenLogprobsFn.apply(logits, tokens, top_k, temperature,
                                                     ignore_index))
    return TokenLogprobs(*ops.token_logprobs(logits, tokens, top_k, temperature,
                                             ignore_index)[:5])


class _DistillTopkFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, index, teacher, weight, temperature, tail):
        loss, _, stats = _ops().distill_topk(logits, index, teacher, weight, temperature, tail,
                                             False, True)
        _save(ctx, {"teacher_index": index, "teacher_logprob": teacher, "weight": weight},
              logits=logits, stats=stats)
        ctx.opts = (temperature, tail)
        return loss

    @staticmethod
    def backward(ctx, g_loss):
        temperature, tail = ctx.opts
        saved = _saved(ctx)
        d = _ops().distill_topk_bwd(**saved, g_loss=g_loss, temperature=temperature, tail=tail)
        return _once(d, saved["logits"]), None, None, None, None, None


def _constant_teacher(teacher_logprob, weight) -> None:
    if torch.is_grad_enabled() and (teacher_logprob.requires_grad
                                    or (weight is not None and weight.requires_grad)):
        raise ValueError("distill_topk_loss: the teacher's list and the weights are constants "
                         "(no gradient reaches them); detach them")


def distill_topk_loss(logits: torch.Tensor, teacher_index: torch.Tensor,
                      teacher_logprob: torch.Tensor, *, weight: Optional[torch.Tensor] = None,
                      temperature: float = 1.0, tail: bool = False) -> torch.Tensor:
    """Kullback-Leibler divergence of every position's teacher list from the student's
    ``p = softmax(logits / temperature)``: (...,) fp32, each position times its ``weight``.

    ``teacher_index`` (..., k) int64 or int32 and ``teacher_logprob`` (..., k), 1 <= k <= 128: the
    teacher's top tokens and their log probabilities at the temperature of the loss, as
    ``token_logprobs(..., top_k=k)`` gives them. ``tail=False`` renormalises them over the list
    (logits / temperature do as well then); ``tail=True`` takes them as they are and makes "every
    other token" one more class, with the probability the list leaves over (up to 2^-16 of it, an
    fp32 list's rounding, counts as none where the student masks every other token; more costs an
    infinite loss there). An index below 0 is an empty slot, one past the vocabulary makes the
    position NaN, the masses of a repeated one add.
    ``weight``: a tensor of the leading shape or with no dimension; a position of weight 0 gives
    exactly 0, whatever it holds. Multiply by temperature ** 2 in the weight where that
    convention is wanted. Differentiable with respect to the logits.
    """
    _constant_teacher(teacher_logprob, weight)
    ops = _ops()
    if ops is not sm100_logits:
        return ops.distill_topk_autograd(logits, teacher_index, teacher_logprob, weight,
                                         temperature, tail)
    if torch.is_grad_enabled() and logits.requires_grad:
        return _DistillTopkFn.apply(logits, teacher_index, teacher_logprob, weight, temperature,
                                    tail)
    return ops.distill_topk(logits, teacher_index, teacher_logprob, weight, temperature, tail)[0]


def distill_topk_loss_grad(logits: torch.Tensor, teacher_index: torch.Tensor,
                           teacher_logprob: torch.Tensor, *,
                           weight: Optional[torch.Tensor] = None, temperature: float = 1.0,
                           tail: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """``(loss, dlogits)``: ``distill_topk_loss`` and the gradient of its sum over all positions in
    one call that reads the logits from memory once (through autograd they are read twice). A
    training step goes on with ``logits.backward(dlogits)``."""
    _constant_teacher(teacher_logprob, weight)
    sm100_logits.check_no_tangent(logits, "distill_topk")  # (detach drops it)
    loss, d, _ = _ops().distill_topk(logits.detach(), teacher_index, teacher_logprob, weight,
                                     temperature, tail, True)
    return loss, d


__all__ = ["TokenLogprobs", "token_logprobs", "distill_topk_loss", "distill_topk_loss_grad"]
