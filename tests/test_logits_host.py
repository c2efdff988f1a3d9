"""The operators on logits without a GPU: the 64-bit oracle's gradients against differences, the
C-ABI's argument checks (made before any launch), and the refusal of CPU tensors."""

import ctypes

import pytest
import torch

import logits_oracle as L


def _difference(f, x, eps=1e-5):
    """Central differences of a scalar f at the 64-bit x: error ~ eps^2 |f'''| / 6 + 2^-52 |f| / eps,
    both below 1e-9 for the O(1) functions here."""
    d = torch.zeros_like(x)
    flat, out = x.reshape(-1), d.reshape(-1)
    for i in range(flat.numel()):
        keep = flat[i].item()
        flat[i] = keep + eps
        hi = f(x)
        flat[i] = keep - eps
        out[i] = (hi - f(x)) / (2 * eps)
        flat[i] = keep
    return d


@pytest.mark.parametrize("temperature", [1.0, 0.7, 2.0])
def test_oracle_logprob_gradient_against_differences(temperature):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(3, 9, generator=g, dtype=torch.float64)
    tok = torch.tensor([2, -100, 8])
    gs = {n: torch.randn(3, generator=g, dtype=torch.float64)
          for n in ("g_logprob", "g_entropy", "g_lse")}
    g_top = torch.randn(3, 4, generator=g, dtype=torch.float64)
    index = L.order(x, 4)

    def f(x):
        o = L.token_logprobs(x, tok, 0, temperature)
        o["top"] = torch.log_softmax(x / temperature, -1).gather(-1, index)
        return sum((gs["g_" + n] * o[n]).sum() for n in ("logprob", "entropy", "lse")) + (g_top * o["top"]).sum()

    d = L.token_logprobs_grad(x, tok, temperature, **gs, g_top=g_top, top_index=index)
    assert (d - _difference(f, x)).abs().max() < 1e-8


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("temperature", [1.0, 1.5])
def test_oracle_distill_gradient_against_differences(tail, temperature):
    g = torch.Generator().manual_seed(2)
    x = torch.randn(4, 11, generator=g, dtype=torch.float64)
    index = torch.tensor([[3, 1, 7], [0, -1, 10], [5, 5, 2], [-1, -1, -1]])  # empty and repeated slots
    teacher = torch.log_softmax(torch.randn(4, 4, generator=g, dtype=torch.float64), -1)[:, :3]
    weight = torch.tensor([1.0, 0.5, 2.0, 1.0])
    f = lambda x: L.distill(x, index, teacher, weight, temperature, tail).sum()  # noqa: E731
    d = L.distill_grad(x, index, teacher, weight, temperature, tail)
    assert (d - _difference(f, x)).abs().max() < 1e-8


def test_oracle_order():
    nan, inf = float("nan"), float("inf")
    x = torch.tensor([[1.0, inf, nan, -0.0, 0.0, nan, -inf, 1.0]])
    assert L.order(x, 8).tolist() == [[2, 5, 1, 0, 7, 3, 4, 6]]


def _s(*v):
    return (ctypes.c_int64 * len(v))(*v)


def _lib():
    from kernels import sm100_logits

    return sm100_logits._lib()


def test_token_logprobs_entries_refuse_on_the_host():
    lib = _lib()
    s = _s(0, 256)

    def fwd(dtype=0, outer=1, inner=4, V=256, K=0, T=1.0, tokens=None, logits=None, logprob=None):
        return lib.bdh_token_logprobs(logits, dtype, s, tokens, s, -100, logprob, None, None, None,
                                      None, None, outer, inner, V, K, T, None)

    for kw, word in (({"dtype": 5}, b"dtype"), ({"inner": -1}, b"negative"), ({"V": 0}, b"vocabulary"),
                     ({"V": 1 << 31}, b"vocabulary"), ({"outer": 1 << 20, "inner": 1 << 20}, b"rows"),
                     ({"K": 129}, b"BDH_TOP_MAX"), ({"K": 9, "V": 8}, b"longer"), ({"T": 0.0}, b"temperature"),
                     ({"T": -1.0}, b"temperature"), ({"T": float("nan")}, b"temperature"),
                     ({"T": float("inf")}, b"temperature"), ({}, b"logits is null"),
                     ({"logits": 1 << 12, "tokens": 1 << 12}, b"come together"),
                     ({"logits": 1 << 12, "K": 3}, b"top_logprob")):
        assert fwd(**kw) == 1, kw
        assert word in lib.bdh_last_error(), (kw, lib.bdh_last_error())
    assert fwd(inner=0) == 0  # nothing to do

    def bwd(stats=1 << 12, entropy=None, tokens=None, glp=None, gen=None, gtop=None, K=0, inner=4):
        return lib.bdh_token_logprobs_bwd(1 << 12, 0, s, tokens, s, -100, stats, entropy, None, glp, s,
                                          None, s, gen, s, gtop, 1 << 12, s, 1, inner, 256, K, 1.0, None)

    for kw, word in (({"stats": None}, b"stats"), ({"gen": 1 << 12}, b"entropy"),
                     ({"glp": 1 << 12}, b"tokens"), ({"gtop": 1 << 12, "K": 2}, b"top_index")):
        assert bwd(**kw) == 1, kw
        assert word in lib.bdh_last_error()
    assert bwd(inner=0) == 0


def test_distill_entries_refuse_on_the_host():
    lib = _lib()
    s, s3 = _s(0, 256), _s(0, 4, 1)

    def fwd(dtype=0, inner=4, V=256, K=4, T=1.0, index=1 << 12):
        return lib.bdh_distill_topk(1 << 12, dtype, s, index, s3, 1 << 12, s3, None, s, 1 << 12, None,
                                    None, s, 1, inner, V, K, T, 0, None)

    for kw, word in (({"dtype": 2}, b"dtype"), ({"K": 0}, b"at least one"), ({"K": 200}, b"BDH_TOP_MAX"),
                     ({"V": 2097153}, b"BDH_DISTILL_VOCAB_MAX"),
                     ({"V": -3}, b"negative"), ({"T": 0.0}, b"temperature"), ({"index": None}, b"null")):
        assert fwd(**kw) == 1, kw
        assert word in lib.bdh_last_error()
    assert fwd(inner=0) == 0
    rc = lib.bdh_distill_topk_bwd(1 << 12, 0, s, 1 << 12, s3, 1 << 12, s3, None, s, None, 1 << 12, s,
                                  1 << 12, s, 1, 4, 256, 4, 1.0, 0, None)
    assert rc == 1 and b"stats" in lib.bdh_last_error()


def test_cpu_tensors_are_refused():
    import kernels
    from kernels import sm100_logits

    x, idx, lp = torch.zeros(2, 8), torch.zeros(2, 3, dtype=torch.long), torch.zeros(2, 3)
    for f in (lambda: kernels.token_logprobs(x), lambda: kernels.distill_topk_loss(x, idx, lp),
              lambda: kernels.distill_topk_loss_grad(x, idx, lp),
              lambda: sm100_logits.token_logprobs(x), lambda: sm100_logits.distill_topk(x, idx, lp)):
        with pytest.raises(RuntimeError, match="requires CUDA tensors"):
            f()


def test_the_teacher_is_a_constant():
    import kernels

    x, idx = torch.zeros(2, 8), torch.zeros(2, 3, dtype=torch.long)
    lp = torch.zeros(2, 3, requires_grad=True)
    with pytest.raises(ValueError, match="constants"):
        kernels.distill_topk_loss(x, idx, lp)
    with pytest.raises(ValueError, match="constants"):
        kernels.distill_topk_loss_grad(x, idx, lp.detach(), weight=torch.ones(2, requires_grad=True))
