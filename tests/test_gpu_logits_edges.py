"""The operators on logits at the ends of their ranges, on a B200: temperatures, the widest vocabularies,
lists that hold all of the mass that a mask leaves, results that are kept or saved, calls from several
threads, and what has to be refused or to leave nothing behind.

Bounds are those of test_gpu_logits.py (``rel(V)`` for a row's sum, 2.5e-7 of a figure's size for its
roundings), with sizes taken over the tokens that have probability."""

import ctypes
import io
import math
import threading

import pytest
import torch

import kernels
import logits_oracle as L
from kernels import sm100_logits
from test_gpu_logits import DT, check_grad, close, lists, make, many_rows, rel, tokens

pytestmark = pytest.mark.gpu

BINDINGS = ["ext", "ctypes"]


def use(binding, monkeypatch):
    monkeypatch.setenv("BDH_SM100_EXT", "1" if binding == "ext" else "0")


# ------------------------------------------------------------------------------ temperatures
def steps_of(T, rows, V, dtype, seed):
    """Rows whose logits are whole steps of T / 2 at or below 0 (both types hold them, and 1 / T, exactly),
    40 at most; of every third row five open tokens, of the others three in four; the rest masked by minus
    infinity, the type's lowest value or 2^30 steps. Returns the logits and which tokens are open."""
    g = torch.Generator().manual_seed(seed)
    x = -torch.randint(41, (rows, V), generator=g).double() * (T / 2)
    is_open = torch.rand(rows, V, generator=g) < 0.75
    few = torch.zeros(rows, V, dtype=torch.bool)
    few.scatter_(1, torch.rand(rows, V, generator=g).topk(5, dim=1).indices, True)
    is_open[::3] = few[::3]
    low = torch.finfo(dtype).min
    mask = torch.tensor([-math.inf, low, max(low, -T * 2.0 ** 29)])[torch.arange(rows) % 3].double()
    x = torch.where(is_open, x, mask.unsqueeze(1))
    return x.to(dtype), is_open


def logprobs_at(T, rows, V, dtype):
    x, is_open = steps_of(T, rows, V, DT[dtype], V)
    tok = is_open.float().argmax(1)
    tok[1::4] = (is_open.size(1) - 1) - is_open.flip(1).float().argmax(1)[1::4]  # the last open one
    z = x.cuda().requires_grad_(True)
    r = kernels.token_logprobs(z, tok.cuda(), top_k=5, temperature=T)
    ref = L.token_logprobs(x.float(), tok, 5, T)
    big = 2.5e-7 * (1 + 20)
    close(r.lse.detach(), ref["lse"], rel(V) + big)
    close(r.logprob.detach(), ref["logprob"], rel(V) + 2 * big)
    close(r.entropy.detach(), ref["entropy"], 2 * rel(V) * (1 + math.log(V)))
    assert torch.equal(r.top_index.cpu(), ref["top_index"])
    close(r.top_logprob.detach(), ref["top_logprob"], rel(V) + 2 * big)
    up = torch.randn(2, rows, generator=torch.Generator().manual_seed(3))
    (d,) = torch.autograd.grad([r.logprob, r.entropy], z, [up[0].cuda(), up[1].cuda()])
    want = L.token_logprobs_grad(x.float(), tok, T, g_logprob=up[0], g_entropy=up[1])
    check_grad(d, want, up.abs().sum(0) / T, V, DT[dtype])


ENDS = [2.0 ** -99, 2.0 ** -60, 2.0 ** -30, 2.0 ** -26, 2.0 ** 60, 2.0 ** 80, 2.0 ** 93, 2.0 ** 98, 2.0 ** 99]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T", ENDS)
@pytest.mark.parametrize("V", [300, 1000, 2048, 40001])
def test_logprobs_at_the_ends_of_the_temperatures(V, T, dtype):
    logprobs_at(T, 6, V, dtype)


@pytest.mark.parametrize("T", [2.0 ** -99, 2.0 ** -30, 2.0 ** 98])
@pytest.mark.parametrize("rows,V,dtype", [(0, 2000, "bf16"), (0, 2000, "f32"), (300, 20011, "bf16"), (300, 33000, "f32")])
def test_logprobs_of_many_rows_at_the_ends_of_the_temperatures(rows, V, dtype, T):
    logprobs_at(T, rows or many_rows(), V, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T", ENDS)
@pytest.mark.parametrize("rows,V", [(6, 300), (6, 1000), (0, 2000), (6, 40001)])
def test_distillation_at_the_ends_of_the_temperatures(rows, V, T, dtype):
    rows = rows or many_rows()
    x, is_open = steps_of(T, rows, V, DT[dtype], V + 1)
    index = is_open.float().topk(4, dim=1).indices  # open tokens
    _, lp = lists((rows,), V, 4, seed=V, empty=False)
    for tail in (False, True):
        want, dwant = L.distill(x.float(), index, lp, None, T, tail), L.distill_grad(x.float(), index, lp, None, T, tail)
        bound = (2 * rel(V) + 1e-6 * (1 + 2 * 20)) * 1.2
        loss, d = kernels.distill_topk_loss_grad(x.cuda(), index.cuda(), lp.cuda(), temperature=T, tail=tail)
        close(loss, want, bound)
        check_grad(d, dwant, torch.full((rows,), 2 / T), V, DT[dtype])
        z = x.cuda().requires_grad_(True)
        loss = kernels.distill_topk_loss(z, index.cuda(), lp.cuda(), temperature=T, tail=tail)
        close(loss.detach(), want, bound)
        (d,) = torch.autograd.grad(loss.sum(), z)
        check_grad(d, dwant, torch.full((rows,), 2 / T), V, DT[dtype])
