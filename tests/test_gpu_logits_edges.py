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


# ---------------------------------------------------------- a list of all that a mask leaves
def masked_to(index, V, dtype, mask, seed):
    """Students that allow the listed tokens alone."""
    x = torch.full((index.size(0), V), mask, dtype=dtype)
    g = torch.Generator().manual_seed(seed)
    return x.scatter_(1, index, (torch.randn(index.shape, generator=g) * 2).to(dtype))


MASKED = [("f32", -math.inf), ("bf16", -math.inf), ("f32", torch.finfo(torch.float32).min), ("bf16", -1e9),
          ("f32", -1e4)]


@pytest.mark.parametrize("dtype,mask", MASKED)
@pytest.mark.parametrize("rows,V,k", [(40, 200, 12), (40, 500, 30), (40, 1000, 60), (0, 1100, 12), (40, 5000, 100),
                                      (300, 20011, 20), (40, 131072, 12)])
def test_a_list_of_every_allowed_token_has_no_rest(rows, V, k, dtype, mask):
    """The list's mass is 1 but for its rounding in fp32, and the student has nothing else to give."""
    rows = rows or many_rows()
    index, lp = lists((rows,), V, k, seed=V, empty=False, outside=0.0)
    assert 0 < ((1 - lp.exp().sum(-1)) > 0).sum() < rows  # (rounded to either side)
    x = masked_to(index, V, DT[dtype], mask, 1)
    want = L.distill(x.float(), index, lp, None, 1.0, True)
    p = torch.log_softmax(x.gather(1, index).double(), -1)  # the definition over the allowed tokens alone
    assert torch.allclose(want, (lp.double().exp() * (lp.double() - p)).sum(-1), rtol=0, atol=2e-5)
    bound = (2 * rel(V) + 1e-6 * (1 + 2 * 10)) * 1.2
    dwant = L.distill_grad(x.float(), index, lp, None, 1.0, True)
    loss, d = kernels.distill_topk_loss_grad(x.cuda(), index.cuda(), lp.cuda(), tail=True)
    close(loss, want, bound)
    check_grad(d, dwant, torch.full((rows,), 2.0), V, DT[dtype])
    z = x.cuda().requires_grad_(True)
    loss = kernels.distill_topk_loss(z, index.cuda(), lp.cuda(), tail=True)
    close(loss.detach(), want, bound)
    (d,) = torch.autograd.grad(loss.sum(), z)
    check_grad(d, dwant, torch.full((rows,), 2.0), V, DT[dtype])
    close(kernels.distill_topk_loss(x.cuda(), index.cuda(), lp.cuda(), tail=True), want, bound)


@pytest.mark.parametrize("V", [256, 3000, 70001])
def test_a_constrained_teacher_and_its_student(V):
    """A teacher's lists as token_logprobs makes them, longer than what the teacher allows (the places after
    its last token hold log probabilities of -inf): a student equal to it has no loss and no gradient."""
    x = masked_to(torch.stack([torch.randperm(V)[:9] for _ in range(200)]), V, torch.float32, -math.inf, 2).cuda()
    for T in (1.0, 1.7):
        top = kernels.token_logprobs(x, top_k=16, temperature=T)
        assert (top.top_logprob[:, 9:] == -math.inf).all()
        loss, d = kernels.distill_topk_loss_grad(x, top.top_index, top.top_logprob, temperature=T, tail=True)
        assert loss.abs().max().item() < 4 * rel(V) and d.abs().max().item() < 4 * rel(V)


@pytest.mark.parametrize("rows,V", [(5, 300), (0, 1100), (5, 30000)])
def test_a_rest_beyond_rounding_that_the_student_forbids_costs_infinitely(rows, V):
    rows = rows or many_rows()
    index, lp = lists((rows,), V, 10, empty=False, outside=1e-4)
    x = masked_to(index, V, torch.float32, -math.inf, 3)
    loss, d = kernels.distill_topk_loss_grad(x.cuda(), index.cuda(), lp.cuda(), tail=True)
    assert (loss == math.inf).all() and torch.isfinite(d).all()
    check_grad(d, L.distill_grad(x, index, lp, None, 1.0, True), torch.full((rows,), 2.0), V, torch.float32)


# ------------------------------------------------------------------------ wide vocabularies
@pytest.mark.parametrize("rows,V,dtype", [(230, 1000003, "f32"), (230, 2097152, "f32"), (230, 2097152, "bf16"),
                                          (230, 1900001, "bf16"), (130, 2097152, "f32"), (3, 2097152, "f32")])
def test_distillation_over_the_widest_vocabularies(rows, V, dtype):
    """One row of logits seen many times, each with a list of its own."""
    x = make((1,), V, DT[dtype], seed=1).expand(rows, V)
    at = torch.randint(V, (rows, 7), generator=torch.Generator().manual_seed(2))
    at[0, :3] = torch.tensor([0, V - 1, V // 2])
    _, lp = lists((rows,), 100, 7, empty=False)
    loss = kernels.distill_topk_loss(x, at.cuda(), lp.cuda(), tail=True)
    z = x.detach().requires_grad_(True)
    loss2 = kernels.distill_topk_loss(z, at.cuda(), lp.cuda(), tail=True)
    assert torch.equal(loss, loss2.detach())
    (d,) = torch.autograd.grad(loss2.sum(), z)
    look = [0, rows // 2, rows - 1]
    xc = x[look].float().cpu()
    want, dwant = (f(xc, at[look], lp[look], None, 1.0, True) for f in (L.distill, L.distill_grad))
    close(loss[look], want, (2 * rel(V) + 1e-6 * (1 + 2 * 20)) * 1.2)
    check_grad(d[look], dwant, torch.full((3,), 2.0), V, DT[dtype])
    del d
    loss3, d = kernels.distill_topk_loss_grad(x, at.cuda(), lp.cuda(), tail=True)
    close(loss3[look], want, (2 * rel(V) + 1e-6 * (1 + 2 * 20)) * 1.2)
    check_grad(d[look], dwant, torch.full((3,), 2.0), V, DT[dtype])


# ------------------------------------------------------------------- results kept and saved
@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("binding", BINDINGS)
def test_results_can_be_saved_and_do_not_hold_the_lists(binding, grad, monkeypatch):
    use(binding, monkeypatch)
    x = make((4, 5), 300, torch.float32).requires_grad_(grad)
    r = kernels.token_logprobs(x, tokens((4, 5), 300).cuda(), top_k=6)
    kept = {name: t.detach() for name, t in r._asdict().items()}
    f = io.BytesIO()
    torch.save(kept, f)
    f.seek(0)
    back = torch.load(f)
    assert back.keys() == kept.keys()
    figures = ("logprob", "entropy", "lse")  # (these three may share a storage)
    for name, t in kept.items():
        assert torch.equal(back[name], t)
        own = t.numel() * t.element_size()
        assert t.untyped_storage().nbytes() <= (3 * (own + 12) if name in figures else own), name
    shared = {kept[name].untyped_storage().data_ptr() for name in figures}
    lists_ = {kept[name].untyped_storage().data_ptr() for name in ("top_logprob", "top_index")}
    assert len(lists_) == 2 and not lists_ & shared


# -------------------------------------------------------------------- forward-mode derivatives
@pytest.mark.parametrize("binding", BINDINGS)
def test_forward_mode_derivatives_are_refused(binding, monkeypatch):
    use(binding, monkeypatch)
    from torch.autograd import forward_ad as fw

    x, tok = make((3,), 50, torch.float32), tokens((3,), 50).cuda()
    index, lp = (t.cuda() for t in lists((3,), 50, 4))
    w = torch.rand(3, device="cuda")
    with fw.dual_level():
        dual = lambda t: fw.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: kernels.token_logprobs(dual(x), tok, top_k=2),
                     lambda: kernels.token_logprobs(dual(x)[:, 1:]),
                     lambda: kernels.distill_topk_loss(dual(x), index, lp),
                     lambda: kernels.distill_topk_loss(x, index, dual(lp)),
                     lambda: kernels.distill_topk_loss(x, index, lp, weight=dual(w)),
                     lambda: kernels.distill_topk_loss_grad(dual(x), index, lp),
                     lambda: kernels.distill_topk_loss_grad(x, index, dual(lp)),
                     lambda: kernels.distill_topk_loss_grad(x, index, lp, weight=dual(w))):
            with pytest.raises(RuntimeError, match="forward"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward"):
                call()
        z = x.clone().requires_grad_(True)
        for call in (lambda: kernels.token_logprobs(dual(z), tok), lambda: kernels.distill_topk_loss(dual(z), index, lp)):
            with pytest.raises(RuntimeError):
                call()
        # a tangent that comes with the upstream gradient
        r = kernels.token_logprobs(z, tok, top_k=2)
        for y in (r.logprob, r.entropy, r.lse, r.top_logprob, kernels.distill_topk_loss(z, index, lp)):
            with pytest.raises(RuntimeError, match="forward"):
                torch.autograd.grad(y, z, dual(torch.ones_like(y.detach())))
        # torch.func's wrappers have no memory to read
        for y in (lambda z: kernels.token_logprobs(z, tok).logprob, lambda z: kernels.distill_topk_loss_grad(z, index, lp)[0]):
            with pytest.raises(RuntimeError):
                torch.func.jvp(y, (x,), (x,))
        # nothing else is refused there
        r = kernels.token_logprobs(x, tok, top_k=2)
    for a, b in zip(r, kernels.token_logprobs(x, tok, top_k=2)):
        assert torch.equal(a, b)


# ------------------------------------------------------------------- errors left behind
def _distill_by_c(x, index, lp, loss, stream):
    rows, V = x.shape
    k = index.size(-1)
    s2, s3 = (ctypes.c_int64 * 2)(0, V), (ctypes.c_int64 * 3)(0, k, 1)
    return sm100_logits._lib().bdh_distill_topk(
        x.data_ptr(), 0, s2, index.data_ptr(), s3, lp.data_ptr(), s3, None, s2, loss.data_ptr(), None, None, s2, 1,
        rows, V, k, 1.0, 0, stream)


def _logprobs_by_c(x, lse, stream, stats=None, k=0, top=None, index=None):
    rows, V = x.shape
    s2 = (ctypes.c_int64 * 2)(0, V)
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    return sm100_logits._lib().bdh_token_logprobs(
        x.data_ptr(), 0, s2, None, s2, -100, None, lse.data_ptr(), None, ptr(stats), ptr(top), ptr(index), 1, rows, V,
        k, 1.0, stream)


@pytest.mark.parametrize("rows,V", [(4, 300), (0, 1100), (300, 20011), (2, 70001)])
def test_a_refused_launch_leaves_the_next_call_alone(rows, V):
    """The runtime refuses a launch on the legacy stream while a blocking stream records a graph. The call
    says so, and the next one, which is valid, goes through."""
    rows = rows or many_rows()
    x = make((rows,), V, torch.float32)
    index, lp = (t.cuda() for t in lists((rows,), 40, 5, empty=False))
    wants = kernels.distill_topk_loss(x, index, lp), kernels.token_logprobs(x).lse
    out = torch.zeros(rows, device="cuda")
    side = torch.cuda.Stream()  # (neither blocks the recording nor is blocked by it)
    rt = ctypes.CDLL("libcudart.so.12")
    rt.cudaStreamBeginCapture.argtypes = [ctypes.c_void_p, ctypes.c_int]
    rt.cudaStreamEndCapture.argtypes = [ctypes.c_void_p, ctypes.c_void_p]
    rt.cudaStreamDestroy.argtypes = [ctypes.c_void_p]
    error = sm100_logits._lib().bdh_last_error
    for call, want in ((lambda s: _distill_by_c(x, index, lp, out, s), wants[0]), (lambda s: _logprobs_by_c(x, out, s), wants[1])):
        stream, graph = ctypes.c_void_p(), ctypes.c_void_p()
        assert rt.cudaStreamCreate(ctypes.byref(stream)) == 0
        torch.cuda.synchronize()
        assert rt.cudaStreamBeginCapture(stream, 2) == 0  # relaxed: what else this thread does is its own affair
        try:
            rc, message = call(None), error()
        finally:
            rt.cudaStreamEndCapture(stream, ctypes.byref(graph))  # (invalid by now: no graph)
            rt.cudaGetLastError()
            rt.cudaStreamDestroy(stream)
        assert rc == 2 and b"captur" in message, (rc, message)
        out.zero_()
        torch.cuda.synchronize()
        assert call(side.cuda_stream) == 0, error()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


# ------------------------------------------------------------------------- host threads
@pytest.mark.parametrize("op", ["token_logprobs", "distill_topk"])
def test_calls_of_several_threads_do_not_limit_one_another(op):
    """The same kernel with more and with less shared memory, from host threads at once (the C entries: a
    binding's own time would keep them apart)."""
    if op == "token_logprobs":
        x = make((1,), 1500000, torch.float32)
        tops = {k: (torch.zeros(1, k, device="cuda"), torch.zeros(1, k, dtype=torch.long, device="cuda")) for k in (128, 1)}
        calls = [(lambda s, k=k, out=torch.zeros(1, device="cuda"): _logprobs_by_c(x, out, s, None, k, *tops[k]))
                 for k in (128, 1, 128, 1)]
    else:
        index, lp = (t.cuda() for t in lists((1,), 1000, 9, empty=False))
        xs = [make((1,), V, torch.float32) for V in (2097152, 1700000)]
        calls = [(lambda s, x=x, out=torch.zeros(1, device="cuda"): _distill_by_c(x, index, lp, out, s)) for x in xs + xs]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    failed, gate = [], threading.Barrier(len(calls))

    def work(n):
        s = streams[n].cuda_stream
        gate.wait(60)
        for _ in range(10000):
            if calls[n](s) != 0:
                failed.append(sm100_logits._lib().bdh_last_error())
                return

    threads = [threading.Thread(target=work, args=(n,)) for n in range(len(calls))]
    for t in threads:
        t.start()
    for t in threads:
        t.join(300)
    torch.cuda.synchronize()
    assert not failed, failed


# ---------------------------------------------------------------------------- alignment
@pytest.mark.parametrize("rows,V,k", [(5, 200, 0), (5, 200, 4), (5, 1000, 3), (0, 1100, 0), (0, 1100, 5), (300, 20011, 0),
                                      (2, 70001, 6)])
def test_statistics_at_any_float(rows, V, k):
    """The C entry writes a row's statistics wherever a float may lie."""
    rows = rows or many_rows()
    x = make((rows,), V, torch.float32)
    top, index = torch.empty(rows, max(k, 1), device="cuda"), torch.empty(rows, max(k, 1), dtype=torch.long, device="cuda")
    want = sm100_logits.token_logprobs(x, None, k, 1.0, -100, True)[5]
    room = torch.full((2 * rows + 2,), 7.0, device="cuda")
    lse = torch.empty(rows, device="cuda")
    rc = _logprobs_by_c(x, lse, torch.cuda.current_stream().cuda_stream, room[1:], k, top, index)
    torch.cuda.synchronize()
    assert rc == 0 and torch.equal(room[1:-1].view(rows, 2), want) and room[0] == 7.0 and room[-1] == 7.0
