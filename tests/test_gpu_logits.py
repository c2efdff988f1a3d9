"""The operators on logits on a B200 against their 64-bit forms (oracle/logits_oracle.py): sizes from
one token up, odd sizes and alignments, masks, ties, NaN and infinities, strides, streams, graphs.

Bounds. EPS = 2^-24. A row's sum of exponentials is off by a relative ``rel(V)``: each exponent
(z - m) log2(e) / T has three roundings (|t| <= 25 for terms that count: 25 * 3 EPS * ln 2 = 3e-6),
ex2.approx 2^-22, and the running sums' roundings, which add like a random walk over at most V / 32
terms in a row, four deviations taken. A log probability or loss adds roundings of figures of the
logits' size; an entropy and a gradient multiply by at most 1 + ln V. bf16 gradients are rounded
once to 8 significant bits: 2^-8 of the value. Gradients of a row are compared elementwise against the size of its
upstream gradients and as a whole (Frobenius)."""

import math

import pytest
import torch

import kernels
import logits_oracle as L
from kernels import sm100_ext, sm100_logits

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -24
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def rel(V):
    return 4e-6 + 4 * math.sqrt(V / 32) * EPS


def close(got, ref, atol):
    """Within ``atol`` (a number, or one per row); NaN and infinities in the same places, a figure
    past the range of fp32 as the infinity that fp32 has for it."""
    got, ref = got.double().cpu(), ref.float().double()
    assert got.shape == ref.shape
    atol = torch.as_tensor(atol, dtype=torch.float64)
    if atol.dim() < got.dim():
        atol = atol.unsqueeze(-1) if atol.dim() else atol.expand(got.shape)
    same = (got == ref) | (torch.isnan(got) & torch.isnan(ref))
    off = torch.where(same, 0.0, (got - ref).abs())
    assert not torch.isnan(off).any(), "NaN or infinity in other places"
    assert (off <= atol).all(), (off - atol).max().item()


def make(shape, V, dtype, seed=0, offset=0, scale=3.0):
    """Logits (*shape, V) starting ``offset`` elements into an allocation."""
    g = torch.Generator().manual_seed(seed)
    n = math.prod(shape) * V
    buf = torch.empty(n + offset, dtype=dtype, device="cuda")
    x = torch.randn(*shape, V, generator=g) * scale
    buf[offset:].copy_(x.reshape(-1))
    return buf[offset:].view(*shape, V)


def tokens(shape, V, seed=1):
    return torch.randint(V, shape, generator=torch.Generator().manual_seed(seed))


def check_forward(x, tok, k, T, r=None):
    V = x.size(-1)
    r = r or kernels.token_logprobs(x, None if tok is None else tok.cuda(), top_k=k, temperature=T)
    ref = L.token_logprobs(x.float().cpu(), tok, k, T)
    xc = x.float().cpu().double()
    big = 2.5e-7 * (1 + torch.where(xc.abs() < math.inf, xc, 0.0).abs().amax(-1) / T)  # a row's own size
    close(r.lse, ref["lse"], rel(V) + big)
    close(r.entropy, ref["entropy"], 2 * rel(V) * (1 + math.log(V)))
    if tok is not None:
        close(r.logprob, ref["logprob"], rel(V) + 2 * big)
    else:
        assert r.logprob is None
    if k:
        assert torch.equal(r.top_index.cpu(), ref["top_index"])
        close(r.top_logprob, ref["top_logprob"], rel(V) + 2 * big)
    else:
        assert r.top_index is None and r.top_logprob is None


SIZES = [1, 2, 5, 31, 32, 33, 64, 255, 256, 257, 511, 1000, 1023, 1024, 1025, 2048, 4099, 8192,
         16385, 50021, 131072, 131073]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", SIZES)
def test_forward_over_sizes(V, dtype):
    shape = (2, 37) if V <= 8192 else (3,)
    for n, (k, T, offset) in enumerate([(min(V, 5), 1.0, 0), (min(V, 64), 0.7, 1), (0, 2.0, 3)]):
        x = make(shape, V, DT[dtype], seed=n, offset=offset)
        check_forward(x, tokens(shape, V), k, T)


@pytest.mark.parametrize("rows", [1, 2, 7, 64, 200, 700])
def test_forward_splits_rows_by_their_number(rows):
    x = make((rows,), 20011, torch.bfloat16, seed=rows)
    check_forward(x, tokens((rows,), 20011), 9, 1.0)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V,k", [(1, 1), (7, 7), (128, 128), (129, 128), (256, 1), (256, 20), (256, 128),
                                 (1500, 128), (4096, 33), (70001, 128), (131072, 1), (131072, 100)])
def test_top_list_lengths(V, k, dtype):
    for rows in (1, 40):
        check_forward(make((rows,), V, DT[dtype], seed=k), None, k, 1.0)


def patterns(V, dtype):
    """Rows that a search for the largest values can trip over."""
    i = torch.arange(V)
    g = torch.Generator().manual_seed(V)
    rows = {
        "equal": torch.zeros(V),
        "rising": i.float() / 64,
        "falling": -i.float() / 64,
        "few values": (i * 7919 % 3).float(),
        "two levels": (torch.rand(V, generator=g) < 0.3).float() * 2,
        "signed zeros": torch.where(i % 3 == 0, -0.0, 0.0),
        "one finite": torch.where(i == V // 2, 1.5, -math.inf),
        "three finite": torch.where((i * 3 % max(V, 1) < 3) & (i > V // 3), 0.25, -math.inf),
        "lowest": torch.full((V,), torch.finfo(dtype).min),
        "all but one lowest": torch.where(i == V - 1, 3.0, torch.finfo(dtype).min),
        "huge": torch.randn(V, generator=g) * 1e4,
        "far up": torch.randn(V, generator=g) + 300.0,
        "none": torch.full((V,), -math.inf),
    }
    for step in (256, 1024, 2048, 4096, 8192):  # the large values all in one thread's share
        rows[f"every {step}th"] = torch.where((i % step) // 8 == 3, 5.0 + i / V, torch.randn(V, generator=g))
    return rows


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [3, 200, 256, 1024, 3001, 65536, 100003])
def test_forward_of_awkward_rows(V, dtype):
    rows = patterns(V, DT[dtype])
    x = torch.stack(list(rows.values())).to(DT[dtype])
    tok = tokens((x.size(0),), V)
    for k in sorted({1, min(V, 20), min(V, 128)}):
        check_forward(x.cuda(), tok, k, 1.0)
    for name, row in rows.items():  # a single row is divided another way
        check_forward(row.to(DT[dtype]).cuda(), tok[0], min(V, 11), 0.5)


@pytest.mark.parametrize("V", [50, 300, 70000])
def test_nan_and_infinity(V):
    x = make((6,), V, torch.float32)
    x[0, V // 2] = math.nan
    x[1, 3] = math.inf
    x[2, 5:9] = math.nan
    x[3, 1::2] = -math.inf
    x[4] = math.nan
    r = kernels.token_logprobs(x, torch.full((6,), 4, device="cuda"), top_k=8)
    for figure in (r.lse, r.entropy, r.logprob):
        assert torch.isnan(figure).tolist() == [True, True, True, False, True, False]
    assert torch.equal(r.top_index.cpu(), L.order(x.cpu(), 8))
    check_forward(x[3:4], torch.tensor([2]), 8, 1.0)


def test_tokens_left_out_and_out_of_range():
    x = make((5,), 300, torch.float32)
    tok = torch.tensor([-100, -1, 300, 1 << 40, 299])
    r = kernels.token_logprobs(x, tok.cuda())
    assert r.logprob[0].item() == 0.0
    assert torch.isnan(r.logprob[1:4]).all() and not torch.isnan(r.logprob[4])
    r = kernels.token_logprobs(x, tok.cuda(), ignore_index=300)
    assert torch.isnan(r.logprob[0]) and r.logprob[2].item() == 0.0


def test_row_strides_and_leading_shapes():
    V = 777
    base = make((3, 9), V, torch.bfloat16)
    tok = tokens((3, 9), V)
    shifted = base[:, :-1]
    check_forward(shifted, tok[:, 1:], 4, 1.0,
                  kernels.token_logprobs(shifted, tok.cuda()[:, 1:], top_k=4))
    check_forward(base[::2, 1::3], tok[::2, 1::3], 4, 1.0)
    check_forward(base.transpose(0, 1), tok.t(), 4, 1.0)
    check_forward(base[1, 2], tok[1, 2], 4, 1.0)  # no leading dimension
    wide = make((4, 5), 2 * V, torch.float32)
    check_forward(wide[..., 5:V], tokens((4, 5), V - 5), 3, 1.0)  # a slice of the vocabulary
    check_forward(wide[..., ::2], tokens((4, 5), V), 3, 1.0)  # strided vocabulary: copied
    four = make((2, 3, 2, 2), 65, torch.float32)
    check_forward(four, tokens((2, 3, 2, 2), 65), 3, 1.0)
    check_forward(four[:, :, :, :1], tokens((2, 3, 2, 1), 65), 3, 1.0)
    row = make((1,), V, torch.float32).expand(6, V)  # one row seen six times
    check_forward(row, tokens((6,), V), 3, 1.0)
    check_forward(base, tok.int(), 2, 1.0, kernels.token_logprobs(base, tok.int().cuda(), top_k=2))


@pytest.mark.parametrize("shape", [(0,), (0, 5), (4, 0), (2, 0, 3)])
def test_no_rows(shape):
    x = torch.empty(*shape, 33, device="cuda", requires_grad=True)
    tok = torch.empty(shape, dtype=torch.long, device="cuda")
    r = kernels.token_logprobs(x, tok, top_k=2)
    assert r.lse.shape == shape and r.top_index.shape == (*shape, 2)
    (d,) = torch.autograd.grad(r.logprob.sum(), x)
    assert d.shape == x.shape
    idx, lp = tok.unsqueeze(-1).expand(*shape, 3), torch.empty(*shape, 3, device="cuda")
    loss = kernels.distill_topk_loss(x, idx, lp)
    (d,) = torch.autograd.grad(loss.sum(), x)
    assert loss.shape == shape and d.shape == x.shape


# ------------------------------------------------------------------------------ gradients
def check_grad(got, ref, size, V, dtype):
    """``size``: per-row sum of the upstream gradients' magnitudes over the temperature."""
    f = 2 * (rel(V) + 4e-6) * (1 + math.log(V))
    round_ = 2.0 ** -8 * 1.01 if dtype == torch.bfloat16 else 0.0
    got, ref = got.double().cpu(), ref.double()
    assert got.shape == ref.shape and not torch.isnan(got).any()
    bound = f * size.double().unsqueeze(-1) + round_ * ref.abs()
    assert ((got - ref).abs() <= bound + 1e-38).all(), ((got - ref).abs() - bound).max().item()
    n = ref.norm().item()
    assert (got - ref).norm().item() <= (f + round_) * n + 1e-30


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", SIZES)
def test_logprob_gradient_over_sizes(V, dtype):
    shape = (2, 19) if V <= 8192 else (3,)
    T, k = 0.8, min(V, 6)
    x = make(shape, V, DT[dtype], seed=3, offset=V % 3).requires_grad_(True)
    tok = tokens(shape, V)
    tok.view(-1)[0] = -100
    g = torch.Generator().manual_seed(4)
    up = {n: torch.randn(shape, generator=g) for n in ("logprob", "entropy", "lse")}
    up_top = torch.randn(*shape, k, generator=g)
    r = kernels.token_logprobs(x, tok.cuda(), top_k=k, temperature=T)
    outs = [r.logprob, r.entropy, r.lse, r.top_logprob]
    (d,) = torch.autograd.grad(outs, x, [up["logprob"].cuda(), up["entropy"].cuda(),
                                         up["lse"].cuda(), up_top.cuda()], retain_graph=True)
    xc = x.detach().float().cpu()
    ref = L.token_logprobs_grad(xc, tok, T, g_logprob=up["logprob"], g_entropy=up["entropy"],
                                g_lse=up["lse"], g_top=up_top, top_index=L.order(xc, k))
    size = (sum(v.abs() for v in up.values()) + up_top.abs().sum(-1)) / T
    assert d.dtype == x.dtype
    check_grad(d, ref, size, V, x.dtype)
    # each figure by itself, a broadcast upstream gradient
    (d,) = torch.autograd.grad(r.logprob.sum(), x, retain_graph=True)
    check_grad(d, L.token_logprobs_grad(xc, tok, T, g_logprob=torch.ones(shape)),
               torch.ones(shape) / T, V, x.dtype)
    (d,) = torch.autograd.grad(r.entropy.sum(), x)
    check_grad(d, L.token_logprobs_grad(xc, tok, T, g_entropy=torch.ones(shape)),
               torch.ones(shape) / T, V, x.dtype)


def test_logprob_gradient_of_awkward_rows():
    V = 3001
    rows = patterns(V, torch.float32)
    x = torch.stack(list(rows.values())).cuda().requires_grad_(True)
    tok = tokens((x.size(0),), V)
    for n, name in enumerate(rows):  # tokens with some probability: others have infinite log odds
        if "finite" in name or "lowest" in name:
            tok[n] = rows[name].argmax()
    r = kernels.token_logprobs(x, tok.cuda())
    g = torch.ones(x.size(0))
    (d,) = torch.autograd.grad([r.logprob, r.entropy], x, [g.cuda(), 0.5 * g.cuda()])
    ref = L.token_logprobs_grad(x.detach().cpu(), tok, g_logprob=g, g_entropy=0.5 * g)
    check_grad(d, ref, 1.5 * g, V, torch.float32)
    assert (d[list(rows).index("none")] == 0).all()


def test_logprob_gradient_of_a_token_out_of_range_is_loud():
    x = make((3,), 100, torch.float32).requires_grad_(True)
    r = kernels.token_logprobs(x, torch.tensor([5, 100, -7], device="cuda"))
    (d,) = torch.autograd.grad(r.logprob, x, torch.ones(3, device="cuda"))
    assert torch.isnan(d).all(-1).tolist() == [False, True, True]
    assert not torch.isnan(d[0]).any()


def test_logprob_gradient_of_shared_and_strided_logits():
    V = 301
    base = make((3, 8), V, torch.float32).requires_grad_(True)
    tok = tokens((3, 8), V)
    r = kernels.token_logprobs(base[:, :-1], tok.cuda()[:, 1:])
    (d,) = torch.autograd.grad(r.logprob.sum(), base)
    ref = L.token_logprobs_grad(base.detach().cpu()[:, :-1], tok[:, 1:], g_logprob=torch.ones(3, 7))
    assert (d[:, -1] == 0).all()
    check_grad(d[:, :-1], ref, torch.ones(3, 7), V, torch.float32)
    row = make((1,), V, torch.float32).requires_grad_(True)  # six uses of one row: their sum
    r = kernels.token_logprobs(row.expand(6, V), tok.view(-1)[:6].cuda())
    (d,) = torch.autograd.grad(r.logprob.sum(), row)
    ref = L.token_logprobs_grad(row.detach().cpu().expand(6, V), tok.view(-1)[:6], g_logprob=torch.ones(6))
    check_grad(d, ref.sum(0, keepdim=True), torch.full((1,), 6.0), V, torch.float32)


def test_gradients_against_differences():
    """Directional differences of the kernels' own figures along random u: with step h the fp32
    figures (~10 in size, summed over 4 rows) give an error of 8 * 40 EPS / (2 h) from rounding and
    h^2 |u|^3 from the third derivative; h = 2^-5 and |u| = 1 put both under 2e-3."""
    V, h = 400, 2.0 ** -5
    x = make((4,), V, torch.float32, scale=2.0)
    g = torch.Generator().manual_seed(9)
    tok = tokens((4,), V).cuda()
    idx = torch.randperm(V, generator=g)[:12].view(1, 12).expand(4, 12).cuda()
    lp = (torch.log_softmax(torch.randn(4, 13, generator=g), -1)[:, :12]).cuda()
    figures = {
        "logprob": lambda z: kernels.token_logprobs(z, tok).logprob.sum(),
        "entropy": lambda z: kernels.token_logprobs(z, tok).entropy.sum(),
        "lse": lambda z: kernels.token_logprobs(z, tok, temperature=0.5).lse.sum(),
        "distill": lambda z: kernels.distill_topk_loss(z, idx, lp).sum(),
        "distill tail": lambda z: kernels.distill_topk_loss(z, idx, lp, tail=True, temperature=2.0).sum(),
    }
    for name, f in figures.items():
        z = x.clone().requires_grad_(True)
        (d,) = torch.autograd.grad(f(z), z)
        for _ in range(3):
            u = torch.randn(4, V, generator=g).cuda()
            u += 4 * d / d.norm() * u.norm()  # not nearly at right angles to the gradient
            u /= u.norm()
            slope = ((f(x + h * u) - f(x - h * u)) / (2 * h)).item()
            assert abs(slope - (d * u).sum().item()) < 2e-3, name


# --------------------------------------------------------------------------- distillation
def lists(shape, V, k, seed=5, empty=True, outside=0.1):
    g = torch.Generator().manual_seed(seed)
    n = math.prod(shape)
    index = torch.stack([torch.randperm(V, generator=g)[:k] for _ in range(n)]).view(*shape, k)
    lp = torch.log_softmax(torch.randn(*shape, k, generator=g) * 2, -1) + math.log1p(-outside)
    if empty and k > 1:
        index = index.masked_fill(torch.rand(*shape, k, generator=g) < 0.15, -1)
    return index, lp


def check_distill(x, index, lp, weight, T, tail):
    V = x.size(-1)
    xc = x.detach().float().cpu()
    opts = {"weight": None if weight is None else weight.cuda(), "temperature": T, "tail": tail}
    loss, d = kernels.distill_topk_loss_grad(x.detach(), index.cuda(), lp.cuda(), **opts)
    w = torch.ones(x.shape[:-1]) if weight is None else weight.expand(x.shape[:-1])
    ref = L.distill(xc, index, lp, weight, T, tail)
    size = torch.where(xc.abs() < math.inf, xc, 0.0).abs().double().amax(-1)
    bound = (2 * rel(V) + 1e-6 * (1 + 2 * size / T)) * w.abs().max().item() * 1.2
    close(loss, ref, bound)
    dref = L.distill_grad(xc, index, lp, weight, T, tail)
    check_grad(d, dref, 2 * w.abs() / T, V, x.dtype)
    z = x.detach().requires_grad_(True)
    loss2 = kernels.distill_topk_loss(z, index.cuda(), lp.cuda(), **opts)
    close(loss2, ref, bound)
    assert torch.equal(loss2.detach(), kernels.distill_topk_loss(x.detach(), index.cuda(), lp.cuda(), **opts))
    up = torch.randn(x.shape[:-1], generator=torch.Generator().manual_seed(6))
    (d2,) = torch.autograd.grad(loss2, z, up.cuda())
    check_grad(d2, dref * up.double().unsqueeze(-1), 2 * w.abs() * up.abs() / T, V, x.dtype)
    (d3,) = torch.autograd.grad(kernels.distill_topk_loss(z, index.cuda(), lp.cuda(), **opts).sum(), z)
    check_grad(d3, dref, 2 * w.abs() / T, V, x.dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", SIZES)
def test_distill_over_sizes(V, dtype):
    shape = (2, 19) if V <= 8192 else (3,)
    for n, (k, T, tail, offset) in enumerate([(min(V, 5), 1.0, False, 0), (min(V, 16), 2.0, True, 1),
                                              (min(V, 100), 0.7, True, 2)]):
        x = make(shape, V, DT[dtype], seed=n, offset=offset)
        index, lp = lists(shape, V, k, seed=n)
        w = torch.rand(shape, generator=torch.Generator().manual_seed(n)) + 0.1
        w.view(-1)[1] = 0.0
        if tail and V < 3:  # the list can hold the whole vocabulary, or one token without mass
            index = index.clamp_min(0)
        check_distill(x, index, lp, w if n else None, T, tail)


@pytest.mark.parametrize("rows", [1, 2, 7, 64, 200, 700])
def test_distill_splits_rows_by_their_number(rows):
    x = make((rows,), 20011, torch.bfloat16, seed=rows)
    index, lp = lists((rows,), 20011, 24)
    check_distill(x, index, lp, None, 1.0, True)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("V", [300, 5000, 60001])
def test_distill_of_awkward_lists(V, tail):
    x = make((9,), V, torch.float32)
    index, lp = lists((9,), V, 8, empty=False)
    index[0] = -1                       # no slot
    index[1, 1:] = -1                   # one slot
    index[2] = torch.tensor([4, 4, 4, 9, 9, 2, 4, 9])  # repeated tokens
    index[3] = torch.arange(8)          # the row's head
    index[4] = torch.arange(V - 8, V)   # the row's end
    lp[5, 3:] = -math.inf               # slots of probability 0
    lp[6] = torch.log_softmax(lp[6], -1)  # everything in the list: r is a rounding's size
    x[7].masked_fill_(torch.rand(V, generator=torch.Generator().manual_seed(1)).cuda() < 0.5, -math.inf)
    x[7, index[7].cuda()] = 1.0
    x[8].fill_(-3.0e38)                 # a student without an opinion
    if tail:
        # the student leaves next to nothing outside the list, far below what fp32 holds of 1 - sum p
        x[3] -= 200.0
        x[3, :8] += 200.0
    check_distill(x, index, lp, None, 1.0, tail)
    check_distill(x, index, lp, torch.tensor(0.25), 1.5, tail)  # a weight without dimensions
    check_distill(x[None].expand(2, 9, V), index[None].expand(2, 9, 8), lp[None].expand(2, 9, 8),
                  torch.rand(1, 9).expand(2, 9), 1.0, tail)


def test_distill_list_of_the_whole_vocabulary():
    x = make((4,), 64, torch.float32)
    index = torch.stack([torch.randperm(64) for _ in range(4)])
    lp = torch.log_softmax(torch.randn(4, 64), -1) - 1e-4  # mass short of 1: no class to hold it
    check_distill(x, index, lp, None, 1.0, True)


def test_distill_impossible_and_invalid():
    V = 500
    x = make((5,), V, torch.float32)
    index, lp = lists((5,), V, 6, empty=False)
    x[0, index[0, 2]] = -math.inf   # the student forbids what the teacher lists
    x[1] = -math.inf                # no student at all
    index[2, 3] = V                 # no such token
    lp[3, 1] = math.nan
    loss, d = kernels.distill_topk_loss_grad(x, index.cuda(), lp.cuda())
    assert loss[:2].tolist() == [math.inf, math.inf]
    assert torch.isnan(loss[2:4]).all() and torch.isfinite(loss[4])
    assert torch.isfinite(d[0]).all() and (d[1] == 0).all() and torch.isfinite(d[4]).all()
    assert torch.isnan(d[2]).all() and torch.isnan(d[3]).all()
    # weight 0: nothing of the row counts, whatever it holds
    w = torch.tensor([0.0, 0.0, 0.0, 0.0, 1.0], device="cuda")
    x[0] = math.nan
    z = x.clone().requires_grad_(True)
    loss = kernels.distill_topk_loss(z, index.cuda(), lp.cuda(), weight=w, tail=True)
    (d,) = torch.autograd.grad(loss.sum(), z)
    loss2, d2 = kernels.distill_topk_loss_grad(x, index.cuda(), lp.cuda(), weight=w, tail=True)
    for l_, g_ in ((loss, d), (loss2, d2)):
        assert (l_[:4] == 0).all() and (g_[:4] == 0).all() and torch.isfinite(l_[4]) and g_[4].abs().sum() > 0


def test_distill_types_and_strides():
    V = 1111
    base = make((3, 7), V, torch.bfloat16)
    index, lp = lists((3, 7), V, 10)
    x = base[:, :-1]
    check_distill(x, index[:, 1:], lp[:, 1:], torch.rand(3, 6), 1.0, True)
    loss = kernels.distill_topk_loss(base, index.int().cuda(), lp.bfloat16().cuda(), weight=torch.ones(3, 7).double().cuda())
    ref = L.distill(base.float().cpu(), index, lp.bfloat16().float())
    close(loss, ref, 2 * rel(V) + 2e-5)
    slots = index.cuda().transpose(0, 1).contiguous().transpose(0, 1)[..., ::2]
    loss = kernels.distill_topk_loss(base, slots, lp.cuda()[..., ::2])
    close(loss, L.distill(base.float().cpu(), index[..., ::2], lp[..., ::2]), 2 * rel(V) + 2e-5)
    check_distill(make((2, 2, 3, 2), 70, torch.float32), *lists((2, 2, 3, 2), 70, 4), None, 1.0, False)


def test_the_teachers_list_feeds_the_students_loss():
    """A student equal to its teacher: no loss, no gradient (up to the two operators' rounding)."""
    x = make((40,), 3000, torch.float32)
    for T in (1.0, 2.0):
        top = kernels.token_logprobs(x, top_k=64, temperature=T)
        loss, d = kernels.distill_topk_loss_grad(x, top.top_index, top.top_logprob, temperature=T, tail=True)
        assert loss.abs().max().item() < 4 * rel(3000) and d.abs().max().item() < 4 * rel(3000)


# ---------------------------------------------------------------- bindings, streams, graphs
def _calls(ops, x, tok, index, lp, w):
    f = ops.token_logprobs(x, tok, 7, 0.9, -100, True)
    g = torch.linspace(-1, 1, tok.numel(), device="cuda").view(tok.shape)
    b = ops.token_logprobs_bwd(x, tok, f[5], f[1], f[4], g, g * 0.1, None, None, 0.9, -100)
    loss, d, st = ops.distill_topk(x, index, lp, w, 1.1, True, True, True)
    return [*f, b, loss, d, st, ops.distill_topk_bwd(x, index, lp, w, st, g, 1.1, True)]


@pytest.mark.parametrize("shape,V", [((3, 50), 256), ((2, 30), 9001), ((2,), 131072)])
def test_both_bindings_and_a_second_call_give_the_same_bits(shape, V):
    x = make(shape, V, torch.bfloat16)
    tok = tokens(shape, V).cuda()
    index, lp = (t.cuda() for t in lists(shape, V, 12))
    w = torch.rand(shape, device="cuda")
    a = _calls(sm100_ext.load_ext(), x, tok, index, lp, w)
    for other in (_calls(sm100_logits, x, tok, index, lp, w), _calls(sm100_ext.load_ext(), x, tok, index, lp, w)):
        for p, q in zip(a, other):
            assert torch.equal(p, q)


def test_other_streams_and_graph_capture():
    V, shape = 5003, (2, 33)
    x = make(shape, V, torch.bfloat16)
    tok = tokens(shape, V).cuda()
    index, lp = (t.cuda() for t in lists(shape, V, 12))
    w = torch.rand(shape, device="cuda")
    ops = sm100_ext.load_ext()
    want = _calls(ops, x, tok, index, lp, w)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = _calls(ops, x, tok, index, lp, w)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = _calls(ops, x, tok, index, lp, w)
    keep = x.clone()
    x.zero_()
    graph.replay()
    x.copy_(keep)
    graph.replay()
    torch.cuda.synchronize()
    for p, q, r in zip(want, got, held):
        assert torch.equal(p, q) and torch.equal(p, r)


def test_offsets_past_32_bits():
    """2^31 elements and more before the last rows, and between the outer rows."""
    V, rows = 65537, 33000
    x = torch.zeros(rows, V, dtype=torch.bfloat16, device="cuda")
    assert x.numel() > 1 << 31
    x[-3:] = make((3,), V, torch.bfloat16)
    tok = torch.zeros(rows, dtype=torch.long, device="cuda")
    tok[-3:] = tokens((3,), V).cuda()
    z = x.requires_grad_(True)
    r = kernels.token_logprobs(z, tok)
    (d,) = torch.autograd.grad(r.logprob.sum(), z)
    xc = x.detach()[-3:].float().cpu()
    ref = L.token_logprobs(xc, tok[-3:].cpu())
    close(r.logprob[-3:].detach(), ref["logprob"], 2 * rel(V) + 1e-5)
    close(r.logprob[:-3].detach(), torch.full((rows - 3,), -math.log(V), dtype=torch.float64), 2 * rel(V))
    check_grad(d[-3:], L.token_logprobs_grad(xc, tok[-3:].cpu(), g_logprob=torch.ones(3)), torch.ones(3), V, torch.bfloat16)
    del d, r, z
    x = x.detach()
    index, lp = lists((3,), V, 9)
    full_i = torch.zeros(rows, 9, dtype=torch.long, device="cuda") - 1
    full_i[-3:] = index.cuda()
    full_l = torch.zeros(rows, 9, device="cuda")
    full_l[-3:] = lp.cuda()
    loss, d = kernels.distill_topk_loss_grad(x, full_i, full_l)
    close(loss[-3:], L.distill(xc, index, lp), 2 * rel(V) + 2e-5)
    check_grad(d[-3:], L.distill_grad(xc, index, lp), torch.full((3,), 2.0), V, torch.bfloat16)
    assert (loss[:-3] == 0).all()
    del d
    far = x.as_strided((2, 3, V), ((rows - 3) * V, V, 1))  # outer stride past 2^31
    check_forward(far, tokens((2, 3), V), 5, 1.0)


def test_refusals():
    x = torch.zeros(2, 3, 16, device="cuda")
    tok = torch.zeros(2, 3, dtype=torch.long, device="cuda")
    idx, lp = torch.zeros(2, 3, 4, dtype=torch.long, device="cuda"), torch.zeros(2, 3, 4, device="cuda")
    for ops in (sm100_ext.load_ext(), sm100_logits):
        for call, error, words in (
                (lambda: ops.token_logprobs(x.half()), TypeError, "float32 or bfloat16"),
                (lambda: ops.token_logprobs(x, tok.float()), TypeError, "int64 or int32"),
                (lambda: ops.token_logprobs(x, tok[:1]), ValueError, "does not go with"),
                (lambda: ops.token_logprobs(x, tok.cpu()), RuntimeError, "device"),
                (lambda: ops.token_logprobs(x, tok, 17), ValueError, "top_k"),
                (lambda: ops.token_logprobs(x, tok, -1), ValueError, "top_k"),
                (lambda: ops.token_logprobs(torch.zeros(2, 200, device="cuda"), None, 129), ValueError, "top_k"),
                (lambda: ops.token_logprobs(x, tok, 0, 0.0), ValueError, "temperature"),
                (lambda: ops.token_logprobs(x, tok, 0, math.nan), ValueError, "temperature"),
                (lambda: ops.token_logprobs(x[..., :0]), ValueError, "empty"),
                (lambda: ops.token_logprobs(torch.zeros((), device="cuda")), ValueError, "must be"),
                (lambda: ops.distill_topk(x, idx, lp[..., :3]), ValueError, "does not go with"),
                (lambda: ops.distill_topk(x, idx.float(), lp), TypeError, "int64 or int32"),
                (lambda: ops.distill_topk(x, idx, lp.long()), TypeError, "floating"),
                (lambda: ops.distill_topk(x, idx[..., :0], lp[..., :0]), ValueError, "slots"),
                (lambda: ops.distill_topk(x, idx, lp, torch.ones(5, device="cuda")), ValueError, "weight"),
                (lambda: ops.distill_topk(x, idx, lp, None, -1.0), ValueError, "temperature"),
        ):
            with pytest.raises(error, match=words):
                call()
    torch.cuda.synchronize()


@pytest.mark.parametrize("binding", ["ext", "ctypes"])
def test_double_backward_is_refused(binding, monkeypatch):
    monkeypatch.setenv("BDH_SM100_EXT", "1" if binding == "ext" else "0")
    x = torch.randn(2, 16, device="cuda", requires_grad=True)
    r = kernels.token_logprobs(x, torch.zeros(2, dtype=torch.long, device="cuda"))
    (d,) = torch.autograd.grad(r.logprob.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        torch.autograd.grad((d * d).sum() + x.sum(), x)
    idx = torch.zeros(2, 3, dtype=torch.long, device="cuda")
    loss = kernels.distill_topk_loss(x, idx, torch.zeros(2, 3, device="cuda"))
    (d,) = torch.autograd.grad(loss.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        torch.autograd.grad((d * d).sum() + x.sum(), x)


def test_both_bindings_autograd_gives_the_same_bits(monkeypatch):
    V, shape = 700, (2, 5)
    x = make(shape, V, torch.bfloat16)
    tok = tokens(shape, V).cuda()
    index, lp = (t.cuda() for t in lists(shape, V, 9))
    got = {}
    for binding in ("1", "0"):
        monkeypatch.setenv("BDH_SM100_EXT", binding)
        z = x.clone().requires_grad_(True)
        r = kernels.token_logprobs(z, tok, top_k=4, temperature=0.9)
        loss = kernels.distill_topk_loss(z, index, lp, temperature=1.2, tail=True)
        (r.logprob.sum() + (r.entropy * 0.3).sum() + r.top_logprob.sum() + loss.sum()).backward()
        assert not r.top_index.requires_grad and r.lse.requires_grad
        got[binding] = [r.logprob, r.entropy, r.lse, r.top_logprob, r.top_index, loss, z.grad]
    for p, q in zip(got["1"], got["0"]):
        assert torch.equal(p, q)


def test_logits_changed_after_the_forward_are_noticed():
    x = torch.randn(3, 50, device="cuda", requires_grad=True)
    y = x * 1.0
    r = kernels.token_logprobs(y, torch.zeros(3, dtype=torch.long, device="cuda"))
    y.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        r.logprob.sum().backward()


@pytest.mark.parametrize("binding", ["ext", "ctypes"])
def test_lists_and_tokens_made_in_inference_mode(binding, monkeypatch):
    """A teacher's pass is often made there; its tensors cannot be saved as variables."""
    monkeypatch.setenv("BDH_SM100_EXT", "1" if binding == "ext" else "0")
    x = make((4,), 500, torch.float32)
    with torch.inference_mode():
        tok = tokens((4,), 500).cuda()
        top = kernels.token_logprobs(x, tok, top_k=6)
        w = torch.rand(4, device="cuda")
    z = (x + 0.1 * torch.randn_like(x)).requires_grad_(True)
    loss = kernels.distill_topk_loss(z, top.top_index, top.top_logprob, weight=w, tail=True)
    r = kernels.token_logprobs(z, tok)
    (d,) = torch.autograd.grad(loss.sum() + r.logprob.sum(), z)
    zc = z.detach().cpu()
    ref = L.distill_grad(zc, top.top_index.cpu(), top.top_logprob.cpu(), w.cpu(), 1.0, True)
    ref = ref + L.token_logprobs_grad(zc, tok.cpu(), g_logprob=torch.ones(4))
    check_grad(d, ref, 2 * w.cpu() + 1, 500, torch.float32)


# ------------------------------------------------------ many rows, which warps take one each
def many_rows():
    return 8 * torch.cuda.get_device_properties(0).multi_processor_count + 5


@pytest.mark.parametrize("dtype,V", [("f32", 1025), ("f32", 3001), ("f32", 8190), ("bf16", 1030), ("bf16", 4096),
                                     ("bf16", 9001), ("bf16", 16384), ("bf16", 16390)])
def test_forward_of_many_rows(V, dtype):
    n = many_rows()
    x = make((n,), V, DT[dtype], seed=V, offset=V % 4)
    rows = torch.stack(list(patterns(V, DT[dtype]).values())).to(DT[dtype])
    x[100:100 + rows.size(0)] = rows.cuda()
    for k in (0, 1, 9, 32, 40):
        check_forward(x, tokens((n,), V), k, 0.9)


@pytest.mark.parametrize("dtype,V", [("f32", 200), ("f32", 512), ("bf16", 999), ("f32", 1025), ("f32", 2048),
                                     ("f32", 2049), ("bf16", 1031), ("bf16", 4096), ("bf16", 4099)])
def test_logprob_gradient_of_many_rows(V, dtype):
    n, T, k = many_rows(), 1.3, 7
    x = make((n,), V, DT[dtype], seed=V, offset=V % 5).requires_grad_(True)
    tok = tokens((n,), V)
    tok[::50] = -100
    g = torch.Generator().manual_seed(4)
    up = {name: torch.randn(n, generator=g) for name in ("logprob", "entropy")}
    up_top = torch.randn(n, k, generator=g)
    xc = x.detach().float().cpu()
    for with_list in (False, True):
        r = kernels.token_logprobs(x, tok.cuda(), top_k=k if with_list else 0, temperature=T)
        outs, ups = [r.logprob, r.entropy], [up["logprob"], up["entropy"]]
        more = {}
        if with_list:
            outs.append(r.top_logprob)
            ups.append(up_top)
            more = {"g_top": up_top, "top_index": L.order(xc, k)}
        (d,) = torch.autograd.grad(outs, x, [u.cuda() for u in ups])
        ref = L.token_logprobs_grad(xc, tok, T, g_logprob=up["logprob"], g_entropy=up["entropy"], **more)
        size = sum(u.abs() if u.dim() == 1 else u.abs().sum(-1) for u in ups) / T
        check_grad(d, ref, size, V, x.dtype)


@pytest.mark.parametrize("dtype,V,k", [("f32", 200, 16), ("bf16", 512, 20), ("f32", 1025, 24), ("bf16", 1031, 100),
                                       ("bf16", 4096, 64), ("f32", 6144, 30), ("f32", 6149, 30), ("bf16", 9001, 24)])
def test_distill_of_many_rows(V, k, dtype):
    n = many_rows()
    x = make((n,), V, DT[dtype], seed=V, offset=V % 4)
    index, lp = lists((n,), V, k)
    index[7::20, 1] = index[7::20, 0]  # a token twice
    w = torch.rand(n, generator=torch.Generator().manual_seed(2)) + 0.1
    w[::30] = 0.0
    check_distill(x, index, lp, None, 2.0, False)
    check_distill(x, index, lp, w, 0.8, True)


@pytest.mark.parametrize("dtype,V", [("f32", 8200), ("f32", 12001), ("f32", 28672), ("bf16", 16400), ("bf16", 40001),
                                     ("bf16", 57344)])
def test_rows_of_a_cta_each(V, dtype):
    """Too many rows to be split over clusters, too long for a warp."""
    n = 2 * torch.cuda.get_device_properties(0).multi_processor_count + 3
    x = make((n,), V, DT[dtype], seed=V, offset=V % 4)
    rows = torch.stack(list(patterns(V, DT[dtype]).values())).to(DT[dtype])
    x[50:50 + rows.size(0)] = rows.cuda()
    for k in (0, 1, 12, 32, 33, 128):
        check_forward(x, tokens((n,), V), k, 1.1)
    x = make((n,), V, DT[dtype], seed=V + 1, offset=V % 3)
    index, lp = lists((n,), V, 40)
    index[7::20, 1] = index[7::20, 0]  # a token twice
    w = torch.rand(n, generator=torch.Generator().manual_seed(2)) + 0.1
    w[::30] = 0.0
    check_distill(x, index, lp, None, 2.0, False)
    check_distill(x, index, lp, w, 0.8, True)


@pytest.mark.parametrize("dtype,V", [("bf16", 1025), ("f32", 1040), ("bf16", 1600), ("f32", 2500), ("bf16", 6000)])
def test_long_lists_of_middling_rows(V, dtype):
    """Lists that hold a good part of what their search can tell apart."""
    for n in (3, many_rows()):
        x = make((n,), V, DT[dtype], seed=V, offset=V % 3)
        if n > 100:
            rows = torch.stack(list(patterns(V, DT[dtype]).values())).to(DT[dtype])
            x[50:50 + rows.size(0)] = rows.cuda()
        for k in (33, 64, 65, 100, 128):
            check_forward(x, None, k, 1.0)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [17, 90, 200, 256, 257, 300, 511, 512])
def test_lists_of_many_short_rows(V, dtype):
    n = 32 * torch.cuda.get_device_properties(0).multi_processor_count + 3
    x = make((n,), V, DT[dtype], seed=V, offset=V % 4)
    rows = torch.stack(list(patterns(V, DT[dtype]).values())).to(DT[dtype])
    x[1001:1001 + rows.size(0)] = rows.cuda()
    x[2000:2100] = (x[2000:2100] * 2).round() / 2  # few values
    x[2200] = -math.inf
    x[2201, V // 2] = -math.inf
    for k in (1, min(5, V // 16), V // 16, min(16, V // 16)):
        check_forward(x, tokens((n,), V), k, 0.7)
    x = x[:, : V - 1]  # rows at every alignment
    check_forward(x, None, max(1, min(16, V // 16 - 1)), 1.0)
