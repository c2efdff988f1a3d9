"""The operators on a language model's logits, as cases to measure: what each one is given, its plain form in
elementary torch operations (32 bits, rounded once at the end) and the calls of this package that compute the same.

Two operators, five calls:

* ``logprobs``        ``kernels.token_logprobs``: for every row of logits the log probability of a given token, the
                      log of the normaliser, the entropy, and the ``k`` most probable tokens with their log
                      probabilities (ties to the lowest index);
* ``logprobs_train``  the same through autograd: the log probabilities and entropies of a policy step and the
                      gradient of their weighted sum with respect to the logits;
* ``distill_grad``    ``kernels.distill_topk_loss_grad``: a student's loss against the log probabilities that a
                      teacher kept for its top tokens, and its gradient, in one call;
* ``distill_train``   ``kernels.distill_topk_loss`` and its gradient through autograd;
* ``distill_loss``    ``kernels.distill_topk_loss`` alone, as an evaluation calls it.

A case: ``call`` (above), ``outer`` x ``inner`` rows of ``vocab`` logits in ``dtype``, ``k`` entries of the top list
(0: none), ``temperature``, ``shifted`` (the logits are the view ``[:, :-1]`` of one position more, the tokens
``[:, 1:]``), ``masked`` (part of the vocabulary at minus infinity, tokens or list slots left out), ``tail`` (the
probability outside the teacher's list is one more class).
"""

import math
import os
import sys

import torch

own = False

_PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "bdh-gpu-fast_b200")
_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
_IGNORED = -100


def _case(name, call, outer, inner, vocab, dtype, k=0, temperature=1.0, shifted=False, masked=False, tail=False):
    return {"name": name, "call": call, "outer": outer, "inner": inner, "vocab": vocab, "dtype": dtype, "k": k,
            "temperature": temperature, "shifted": shifted, "masked": masked, "tail": tail}


def listed():
    return [
        # one decode step of the byte model at its benchmark's batch: the alternatives that a caller is shown
        _case("bytes_step", "logprobs", 64, 1, 256, "f32", k=5, temperature=0.8),
        # a prompt's bytes scored against the model's own logits, position by position (32 sequences of 512)
        _case("bytes_prompt", "logprobs", 32, 511, 256, "bf16", shifted=True),
        # one decode step of one sequence over a large vocabulary: one row to split over the GPU
        _case("one_row", "logprobs", 1, 1, 131072, "f32", k=20),
        # constrained scoring over a vocabulary of odd size: rows start at any element, most tokens allowed
        _case("odd_vocab", "logprobs", 3, 701, 50021, "f32", k=8, temperature=0.7, shifted=True, masked=True),
        # a teacher's pass over training text: the lists that the distillation cases below are given
        _case("teacher_top", "logprobs", 4, 512, 65536, "bf16", k=64),
        # rollouts scored again: log probability and entropy alone, the largest read
        _case("rollouts", "logprobs", 4, 1024, 131072, "bf16"),
        # policy steps: log probabilities with an entropy bonus, and the gradient; bytes, then a large vocabulary
        _case("bytes_policy", "logprobs_train", 32, 512, 256, "f32"),
        _case("policy", "logprobs_train", 2, 512, 131072, "bf16", masked=True),
        # distillation steps: bytes; a large vocabulary with the tail as a class; an odd one through autograd
        _case("bytes_distill", "distill_grad", 32, 512, 256, "bf16", k=16, temperature=2.0),
        _case("distill_tail", "distill_grad", 4, 512, 131072, "bf16", k=64, tail=True),
        _case("odd_distill", "distill_train", 2, 515, 50021, "f32", k=50, temperature=1.5, masked=True),
        # a held-out set's loss, no gradient
        _case("distill_eval", "distill_loss", 3, 200, 100003, "bf16", k=100, masked=True, tail=True),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


_MOST_BYTES = 1 << 30  # of logits read and gradients written: the largest listed case


def draw(rng):
    call = rng.choice(["logprobs", "logprobs", "logprobs_train", "distill_grad", "distill_train", "distill_loss"])
    dtype = rng.choice(["f32", "bf16"])
    vocab = 256 if rng.random() < 0.15 else _log_uniform(rng, 48, 200000)
    row_bytes = vocab * (4 if dtype == "f32" else 2) * (1 if call in ("logprobs", "distill_loss") else 2)
    rows = _log_uniform(rng, 1, max(1, min(20000, _MOST_BYTES // row_bytes)))
    outer = rng.randint(1, min(rows, 8))
    most_k = min(128, vocab // 2)  # a list leaves most of a vocabulary out
    k = _log_uniform(rng, 1, most_k) if call.startswith("distill") or (call == "logprobs" and rng.random() < 0.6) else 0
    c = _case("", call, outer, max(1, rows // outer), vocab, dtype, k=k,
              temperature=rng.choice([1.0, 1.0, 0.7, 1.5, 2.0]), shifted=rng.random() < 0.3,
              masked=rng.random() < 0.4, tail=call.startswith("distill") and rng.random() < 0.5)
    del c["name"]
    return c


def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    outer, inner, vocab, k = case["outer"], case["inner"], case["vocab"], case["k"]
    more = 1 if case["shifted"] else 0
    shape = (outer, inner + more)
    logits = torch.empty(*shape, vocab, device=dev, dtype=_DTYPES[case["dtype"]]).normal_(0.0, 2.0, generator=g)
    tokens = torch.randint(vocab, shape, device=dev, generator=g)
    # the model favours most of the tokens that were taken, some of them strongly
    lift = torch.rand(*shape, 1, device=dev, generator=g) * 12.0 - 2.0
    target = (tokens.roll(-1, 1) if more else tokens).unsqueeze(-1)  # the token that each position's logits are for
    logits.scatter_add_(-1, target, lift.to(logits.dtype))
    state = {"case": dict(case), "keep": logits}
    if case["masked"]:  # a quarter of the vocabulary is never allowed; the tokens taken are
        banned = torch.rand(vocab, device=dev, generator=g) < 0.25
        taken = logits.gather(-1, target)
        logits.masked_fill_(banned, float("-inf"))
        logits.scatter_(-1, target, taken)
        out = torch.rand(shape, device=dev, generator=g) < 0.1  # prompt or padding positions
    if not case["call"].startswith("distill"):
        if case["masked"]:
            tokens = tokens.masked_fill(out, _IGNORED)
        state["logits"] = logits[:, :-1] if more else logits
        state["tokens"] = tokens[:, 1:] if more else tokens
        if case["call"] == "logprobs_train":
            state["advantage"] = torch.randn(outer, inner, device=dev, generator=g)
            state["bonus"] = torch.full((outer, inner), 0.01, device=dev)
        return state
    rows = (outer, inner)
    logits = logits[:, :-1] if more else logits
    # the teacher's list: distinct tokens, the most probable first, some mass outside it
    step = 1 + torch.randint(max(1, vocab // max(1, k)), rows, device=dev, generator=g)
    at = torch.randint(vocab, rows, device=dev, generator=g)
    index = (at.unsqueeze(-1) + step.unsqueeze(-1) * torch.arange(k, device=dev)) % vocab
    score = (torch.randn(*rows, k, device=dev, generator=g) * 2.0).sort(dim=-1, descending=True).values
    outside = 0.01 + 0.2 * torch.rand(*rows, 1, device=dev, generator=g)
    teacher = score - score.exp().sum(-1, keepdim=True).log() + torch.log1p(-outside)
    # the student is on its way there, and allows what the teacher lists
    there = (score + torch.randn(*rows, k, device=dev, generator=g)).to(logits.dtype)
    logits.scatter_(-1, index, there)
    weight = torch.full(rows, 1.0, device=dev)
    if case["masked"]:
        weight = weight.masked_fill(out[:, :inner], 0.0)
        empty = torch.rand(*rows, k, device=dev, generator=g) < 0.1
        empty[..., 0] = False
        index = index.masked_fill(empty, -1)
    state.update(logits=logits, index=index, teacher=teacher, weight=weight / weight.sum().clamp_min(1.0))
    return state


def _ordered_keys(z):
    """Whole numbers in the order of the values of ``z``, an equal value's lowest index first."""
    bits = (z.float() + 0.0).view(torch.int32)
    bits = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).to(torch.int64)
    return bits * (1 << 32) + torch.arange(z.size(-1) - 1, -1, -1, device=z.device)


def _plain_logprobs(logits, tokens, k, temperature):
    z = logits.float() / temperature
    top = z.max(dim=-1, keepdim=True).values
    e = torch.exp(z - top)
    total = e.sum(dim=-1, keepdim=True)
    lse = top + torch.log(total)
    given = tokens != _IGNORED
    picked = z.gather(-1, tokens.clamp_min(0).unsqueeze(-1)) - lse
    out = {"logprob": torch.where(given, picked.squeeze(-1), 0.0), "lse": lse.squeeze(-1),
           "entropy": (torch.log(total) - (e * torch.where(e > 0, z - top, 0.0)).sum(-1, keepdim=True) / total).squeeze(-1)}
    if k:
        keys = torch.topk(_ordered_keys(logits), k, dim=-1).values
        index = logits.size(-1) - 1 - (keys & 0xFFFFFFFF)
        out["top_logprob"] = z.gather(-1, index) - lse
        out["top_index"] = index
    return out


def _plain_logprobs_grad(logits, tokens, temperature, out, g_logprob, g_entropy):
    logp = logits.float() / temperature - out["lse"].unsqueeze(-1)
    p = torch.exp(logp)
    given = tokens != _IGNORED
    g = torch.where(given, g_logprob, 0.0).unsqueeze(-1)
    d = -p * g - g_entropy.unsqueeze(-1) * p * (torch.where(p > 0, logp, 0.0) + out["entropy"].unsqueeze(-1))
    d.scatter_add_(-1, tokens.clamp_min(0).unsqueeze(-1), g)
    return (d / temperature).to(logits.dtype)


def _plain_distill(logits, index, teacher, weight, temperature, tail, grad):
    vocab = logits.size(-1)
    z = logits.float() / temperature
    top = z.max(dim=-1, keepdim=True).values
    lse = top + torch.log(torch.exp(z - top).sum(dim=-1, keepdim=True))
    valid = index >= 0
    at = torch.where(valid, index, vocab)  # an empty slot's place is one past the vocabulary
    t = teacher.masked_fill(~valid, float("-inf"))
    if not tail:
        t = t - t.max(dim=-1, keepdim=True).values
        t = t - torch.log(torch.exp(t).sum(dim=-1, keepdim=True))
    q = torch.exp(t)
    logp = z.gather(-1, index.clamp_min(0)) - lse
    loss = torch.where(q > 0, q * (torch.where(q > 0, t, 0.0) - logp), 0.0).sum(-1)
    total, ratio = q.sum(-1, keepdim=True), None
    p = torch.exp(z - lse)
    if tail:
        listed_ = torch.zeros(*z.shape[:-1], vocab + 1, dtype=torch.bool, device=z.device)
        listed_.scatter_(-1, at, True)
        p_out = p.masked_fill(listed_[..., :vocab], 0.0)
        r = (1.0 - total).clamp_min(0.0)
        s = p_out.sum(-1, keepdim=True)
        loss = loss + torch.where(r > 0, r * (torch.log(r) - torch.log(s)), 0.0).squeeze(-1)
        total, ratio = total + r, torch.where(r > 0, r / s, 0.0)
    loss = torch.where(weight != 0, loss * weight, 0.0)
    if not grad:
        return {"loss": loss}
    d = torch.zeros(*z.shape[:-1], vocab + 1, device=z.device)
    d[..., :vocab] = p * total
    if tail:
        d[..., :vocab] -= p_out * ratio
    d.scatter_add_(-1, at, -q)
    d = d[..., :vocab] * (weight / temperature).unsqueeze(-1)
    return {"loss": loss, "grad": torch.where(weight.unsqueeze(-1) != 0, d, 0.0).to(logits.dtype)}


def _run_own(state):
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    import kernels

    case, x = state["case"], state["logits"]
    call, k, temperature = case["call"], case["k"], case["temperature"]
    if call == "logprobs":
        r = kernels.token_logprobs(x, state["tokens"], top_k=k, temperature=temperature)
        out = {"logprob": r.logprob, "lse": r.lse, "entropy": r.entropy}
        if k:
            out.update(top_logprob=r.top_logprob, top_index=r.top_index)
        return out
    if call == "logprobs_train":
        x = x.detach().requires_grad_(True)
        r = kernels.token_logprobs(x, state["tokens"], temperature=temperature)
        (d,) = torch.autograd.grad((r.logprob, r.entropy), x, (state["advantage"], state["bonus"]))
        return {"logprob": r.logprob.detach(), "lse": r.lse.detach(), "entropy": r.entropy.detach(), "grad": d}
    args = (state["index"], state["teacher"])
    opts = {"weight": state["weight"], "temperature": temperature, "tail": case["tail"]}
    if call == "distill_grad":
        loss, d = kernels.distill_topk_loss_grad(x, *args, **opts)
        return {"loss": loss, "grad": d}
    if call == "distill_loss":
        return {"loss": kernels.distill_topk_loss(x, *args, **opts)}
    x = x.detach().requires_grad_(True)
    loss = kernels.distill_topk_loss(x, *args, **opts)
    (d,) = torch.autograd.grad(loss.sum(), x)
    return {"loss": loss.detach(), "grad": d}


def run(state):
    if own:
        return _run_own(state)
    case, x = state["case"], state["logits"]
    call, temperature = case["call"], case["temperature"]
    if call == "logprobs":
        return _plain_logprobs(x, state["tokens"], case["k"], temperature)
    if call == "logprobs_train":
        out = _plain_logprobs(x, state["tokens"], 0, temperature)
        out["grad"] = _plain_logprobs_grad(x, state["tokens"], temperature, out, state["advantage"], state["bonus"])
        return out
    return _plain_distill(x, state["index"], state["teacher"], state["weight"], temperature, case["tail"],
                          grad=call != "distill_loss")


def work(case):
    rows, vocab, k = case["outer"] * case["inner"], case["vocab"], case["k"]
    size = 4 if case["dtype"] == "f32" else 2
    elements = rows * vocab
    call = case["call"]
    if call == "logprobs":  # logits and tokens in; three figures a row and the list out
        return {"bytes": elements * size + rows * (8 + 12 + 12 * k), "flops": 6 * elements}
    if call == "logprobs_train":
        return {"bytes": 2 * elements * size + rows * (8 + 8 + 12), "flops": 12 * elements}
    listed_ = rows * (12 * k + 8)
    if call == "distill_loss":
        return {"bytes": elements * size + listed_, "flops": 4 * elements}
    return {"bytes": 2 * elements * size + listed_, "flops": 9 * elements}


def _exact_distill(x, state, temperature, tail, grad):
    """Row sums written as the cross entropy of two distributions over the listed tokens (and the rest)."""
    x = x.double().div_(temperature)
    index, weight = state["index"], state["weight"].double()
    on = index >= 0
    t = torch.where(on, state["teacher"].double(), -math.inf)
    if not tail:
        t = torch.log_softmax(t, dim=-1)
    q = t.exp()
    logp = torch.log_softmax(x, dim=-1)
    del x
    mine = torch.where(on, logp.gather(-1, index.clamp_min(0)), 0.0)
    loss = (torch.special.xlogy(q, q) - q * mine).sum(-1)
    mass = q.sum(-1)
    rest = None
    if tail:
        r = (1.0 - mass).clamp_min(0.0)
        outside = torch.ones(logp.shape[:-1] + (logp.size(-1) + 1,), dtype=torch.bool, device=logp.device)
        outside.scatter_(-1, torch.where(on, index, logp.size(-1)), False)
        rest = torch.where(outside[..., :-1], logp.exp(), 0.0)
        s = rest.sum(-1)
        loss = loss + torch.special.xlogy(r, r / s)
        mass, rest = mass + r, rest.mul_((r / s).unsqueeze(-1))
    loss = torch.where(weight == 0, 0.0, weight * loss)
    if not grad:
        return {"loss": loss}
    d = logp.exp_().mul_(mass.unsqueeze(-1))
    if rest is not None:
        d -= rest
    d.scatter_add_(-1, index.clamp_min(0), torch.where(on, -q, 0.0))
    return {"loss": loss, "grad": d.mul_((weight / temperature).unsqueeze(-1))}


def exact(case, seed):
    state = prepare(case, seed)
    state.pop("keep")
    x, call, temperature = state.pop("logits"), case["call"], case["temperature"]
    if call.startswith("distill"):
        return _exact_distill(x, state, temperature, case["tail"], call != "distill_loss")
    tokens = state["tokens"]
    out = {}
    if case["k"]:
        order = torch.sort(x.double(), dim=-1, descending=True, stable=True).indices[..., :case["k"]].clone()
    z = x.double().div_(temperature)
    lse = torch.logsumexp(z, dim=-1)
    logp = z.sub_(lse.unsqueeze(-1))
    on = tokens != _IGNORED
    out = {"logprob": torch.where(on, logp.gather(-1, tokens.clamp_min(0).unsqueeze(-1)).squeeze(-1), 0.0),
           "lse": lse, "entropy": torch.special.entr(logp.exp()).sum(-1)}
    if case["k"]:
        out.update(top_logprob=logp.gather(-1, order), top_index=order)
    if call == "logprobs_train":
        g, b = torch.where(on, state["advantage"].double(), 0.0), state["bonus"].double()
        p = logp.exp()
        d = p.mul(-(g + b * out["entropy"]).unsqueeze(-1))
        d += torch.special.entr(p).mul_(b.unsqueeze(-1))  # -p log p, nothing where p is 0
        d.scatter_add_(-1, tokens.clamp_min(0).unsqueeze(-1), g.unsqueeze(-1))
        out["grad"] = d.div_(temperature)
    return out
