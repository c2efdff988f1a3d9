"""Plain 64-bit forms of the operators on logits (kernels/logits.py), written from their formulas in
torch on the CPU: test infrastructure only.

    token_logprobs(x, tokens, k, temperature, ignore)  -> dict of figures
    token_logprobs_grad(x, tokens, ..., g_*)           -> d/dx of sum g_* . figure_*
    distill(x, index, teacher, weight, temperature, tail)       -> loss per row
    distill_grad(same)                                          -> d/dx of sum of the losses
"""

import torch

NEG = float("-inf")


def _softmax(x, temperature):
    z = x.double() / temperature
    m = z.max(dim=-1, keepdim=True).values
    none = m == NEG
    e = torch.exp(z - torch.where(none, 0.0, m))
    s = e.sum(-1, keepdim=True)
    lse = torch.where(none, NEG, m + torch.log(s))
    logp = torch.where(none, NEG, (z - m) - torch.log(s))  # z - lse has no digits left beside 1e38
    return logp, lse.squeeze(-1), none.squeeze(-1)


def order(x, k):
    """Indices of the k largest, an equal value's lower index first, NaN before everything."""
    key = torch.where(torch.isnan(x), torch.tensor(float("inf"), dtype=torch.float64), x.double())
    nan_first = torch.argsort((~torch.isnan(x)).long(), dim=-1, stable=True)
    by_nan = key.gather(-1, nan_first)
    # sort by value with NaN rows' entries already in front of equal +inf
    at = torch.sort(by_nan, dim=-1, descending=True, stable=True).indices
    return nan_first.gather(-1, at)[..., :k]


def token_logprobs(x, tokens=None, k=0, temperature=1.0, ignore=-100):
    logp, lse, none = _softmax(x, temperature)
    p = torch.exp(logp)
    out = {"lse": lse,
           "entropy": torch.where(none, 0.0, -torch.where(p > 0, p * logp, p).sum(-1))}
    if torch.isnan(x).any():
        out["entropy"] = torch.where(torch.isnan(lse), lse, out["entropy"])
    if tokens is not None:
        V = x.size(-1)
        ok = (tokens >= 0) & (tokens < V)
        lp = logp.gather(-1, tokens.clamp(0, V - 1).unsqueeze(-1)).squeeze(-1)
        lp = torch.where(ok, lp, float("nan"))
        out["logprob"] = torch.where(tokens == ignore, 0.0, lp)
    if k:
        out["top_index"] = order(x, k)
        out["top_logprob"] = logp.gather(-1, out["top_index"])
    return out


def token_logprobs_grad(x, tokens=None, temperature=1.0, ignore=-100, g_logprob=None,
                        g_entropy=None, g_lse=None, g_top=None, top_index=None):
    logp, lse, none = _softmax(x, temperature)
    p = torch.exp(logp)
    d = torch.zeros_like(p)
    if g_lse is not None:
        d += p * g_lse.double().unsqueeze(-1)
    if g_entropy is not None:
        ent = -torch.where(p > 0, p * logp, p).sum(-1, keepdim=True)
        d -= g_entropy.double().unsqueeze(-1) * p * (torch.where(p > 0, logp, 0.0) + ent)
    if g_logprob is not None:
        g = torch.where(tokens == ignore, 0.0, g_logprob.double()).unsqueeze(-1)
        d -= p * g
        d.scatter_add_(-1, tokens.clamp_min(0).unsqueeze(-1), g)
    if g_top is not None:
        d -= p * g_top.double().sum(-1, keepdim=True)
        d.scatter_add_(-1, top_index, g_top.double())
    return torch.where(none.unsqueeze(-1), 0.0, d / temperature)


def _list(index, teacher, tail, V):
    on = index >= 0
    t = torch.where(on, teacher.double(), NEG)
    if not tail:
        m = t.max(-1, keepdim=True).values
        m = torch.where(m == NEG, 0.0, m)
        s = torch.exp(t - m).sum(-1, keepdim=True)
        t = torch.where(s > 0, t - m - torch.log(s), NEG)
    q = torch.exp(t)
    mass = torch.zeros(*index.shape[:-1], V + 1, dtype=torch.float64)
    mass.scatter_add_(-1, torch.where(on, index, V), q)
    listed = torch.zeros(mass.shape, dtype=torch.bool)
    listed.scatter_(-1, torch.where(on, index, V), True)
    listed = listed[..., :V]
    r = torch.zeros(index.shape[:-1], dtype=torch.float64)
    if tail:
        r = torch.where(listed.all(-1), 0.0, (1.0 - q.sum(-1)).clamp_min(0.0))
    return t, q, mass[..., :V], listed, r


def _settled(r, rest):
    """A list's remainder that may be its fp32 rounding, where the student's tokens outside the list are
    masked: there is no other class."""
    return torch.where((r <= 2.0 ** -16) & (rest < -1000.0), 0.0, r)


def distill(x, index, teacher, weight=None, temperature=1.0, tail=False):
    V = x.size(-1)
    logp, lse, none = _softmax(x, temperature)
    t, q, mass, listed, r = _list(index, teacher, tail, V)
    lp = logp.gather(-1, index.clamp_min(0))
    loss = torch.where(q > 0, q * (torch.where(q > 0, t, 0.0) - lp), 0.0).sum(-1)
    rest = torch.logsumexp(torch.where(listed, NEG, logp), dim=-1)
    r = _settled(r, rest)
    loss = loss + torch.where(r > 0, r * (torch.log(torch.where(r > 0, r, 1.0)) - rest), 0.0)
    w = torch.ones_like(loss) if weight is None else weight.double().expand(loss.shape)
    return torch.where(w == 0, 0.0, w * loss)


def distill_grad(x, index, teacher, weight=None, temperature=1.0, tail=False):
    V = x.size(-1)
    logp, lse, none = _softmax(x, temperature)
    t, q, mass, listed, r = _list(index, teacher, tail, V)
    p = torch.exp(logp)
    rest_logp = torch.where(listed, NEG, logp)
    rest = torch.logsumexp(rest_logp, dim=-1, keepdim=True)
    r = _settled(r, rest.squeeze(-1))
    cond = torch.where(listed | (rest == NEG), 0.0, torch.exp(rest_logp - rest))
    d = p * (q.sum(-1) + r).unsqueeze(-1) - r.unsqueeze(-1) * cond - mass
    w = torch.ones_like(lse) if weight is None else weight.double().expand(lse.shape)
    d = torch.where((w == 0).unsqueeze(-1), 0.0, d * (w / temperature).unsqueeze(-1))
    return torch.where(none.unsqueeze(-1), 0.0, d)
