"""Class scoring and distillation in float64 torch on the CPU: the definitions of include/mica_hip.h, restated for the tests.
The class axis is the last one; rows are everything in front of it."""
import torch

NEG = float("-inf")


def order(z, k):
    """Indices of the k largest along the last axis: NaN counts as -inf, ties go to the lowest index."""
    z = torch.where(torch.isnan(z), torch.full_like(z, NEG), z.double())
    return torch.sort(z, dim=-1, descending=True, stable=True).indices[..., :k]


def log_softmax(y):
    """log softmax with rows of -inf only -> -inf (and NaN where a NaN or +inf is)"""
    m = y.amax(-1, keepdim=True)
    empty = m == NEG
    ref = torch.where(empty, torch.zeros_like(m), m)
    log_s = torch.log(torch.exp(y - ref).sum(-1, keepdim=True))
    # (y - ref) - log_s: the sum of a huge maximum and log_s would lose log_s
    return torch.where(empty, torch.full_like(y, NEG), (y - ref) - log_s), (ref + log_s).squeeze(-1)


def score(z, tokens=None, top=0, temperature=1.0, ignore_index=-100):
    """-> dict(logprob, entropy, lse, top_logprob, top_index)"""
    y = z.double() / temperature
    logp, lse = log_softmax(y)
    p = torch.exp(logp)
    ent = -torch.where(p == 0, torch.zeros_like(p), p * logp).sum(-1)
    out = dict(entropy=ent, lse=lse, logp=logp)
    if tokens is not None:
        t = tokens.long()
        ok = (t >= 0) & (t < z.shape[-1])
        lp = torch.gather(logp, -1, torch.where(ok, t, torch.zeros_like(t)).unsqueeze(-1)).squeeze(-1)
        lp = torch.where(ok, lp, torch.full_like(lp, float("nan")))
        out["logprob"] = torch.where(t == ignore_index, torch.zeros_like(lp), lp)
    if top:
        idx = order(z, top)
        out["top_index"] = idx
        out["top_logprob"] = torch.gather(logp, -1, idx)
    return out


def score_grad(z, tokens, g_logprob=None, g_entropy=None, g_lse=None, temperature=1.0, ignore_index=-100):
    """The gradient by its formula (rows with a finite class; others 0)."""
    y = z.double() / temperature
    logp, lse = log_softmax(y)
    p = torch.exp(logp)
    safe = torch.where(p == 0, torch.zeros_like(p), logp)
    H = -(p * safe).sum(-1, keepdim=True)
    g = torch.zeros_like(p)
    if g_logprob is not None:
        t = tokens.long()
        used = t != ignore_index
        gl = torch.where(used, g_logprob.double(), torch.zeros_like(lse)).unsqueeze(-1)
        g = g - gl * p
        g.scatter_add_(-1, torch.where(used, t, torch.zeros_like(t)).unsqueeze(-1), gl)
    if g_lse is not None:
        g = g + g_lse.double().unsqueeze(-1) * p
    if g_entropy is not None:
        g = g - g_entropy.double().unsqueeze(-1) * p * (safe + H)
    return torch.where((lse == NEG).unsqueeze(-1), torch.zeros_like(g), g / temperature)


def _teacher(index, value, tail, classes):
    """-> (p [.., K] with 0 at unused entries, log p, target [.., C], listed [.., C], rest [..])"""
    idx = index.long()
    used = idx >= 0
    t = torch.where(used, value.double(), torch.full_like(value, NEG, dtype=torch.float64))
    if not tail:
        t = log_softmax(t)[0]
    p = torch.exp(t)
    slot = torch.where(used, idx, torch.full_like(idx, classes))
    target = torch.zeros(idx.shape[:-1] + (classes + 1,), dtype=torch.float64).scatter_add_(-1, slot, p)[..., :classes]
    listed = torch.zeros(idx.shape[:-1] + (classes + 1,), dtype=torch.bool).scatter_(-1, slot, True)[..., :classes]
    rest = (1.0 - p.sum(-1)).clamp(min=0.0) if tail else torch.zeros(idx.shape[:-1], dtype=torch.float64)
    return p, t, target, listed, rest


def distill(z, index, value, temperature=1.0, tail=False):
    """-> (loss [..], gradient of loss.sum() with respect to z [.., C], parts for error bounds)"""
    C = z.shape[-1]
    y = z.double() / temperature
    logq, lse = log_softmax(y)
    q = torch.exp(logq)
    p, logp, target, listed, rest = _teacher(index, value, tail, C)
    at = index.long().clamp(min=0)
    lq = torch.gather(logq, -1, at)
    loss = torch.where(p == 0, torch.zeros_like(p), p * (logp - lq)).sum(-1)
    free = torch.where(listed, torch.full_like(y, NEG), y)         # of y, not of logq: beside a class at 1e12 logq has lost their distances
    some = (free > NEG).any(-1)
    rest = torch.where(some, rest, torch.zeros_like(rest))
    lfree = log_softmax(free)[0]
    lqr = (free.amax(-1) - y.amax(-1)) - lfree.amax(-1) + logq.amax(-1)      # maxima apart, log sums apart: a huge maximum would swallow the sum
    loss = loss + torch.where(rest > 0, rest * (torch.log(rest.clamp(min=1e-300)) - torch.where(rest > 0, lqr, torch.zeros_like(lqr))), torch.zeros_like(rest))
    mass = (p.sum(-1) + rest).unsqueeze(-1)
    grad = mass * q - target - torch.where((rest > 0).unsqueeze(-1) & ~listed, rest.unsqueeze(-1) * torch.exp(lfree), torch.zeros_like(q))
    grad = torch.where((lse == NEG).unsqueeze(-1), torch.zeros_like(grad), grad * temperature)
    share = torch.where((rest > 0).unsqueeze(-1) & ~listed, torch.exp(lfree), torch.zeros_like(q))
    return loss * temperature ** 2, grad, dict(q=q, target=target, share=share, rest=rest, mass=mass, lq=torch.where(p == 0, torch.zeros_like(lq), lq), lse=lse)
