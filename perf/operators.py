"""Performance cases of the class-scoring operators: log probabilities of given classes (with entropy and the top alternatives) and
distillation from a teacher's top alternatives, each with its gradient.

Every case has two ways to run: the plain form (elementary torch operations in float32, whatever the inputs' type) and, where `own` is
set, the calls a user of mica_amd makes.  `exact` restates the definitions in float64."""
import functools
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZES = {"f32": 4, "bf16": 2, "f16": 2}
IGNORE = -100


def listed():
    return [
        # the residue profiles of the C-alpha candidates of one map: 20 amino acids, the assigned residue, five alternatives
        dict(name="score_candidates", op="score", layout="rows", dtype="f32", batch=1, rows=1537, classes=20, top=5, shift=0, temperature=1.0, mask=0.0),
        # one decoding step of a few sequences over a large vocabulary: the sampled token and the twenty alternatives an answer reports
        dict(name="score_decode", op="score", layout="rows", dtype="bf16", batch=1, rows=4, classes=128000, top=20, shift=0, temperature=0.7, mask=0.5),
        # prompts scored against their own next tokens: logits [B, S, C] with the last position cut off, an odd vocabulary
        dict(name="score_prompt", op="score", layout="rows", dtype="f16", batch=2, rows=1024, classes=50001, top=5, shift=1, temperature=1.0, mask=0.0),
        # one batch of sub-grids: the amino-acid head's logits without the background class, labels at a few voxels, three alternatives
        dict(name="score_voxels", op="score", layout="voxels", dtype="f32", batch=8, side=64, classes=21, top=3, temperature=1.0, ignore=0.85),
        # a policy or fine-tuning step: log probability and entropy of each position, and the gradient of both
        dict(name="train_tokens", op="train", layout="rows", dtype="bf16", batch=1, rows=4096, classes=32000, top=0, shift=0, temperature=1.0, mask=0.0),
        # the amino-acid head trained on labelled voxels, background voxels ignored
        dict(name="train_voxels", op="train", layout="voxels", dtype="f32", batch=4, side=64, classes=21, top=0, temperature=1.0, ignore=0.85),
        # a small classifier head distilled with a short list: latency
        dict(name="distill_small", op="step", layout="rows", dtype="f32", batch=1, rows=64, classes=1000, k=8, temperature=2.0, tail=False, pad=0.0),
        # held-out loss of a student, the teacher's remaining mass as one bucket
        dict(name="distill_eval", op="loss", layout="rows", dtype="bf16", batch=1, rows=513, classes=32003, k=16, temperature=1.0, tail=True, pad=0.1),
        # a smaller network distilled from the amino-acid head's top four classes per voxel
        dict(name="distill_voxels", op="grad", layout="voxels", dtype="f32", batch=4, side=64, classes=21, k=4, temperature=1.0, tail=True, pad=0.0),
        # distillation inside an autograd graph, odd rows and vocabulary
        dict(name="distill_graph", op="grad", layout="rows", dtype="f16", batch=1, rows=1999, classes=65537, k=32, temperature=1.5, tail=True, pad=0.1),
        # the training step of a large student: loss and gradient of a whole micro-batch in one call
        dict(name="distill_step", op="step", layout="rows", dtype="bf16", batch=1, rows=4096, classes=128000, k=64, temperature=1.0, tail=False, pad=0.1),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["score", "score", "train", "loss", "grad", "step"])
    layout = rng.choice(["rows", "rows", "rows", "voxels"])
    case = dict(op=op, layout=layout)
    if layout == "voxels":
        case.update(dtype=rng.choice(["f32", "f32", "bf16", "f16"]), batch=rng.randint(1, 8), side=rng.randint(4, 64), classes=21)
    else:
        classes = _log_int(rng, 2, 131072)
        rows = _log_int(rng, 1, max(1, min(8192, 500_000_000 // classes)))
        case.update(dtype=rng.choice(["f32", "bf16", "bf16", "f16"]), batch=rng.choice([1, 1, 2, 3]), classes=classes)
        case["rows"] = max(1, rows // case["batch"])
    if op in ("score", "train"):
        case.update(top=rng.choice([0, 1, 3, 5, 20, 64]) if op == "score" else 0, temperature=rng.choice([1.0, 1.0, 0.7, 1.3]))
        if layout == "voxels":
            case["ignore"] = rng.choice([0.0, 0.5, 0.85])
        else:
            case.update(shift=rng.choice([0, 1]), mask=rng.choice([0.0, 0.0, 0.5]))
        case["top"] = min(case["top"], case["classes"] - (1 if layout == "voxels" else 0))
    else:
        case.update(k=min(case["classes"], rng.choice([1, 2, 4, 8, 16, 32, 64, 100])), temperature=rng.choice([1.0, 1.0, 1.5, 2.0]), tail=rng.random() < 0.5,
                    pad=rng.choice([0.0, 0.1, 0.5]))
    return case


# ---- inputs ---------------------------------------------------------------------------------------------------------------------

def _shape(case):
    """-> (shape of the logits tensor, class axis, shape without the class axis after any cut)"""
    if case["layout"] == "voxels":
        s = case["side"]
        return (case["batch"], case["classes"], s, s, s), 1
    return (case["batch"], case["rows"] + case.get("shift", 0), case["classes"]), 2


def _inputs(case, seed):
    """All tensors of a case.  Logits: unit normals times two with one strong class per row, as a trained head gives them; with `mask`
    that share of the classes of every second row is forbidden (-inf).  Teacher lists: the top k of a noisy copy, as log probabilities;
    `pad` of the list's ends are unused entries (-1)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    shape, dim = _shape(case)
    z = torch.randn(shape, generator=g, device="cuda").mul_(2.0)
    rows_shape = shape[:dim] + shape[dim + 1:]
    strong = torch.randint(0, case["classes"], rows_shape, generator=g, device="cuda").unsqueeze(dim)
    z.scatter_add_(dim, strong, torch.rand(strong.shape, generator=g, device="cuda") * 14.0)
    out = {}
    if case["op"] in ("score", "train"):
        if case.get("mask", 0.0) > 0.0:
            drop = torch.rand((1,) * dim + (case["classes"],), generator=g, device="cuda") < case["mask"]
            drop[..., 0] = False
            even = (torch.arange(shape[1], device="cuda") % 2 == 0).view(1, -1, 1)
            z.masked_fill_(drop & even, float("-inf"))
        x = z.to(DTYPES[case["dtype"]])
        if case["layout"] == "voxels" and case["op"] == "score":
            x = x[:, 1:]                                   # the head's background class takes no part
        if case.get("shift", 0):
            x = x[:, :-1]
        rows_shape = tuple(x.shape[:dim]) + tuple(x.shape[dim + 1:])
        tok = torch.randint(0, x.shape[dim], rows_shape, generator=g, device="cuda")
        if case.get("mask", 0.0) > 0.0:                    # a sampled token is an allowed one
            tok = torch.where(drop.view(-1)[tok] & even[:, :rows_shape[1], 0], torch.zeros_like(tok), tok)
        if case.get("ignore", 0.0) > 0.0:
            tok[torch.rand(rows_shape, generator=g, device="cuda") < case["ignore"]] = IGNORE
        out.update(logits=x, tokens=tok)
        if case["op"] == "train":
            n = tok.numel()
            scale = 65536.0 if case["dtype"] == "f16" else 1.0   # float16 gradients are scaled, as mixed-precision training does
            out["g_logprob"] = -torch.rand(rows_shape, generator=g, device="cuda") * (2.0 * scale / n)
            out["g_entropy"] = torch.full(rows_shape, -0.01 * scale / n, device="cuda")
    else:
        k = case["k"]
        teach = torch.randn(shape, generator=g, device="cuda").add_(z)
        t, idx = torch.topk(teach, k, dim=dim)
        t = t / case["temperature"] - torch.logsumexp(teach / case["temperature"], dim=dim, keepdim=True)
        del teach
        idx = idx.to(torch.int32)
        if case["pad"] > 0.0:
            keep = torch.rand(rows_shape, generator=g, device="cuda").unsqueeze(dim) >= case["pad"]
            at = torch.arange(k, device="cuda").view([k if a == dim else 1 for a in range(len(shape))])
            idx = torch.where(keep | (at < (k + 1) // 2), idx, torch.full_like(idx, -1))
        out.update(logits=z.to(DTYPES[case["dtype"]]), index=idx, teacher=t.contiguous())
        n = idx.numel() // k
        scale = 65536.0 if case["dtype"] == "f16" else 1.0   # float16 gradients are scaled, as mixed-precision training does
        out["weight"] = (torch.rand(rows_shape, generator=g, device="cuda") + 0.5) * (scale / n)
    return out


@functools.lru_cache(maxsize=None)
def _engine():
    from mica_amd.engine import Engine
    return Engine(0, max_batch=1, tile_size=4)             # the handle such a program keeps; these operators use none of its workspace


def prepare(case, seed):
    state = dict(case=case, dim=_shape(case)[1], **_inputs(case, seed))
    if own:
        state["engine"] = _engine()
    return state


# ---- the framework's calls ------------------------------------------------------------------------------------------------------

def _run_own(s):
    from mica_amd import scoring
    c, eng = s["case"], s["engine"]
    if c["op"] == "score":
        r = eng.token_logprobs(s["logits"], s["tokens"], top=c["top"], dim=s["dim"], temperature=c["temperature"], ignore_index=IGNORE)
        return [r.logprob, r.entropy, r.lse] + ([r.top_logprob, r.top_index] if c["top"] else [])
    if c["op"] == "train":
        x = s["logits"].detach().requires_grad_()
        r = scoring.token_logprobs(eng, x, s["tokens"], dim=s["dim"], temperature=c["temperature"], ignore_index=IGNORE)
        grad, = torch.autograd.grad([r.logprob, r.entropy], [x], [s["g_logprob"], s["g_entropy"]])
        return [r.logprob.detach(), r.entropy.detach(), grad]
    if c["op"] == "loss":
        loss, _ = eng.distill_loss(s["logits"], s["index"], s["teacher"], dim=s["dim"], temperature=c["temperature"], tail=c["tail"])
        return [loss]
    if c["op"] == "grad":
        x = s["logits"].detach().requires_grad_()
        loss = scoring.distill_loss(eng, x, s["index"], s["teacher"], dim=s["dim"], temperature=c["temperature"], tail=c["tail"])
        grad, = torch.autograd.grad([loss], [x], [s["weight"]])
        return [loss.detach(), grad]
    loss, grad = eng.distill_step(s["logits"], s["index"], s["teacher"], dim=s["dim"], temperature=c["temperature"], tail=c["tail"], weight=s["weight"])
    return [loss, grad]


# ---- the plain form -------------------------------------------------------------------------------------------------------------

def _lse(y, dim, dtype=torch.float32):
    """dtype: in which the exponentials are summed and the logarithm is taken"""
    m = y.amax(dim, keepdim=True)
    m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
    return (y - m).exp_().sum(dim, keepdim=True, dtype=dtype).log_() + m


def _top(z, k, dim):
    """The k largest along dim, ties to the lowest index: unique integer keys (value in order, index reversed)."""
    z = z + 0.0                                            # -0 -> +0
    bits = z.view(torch.int32)
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).to(torch.int64)
    n = z.shape[dim]
    pos = torch.arange(n - 1, -1, -1, device=z.device).view([n if a == dim else 1 for a in range(z.dim())])
    key = torch.topk(order.mul_(1 << 32).add_(pos), k, dim=dim).values
    return (n - 1) - (key & 0xFFFFFFFF)


def _run_plain(s):
    c, dim = s["case"], s["dim"]
    x = s["logits"]
    inv_t = 1.0 / c["temperature"]
    if c["op"] in ("score", "train"):
        z = x.float()
        y = z * inv_t if inv_t != 1.0 else z
        lse = _lse(y, dim)
        logp = y - lse
        tok = s["tokens"].unsqueeze(dim)
        used = tok != IGNORE
        lp = torch.where(used, logp.gather(dim, tok.clamp(min=0)), torch.zeros_like(lse))
        p = logp.exp()
        plogp = torch.where(p > 0, p * logp, torch.zeros_like(p))
        ent = -plogp.sum(dim, keepdim=True)
        if c["op"] == "score":
            out = [lp.squeeze(dim), ent.squeeze(dim), lse.squeeze(dim)]
            if c["top"]:
                idx = _top(z, c["top"], dim)
                out += [logp.gather(dim, idx), idx.to(torch.int32)]
            return out
        g = torch.where(used, s["g_logprob"].unsqueeze(dim), torch.zeros_like(lse))
        ge = s["g_entropy"].unsqueeze(dim)
        grad = -(g * p) - ge * (plogp + p * ent)
        grad.scatter_add_(dim, tok.clamp(min=0), g)
        return [lp.squeeze(dim), ent.squeeze(dim), grad.mul_(inv_t).to(x.dtype)]

    # distances to the row's maximum are exact in float32 where the logits themselves, divided by the temperature, are not; the row's few
    # scalars (log sums, the listed terms, which nearly cancel for a good student) are combined in 64 bits
    t2 = c["temperature"] ** 2
    d = x.float()
    d = (d - d.amax(dim, keepdim=True)) * inv_t
    lse = _lse(d, dim, torch.float64)
    at = s["index"].long()
    valid = at >= 0
    at = at.clamp(min=0)
    t = s["teacher"].double()
    t = torch.where(valid, t, torch.full_like(t, float("-inf")))
    logq = d.gather(dim, at).double() - lse
    zero = torch.zeros_like(t)
    if c["tail"]:
        p = t.exp()
        rest = (1.0 - p.sum(dim, keepdim=True)).clamp_(min=0.0)
        others = d.clone()                                  # the classes that are not listed
        spot = torch.where(valid, at, at[(slice(None),) * dim + (slice(0, 1),)].expand_as(at))
        others.scatter_(dim, spot, float("-inf"))
        lse_rest = _lse(others, dim, torch.float64)
        per = torch.where(p > 0, p * (t - logq), zero).sum(dim, keepdim=True)
        bucket = (rest > 0) & (lse_rest > float("-inf"))
        per = per + torch.where(bucket, rest * (rest.clamp(min=1e-300).log() - (lse_rest - lse)), torch.zeros_like(lse))
        rest = torch.where(bucket, rest, torch.zeros_like(rest))
    else:
        m = t.amax(dim, keepdim=True)
        e = (t - m).exp()
        z = e.sum(dim, keepdim=True)
        p = e / z
        per = torch.where(p > 0, p * ((t - m) - z.log() - logq), zero).sum(dim, keepdim=True)
    loss = (per * t2).squeeze(dim)
    if c["op"] == "loss":
        return [loss.float()]
    w = s["weight"].unsqueeze(dim)
    grad = d.sub_(lse.float()).exp_()
    if c["tail"]:
        grad.mul_((p.sum(dim, keepdim=True) + rest).float())
        share = torch.where(bucket, lse_rest, torch.zeros_like(lse)).float()
        grad -= others.sub_(share).exp_().mul_(rest.float())
    grad.scatter_add_(dim, at, -torch.where(valid, p, zero).float())
    grad = (grad * (w * c["temperature"])).to(x.dtype)
    return [(loss * s["weight"]).float() if c["op"] == "step" else loss.float(), grad]


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------------------

def exact(case, seed):
    s = _inputs(case, seed)
    if s["logits"].numel() > 700_000_000:
        return None
    dim = _shape(case)[1]
    T = float(case["temperature"])
    rows_first = [a for a in range(s["logits"].dim()) if a != dim] + [dim]
    y = s["logits"].permute(rows_first).double() / T                       # [..., C]
    back = [rows_first.index(a) for a in range(len(rows_first))]
    logq = torch.log_softmax(y, dim=-1)
    q = logq.exp()
    C = y.shape[-1]
    if case["op"] in ("score", "train"):
        tok = s["tokens"]
        hit = torch.nn.functional.one_hot(tok.clamp(min=0), C) if C <= 64 else None
        lp = torch.take_along_dim(logq, tok.clamp(min=0)[..., None], -1)[..., 0]
        lp = torch.where(tok == IGNORE, 0.0, lp)
        safe = torch.where(q > 0, logq, 0.0)
        H = -(q * safe).sum(-1)
        if case["op"] == "score":
            out = [lp, H, torch.logsumexp(y, -1)]
            if case["top"]:
                srt = torch.sort(s["logits"].permute(rows_first).float(), dim=-1, descending=True, stable=True).indices[..., :case["top"]]
                out += [torch.take_along_dim(logq, srt, -1).permute(back), srt.permute(back).to(torch.int32)]
            return out
        g = torch.where(tok == IGNORE, 0.0, s["g_logprob"].double())
        grad = -q * g[..., None] - s["g_entropy"].double()[..., None] * q * (safe + H[..., None])
        if hit is not None:
            grad += hit * g[..., None]
        else:
            grad.scatter_add_(-1, tok.clamp(min=0)[..., None], g[..., None])
        return [lp, H, (grad / T).permute(back)]
    idx = s["index"].permute(rows_first).long()
    t = s["teacher"].permute(rows_first).double()
    ok = idx >= 0
    t = torch.where(ok, t, float("-inf"))
    slot = torch.where(ok, idx, C)                                          # one spare class takes the unused entries
    logp = t if case["tail"] else torch.log_softmax(t, -1)
    p = logp.exp()
    target = torch.zeros(y.shape[:-1] + (C + 1,), dtype=torch.float64, device=y.device).scatter_add_(-1, slot, p)[..., :C]
    terms = torch.where(p > 0, p * (logp - torch.take_along_dim(logq, idx.clamp(min=0), -1)), 0.0)
    loss = terms.sum(-1)
    grad = q * p.sum(-1, keepdim=True) - target
    if case["tail"]:
        named = torch.zeros(y.shape[:-1] + (C + 1,), dtype=torch.bool, device=y.device).scatter_(-1, slot, True)[..., :C]
        r = (1.0 - p.sum(-1, keepdim=True)).clamp(min=0.0)
        free = torch.where(named, float("-inf"), logq)
        some = (r > 0) & ~named.all(-1, keepdim=True)
        lr = torch.where(some, torch.logsumexp(free, -1, keepdim=True), 0.0)
        loss = loss + torch.where(some, r * (torch.log(torch.where(some, r, 1.0)) - lr), 0.0)[..., 0]
        grad = grad + torch.where(some, r * (q - (free - lr).exp()), 0.0)
    loss = loss * T * T
    if case["op"] == "loss":
        return [loss]
    w = s["weight"].double()
    return [loss * w if case["op"] == "step" else loss, (grad * T * w[..., None]).permute(back)]


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------------

def work(case):
    if case["layout"] == "voxels":
        rows = case["batch"] * case["side"] ** 3
        classes = case["classes"] - (1 if case["op"] == "score" else 0)
    else:
        rows, classes = case["batch"] * case["rows"], case["classes"]
    logits = rows * classes * SIZES[case["dtype"]]
    if case["op"] == "score":
        nbytes = logits + rows * (8 + 12 + 8 * case["top"])                 # tokens in; log probability, entropy, lse, alternatives out
    elif case["op"] == "train":
        nbytes = 2 * logits + rows * (8 + 8 + 8)                            # tokens and two upstream gradients in; two results out
    else:
        nbytes = logits + rows * (8 * case["k"] + 4)                        # the teacher's list in; the loss out
        if case["op"] != "loss":
            nbytes += logits + rows * 4
    per_logit = {"score": 5, "train": 11, "loss": 4, "grad": 8, "step": 8}[case["op"]]
    return {"bytes": nbytes, "flops": rows * classes * per_logit}
