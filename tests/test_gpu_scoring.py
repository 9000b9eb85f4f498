"""Class scoring and distillation on the GPU against float64 (oracle/score_oracle.py).

Error bounds.  u = 2^-24 (half a step of float32, relative).  The kernels sum float32 exponentials: at most ~n/64 terms one after the
other per thread, each off by a few u (2^x of the hardware: 2 u) plus u times its exponent's rounding, |x| <= ~3 |y - m|, weighted with the
probabilities; a distribution over C classes has a mean |y - m| of at most ~log C + a few.  Gradients take p = 2^(z c - lse log2 e) whose
exponent is off by u times the magnitudes of z c and of the stored float32 lse.  Results of fewer bits add half a step of their type."""
import math

import numpy as np
import pytest
import torch

from oracle import score_oracle as so

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
NEG = float("-inf")


@pytest.fixture(scope="module")
def eng():
    from mica_amd.engine import Engine
    e = Engine(0, max_batch=1, tile_size=4)
    yield e
    e.close()


def _rng(seed):
    return torch.Generator().manual_seed(seed)


def _logits(shape, seed, dtype, scale=3.0):
    g = _rng(seed)
    z = torch.randn(shape, generator=g) * scale
    z = z + (torch.rand(shape, generator=g) < 2.0 / max(2, shape[-1])) * 12.0
    return z.to(DT[dtype])


def _log2c(c):
    return math.log2(c) + 4.0


def _near(got, want, tol):
    """got against want, both infinities and NaN at the same places; tol per element"""
    got = got.detach().cpu().double()
    want = want.double()
    assert got.shape == want.shape
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    inf = torch.isinf(want)
    assert torch.equal(torch.isinf(got), inf) and torch.equal(got[inf], want[inf])
    ok = ~(inf | torch.isnan(want))
    tol = torch.as_tensor(tol, dtype=torch.float64).expand(want.shape)
    worst = float(((got - want).abs() / tol)[ok].max()) if bool(ok.any()) else 0.0
    assert worst <= 1.0, f"{worst} times the bound"


def _check_score(eng, z, tok, top, temperature=1.0, dim=-1, rows_last=None):
    """z on the CPU (class axis dim); runs the GPU and compares"""
    r = eng.token_logprobs(z if z.is_cuda else z.cuda(), None if tok is None else tok.cuda(), top=top, dim=dim, temperature=temperature)
    zc = z.cpu().movedim(dim, -1)
    w = so.score(zc, tok, top, temperature)
    C = zc.shape[-1]
    terms = 16 + C / 64 + 4 * _log2c(C)
    lse_mag = torch.nan_to_num(w["lse"].abs(), posinf=0.0, neginf=0.0)
    _near(r.lse, w["lse"], U * (terms + 2 * lse_mag))
    if tok is not None:
        _near(r.logprob, w["logprob"], U * (terms + 6 * torch.nan_to_num(w["logprob"].abs(), posinf=0.0, neginf=0.0)))
    else:
        assert r.logprob is None
    # entropy: the same terms weighted once more with |log p|
    _near(r.entropy, w["entropy"], U * (32 + C / 32 + 6 * _log2c(C) ** 2))
    if top:
        idx = r.top_index.cpu().movedim(dim, -1)
        assert idx.dtype == torch.int32 and torch.equal(idx.long(), w["top_index"])
        tv = w["top_logprob"]
        _near(r.top_logprob.movedim(dim, -1), tv, U * (terms + 6 * torch.nan_to_num(tv.abs(), posinf=0.0, neginf=0.0)))
    else:
        assert r.top_logprob is None and r.top_index is None
    return r


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,classes,top", [
    (1, 1, 1), (3, 2, 2), (257, 20, 5), (1, 21, 21), (300, 24, 0), (65, 25, 3), (5, 33, 33), (70, 64, 64), (2, 65, 64), (9, 100, 5), (5, 255, 20),
    (3, 256, 64), (6, 1000, 1), (2, 4095, 64), (3, 4096, 20), (2, 4097, 5), (600, 4103, 3), (3, 9001, 64), (1, 33000, 20), (515, 8200, 0), (2, 70001, 64),
])
def test_scores(eng, dtype, rows, classes, top):
    z = _logits((rows, classes), rows * 7 + classes, dtype)
    tok = torch.randint(0, classes, (rows,), generator=_rng(3))
    tok[rows // 2] = -100 if rows > 2 else tok[rows // 2]
    _check_score(eng, z, tok, top)
    _check_score(eng, z, tok.int(), top, temperature=0.7)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("classes", [7, 20, 64, 129, 4100, 20000])
@pytest.mark.parametrize("top", [1, 20])
def test_masked_rows(eng, dtype, classes, top):
    """-inf and the type's lowest value in masked places, rows with one class left, with none, with NaN and +inf"""
    top = min(top, classes)
    low = torch.finfo(DT[dtype]).min
    z = _logits((12, classes), 5 + classes, dtype)
    g = _rng(9)
    drop = torch.rand((classes,), generator=g) < 0.7
    z[0, drop] = NEG
    z[1, drop] = low
    z[2] = NEG
    z[3] = low
    z[4] = NEG
    z[4, classes // 2] = -3.0
    z[5] = low
    z[5, classes - 1] = 2.0
    z[6] = NEG
    z[6, ::3] = low
    z[7] = 0.0
    z[8] = -0.0
    z[8, ::2] = 0.0
    z[9] = torch.finfo(DT[dtype]).max
    z[10] = NEG
    z[10, classes - 1] = low
    z[11, drop] = -1e4
    tok = torch.tensor([classes - 1, 0, 0, classes - 1, classes // 2, classes - 1, 0, 0, 1, 2, classes - 1, 0])
    _check_score(eng, z, tok, top)
    # NaN and +inf: NaN results, and alternatives that stay distinct classes; the other rows are not touched by it
    y = z.clone()
    y[0, classes // 3] = float("nan")
    y[1, 2] = float("inf")
    y[2] = float("nan")
    r = eng.token_logprobs(y.cuda(), tok.cuda(), top=top)
    assert bool(torch.isnan(torch.stack([r.logprob[:3], r.entropy[:3], r.lse[:3]])).all()) and bool(torch.isnan(r.top_logprob[:3]).all())
    for i in range(12):
        idx = r.top_index[i].cpu()
        assert len(set(idx.tolist())) == top and int(idx.min()) >= 0 and int(idx.max()) < classes
    clean = eng.token_logprobs(z.cuda(), tok.cuda(), top=top)
    assert torch.equal(r.logprob[3:], clean.logprob[3:]) and torch.equal(r.top_index[3:], clean.top_index[3:])


@pytest.mark.parametrize("classes", [20, 64, 300, 5000, 40000])
@pytest.mark.parametrize("order", ["few", "equal", "ascending", "descending", "blocks"])
def test_top_alternatives_ties_and_orders(eng, classes, order):
    z = torch.zeros(3, classes)
    if order == "few":
        z = torch.randint(0, 4, (3, classes), generator=_rng(1)).float()
    elif order == "ascending":
        z += torch.arange(classes) / classes
    elif order == "descending":
        z -= torch.arange(classes) / classes
    elif order == "blocks":                         # everything large in one place
        z[:, classes // 2: classes // 2 + min(200, classes // 4)] = 5.0
    for top in (1, 7, min(64, classes)):
        _check_score(eng, z, None, top)
        if order != "ascending" and order != "descending":
            _check_score(eng, z.bfloat16(), None, top)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("rows,classes", [(1, 131072), (2, 131073), (1, 300001), (3, 66000)])
def test_few_long_rows_are_cut_and_joined(eng, dtype, rows, classes):
    z = _logits((rows, classes), classes, dtype)
    z[0, classes - 3:] = NEG
    tok = torch.full((rows,), classes - 4)
    for top in (0, 20, 64):
        _check_score(eng, z, tok, top, temperature=1.3)
    z[0] = NEG
    _check_score(eng, z, tok, 5)
    z[0, 70] = 1.0
    _check_score(eng, z, tok, 64)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_layouts_and_strides(eng, dtype):
    z = _logits((2, 21, 5, 6, 7), 11, dtype)
    d = z.cuda()
    tok = torch.randint(0, 20, (2, 5, 6, 7), generator=_rng(2))
    _check_score(eng, d[:, 1:], tok, 3, dim=1)                                       # a head's slice, in place
    _check_score(eng, d, None, 21, dim=1)
    _check_score(eng, d[:, :, 1:4, :, ::2], None, 2, dim=1)                          # a crop: copied
    _check_score(eng, d.movedim(1, -1), None, 4, dim=-1)                             # few classes at a stride, last
    _check_score(eng, d.permute(1, 0, 2, 3, 4), None, 4, dim=0)
    s = _logits((3, 9, 501), 12, dtype).cuda()
    nxt = torch.randint(0, 501, (3, 8), generator=_rng(4))
    _check_score(eng, s[:, :-1], nxt, 5)                                             # shifted: two row axes
    _check_score(eng, s[:, 1:, 3:], nxt * 0, 5)                                      # every row at another alignment
    _check_score(eng, s[:, :, ::2], None, 5)
    _check_score(eng, s.transpose(1, 2), None, 5, dim=1)                             # many classes in the middle
    _check_score(eng, s[:1].expand(3, 9, 501), None, 5)                              # broadcast rows
    long = _logits((5, 9003), 13, dtype).cuda()
    _check_score(eng, long[:, 1:], None, 20)
    _check_score(eng, long[1:, 2:-1], None, 0)
    _check_score(eng, long[0], None, 3, dim=0)                                       # a single distribution


def test_tokens_out_of_range_are_nan_and_nothing_else_changes(eng):
    for classes in (20, 500, 9000):
        z = _logits((6, classes), classes, "f32").cuda()
        tok = torch.tensor([0, classes, -1, -100, 2 ** 40, classes - 1]).cuda()
        r = eng.token_logprobs(z, tok)
        assert torch.isnan(r.logprob).tolist() == [False, True, True, False, True, False] and float(r.logprob[3]) == 0.0
        assert not bool(torch.isnan(r.entropy).any())
        g = eng.token_logprobs_backward(z, tok, r.lse, r.entropy, g_logprob=torch.ones(6, device="cuda"))
        assert torch.isnan(g).all(-1).tolist() == [False, True, True, False, True, False] and torch.isnan(g).any(-1).tolist() == [False, True, True, False, True, False]
        assert float(g[3].abs().max()) == 0.0
        assert float(eng.token_logprobs(z, tok, ignore_index=classes).logprob[1]) == 0.0


def test_offsets_beyond_32_bits(eng):
    """2.2e9 logits: the last rows lie beyond 2^31 elements (and 2^32 bytes)"""
    rows, classes = 17000, 131072
    z = torch.zeros((rows, classes), dtype=torch.bfloat16, device="cuda")
    z[-3:] = _logits((3, classes), 1, "bf16").cuda()
    tok = torch.full((rows,), 77, device="cuda")
    r = eng.token_logprobs(z, tok, top=5)
    want = eng.token_logprobs(z[-3:].clone(), tok[-3:], top=5)
    w = so.score(z[-3:].cpu(), tok[-3:].cpu(), 5)
    assert torch.equal(r.top_index[-3:].cpu().long(), w["top_index"])
    assert float((r.logprob[-3:].cpu().double() - w["logprob"]).abs().max()) < U * 4096 and torch.equal(want.top_index, r.top_index[-3:])
    assert r.top_index[:-3].unique(dim=0).tolist() == [[0, 1, 2, 3, 4]]
    g = eng.token_logprobs_backward(z, tok, r.lse, r.entropy, g_logprob=torch.ones(rows, device="cuda"))
    part = eng.token_logprobs_backward(z[-3:].clone(), tok[-3:], r.lse[-3:].clone(), r.entropy[-3:].clone(), g_logprob=torch.ones(3, device="cuda"))
    assert torch.equal(g[-3:], part)
    del z, g
    torch.cuda.empty_cache()


# ---- gradients of the scores --------------------------------------------------------------------------------------------------------------

def _half_step(dtype, want):
    t = DT[dtype]
    if t == torch.float32:
        return U * want.abs() + 1e-37
    return torch.finfo(t).eps / 2 * want.abs() + (torch.finfo(t).smallest_normal * torch.finfo(t).eps)


def _check_score_grad(eng, z, tok, dtype, gl, ge, gs, temperature=1.0, dim=-1):
    """through autograd, against the formula"""
    from mica_amd import scoring
    x = (z if z.is_cuda else z.cuda()).detach().requires_grad_()
    r = scoring.token_logprobs(eng, x, None if tok is None else tok.cuda(), dim=dim, temperature=temperature, top=min(3, z.shape[dim]))
    outs, ups = [], []
    for o, g in ((r.logprob, gl), (r.entropy, ge), (r.lse, gs)):
        if g is not None:
            outs.append(o)
            ups.append(g.cuda())
    got, = torch.autograd.grad(outs, [x], ups)
    assert got.dtype == x.dtype and got.shape == x.shape
    zc = z.cpu().movedim(dim, -1)
    want = so.score_grad(zc, tok, gl, ge, gs, temperature)
    w = so.score(zc, tok, temperature=temperature)
    p = torch.exp(w["logp"])
    y = torch.nan_to_num(zc.double().abs() / temperature, posinf=0.0)
    y = torch.where(p > 0, y, torch.zeros_like(y))
    lse = torch.nan_to_num(w["lse"].abs(), posinf=0.0)[..., None]
    logp = torch.where(p > 0, w["logp"].abs(), torch.zeros_like(p))
    zero = torch.zeros_like(lse[..., 0])
    a = ((gl if gl is not None else zero).double().abs() + (gs if gs is not None else zero).double().abs())[..., None]
    e = (ge if ge is not None else zero).double().abs()[..., None]
    H = w["entropy"][..., None]
    # e carries the entropy's own error (bounded above by its test) besides the roundings of p
    herr = U * (32 + zc.shape[-1] / 32 + 6 * _log2c(zc.shape[-1]) ** 2)
    tol = p * (U * (16 + 3 * y + 4 * lse) * (a + e * (logp + H)) + e * (herr + U * (4 * y + 4 * lse))) / temperature
    tol = tol + 4 * U * a / temperature * (want.abs() > 0) + _half_step(dtype, want) + 1e-37
    _near(got.movedim(dim, -1), want, tol)
    return got


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,classes", [(1, 1), (3, 2), (257, 20), (70, 64), (3, 65), (9, 1001), (3, 4096), (2, 4099), (40, 9001), (1, 70001)])
def test_score_gradients(eng, dtype, rows, classes):
    z = _logits((rows, classes), rows + classes, dtype)
    g = _rng(8)
    tok = torch.randint(0, classes, (rows,), generator=g)
    gl, ge, gs = (torch.randn((rows,), generator=g) for _ in range(3))
    tok[0] = -100
    _check_score_grad(eng, z, tok, dtype, gl, ge, gs)
    _check_score_grad(eng, z, tok, dtype, gl, None, None, temperature=0.6)
    _check_score_grad(eng, z, None, dtype, None, ge, None, temperature=1.4)
    _check_score_grad(eng, z, None, dtype, None, None, gs)


@pytest.mark.parametrize("classes", [20, 300, 5000])
def test_score_gradients_of_masked_rows(eng, classes):
    z = _logits((5, classes), classes, "f32")
    z[0, ::2] = NEG
    z[1] = NEG
    z[2] = torch.finfo(torch.float32).min
    z[2, 3] = 1.0
    z[3] = NEG
    z[3, 4] = 1.0
    tok = torch.tensor([1, 0, 3, 4, 2])
    gl, ge = torch.tensor([1., 2., -1., .5, 1.]), torch.tensor([.1, .2, .3, -.5, 1.])
    got = _check_score_grad(eng, z, tok, "f32", gl, ge, None)
    assert float(got[1].abs().max()) == 0.0


def test_score_gradients_layouts_and_broadcast(eng):
    z = _logits((2, 21, 4, 5, 6), 3, "f32")
    g = _rng(4)
    tok = torch.randint(0, 21, (2, 4, 5, 6), generator=g)
    tok[torch.rand(tok.shape, generator=g) < 0.5] = -100
    gl, ge = torch.randn(tok.shape, generator=g), torch.randn(tok.shape, generator=g)
    _check_score_grad(eng, z, tok, "f32", gl, ge, None, dim=1)
    _check_score_grad(eng, z.cuda().movedim(1, -1), tok, "f32", gl, ge, None)
    s = _logits((3, 400, 5), 5, "bf16")
    t2 = torch.randint(0, 400, (3, 5), generator=g)
    _check_score_grad(eng, s, t2, "bf16", torch.randn((3, 5), generator=g), None, None, dim=1)
    sl = _logits((3, 6, 501), 6, "bf16").cuda()[:, :-1]
    _check_score_grad(eng, sl, torch.randint(0, 501, (3, 5), generator=g), "bf16", torch.randn((3, 5), generator=g), None, None)
    # a broadcast input's gradient is the sum over what it was broadcast to
    from mica_amd import scoring
    leaf = _logits((1, 300), 7, "f32").cuda().requires_grad_()
    tk = torch.arange(4).cuda()
    scoring.token_logprobs(eng, leaf.expand(4, 300), tk).logprob.sum().backward()
    want = so.score_grad(leaf.detach().cpu().expand(4, 300), tk.cpu(), torch.ones(4)).sum(0)
    assert float((leaf.grad.cpu().double()[0] - want).abs().max()) < U * 600
    # the sum's expanded upstream gradient, and a slice that torch differentiates itself
    full = _logits((2, 21, 3, 3, 3), 8, "f32").cuda().requires_grad_()
    scoring.token_logprobs(eng, full[:, 1:], dim=1).entropy.mean().backward()
    want = so.score_grad(full.detach().cpu()[:, 1:].movedim(1, -1), None, g_entropy=torch.full((2, 3, 3, 3), 1 / 54)).movedim(-1, 1)
    assert float(full.grad[:, 0].abs().max()) == 0.0 and float((full.grad[:, 1:].cpu().double() - want).abs().max()) < U * 200


# ---- distillation -------------------------------------------------------------------------------------------------------------------------

def _teacher(z, k, seed, index_dtype=torch.int32, pad=0.0, dim=-1, temperature=1.0):
    t = z.float() + torch.randn(z.shape, generator=_rng(seed))
    t = torch.where(torch.isneginf(z.float()), torch.full_like(t, -20.0), t) / temperature
    lp = torch.log_softmax(t.double(), dim).float()
    v, i = torch.topk(lp, k, dim=dim)
    i = i.to(index_dtype)
    if pad:
        i[torch.rand(i.shape, generator=_rng(seed + 1)) < pad] = -1
    return i, v


def _check_distill(eng, z, idx, val, dtype, temperature=1.0, tail=False, dim=-1, weight=None):
    """loss, autograd gradient and the one-call step against the formula"""
    from mica_amd import scoring
    zg, ig, vg = (t if t.is_cuda else t.cuda() for t in (z, idx, val))
    zc, ic, vc = (t.cpu().movedim(dim, -1) for t in (z, idx, val))
    want, wgrad, parts = so.distill(zc, ic, vc, temperature, tail)
    C = zc.shape[-1]
    terms = 16 + C / 64 + 4 * _log2c(C)
    lq = torch.nan_to_num(parts["lq"].abs(), posinf=0.0, neginf=0.0).amax(-1)
    t2 = temperature ** 2
    fin = torch.nan_to_num(want.abs(), posinf=0.0, nan=0.0)
    mass = parts["mass"][..., 0].clamp(min=1.0)
    loss_tol = t2 * U * (terms + 6 * lq) * mass + 2 * U * fin
    x = zg.detach().requires_grad_()
    loss = scoring.distill_loss(eng, x, ig, vg, dim=dim, temperature=temperature, tail=tail)
    _near(loss, want, loss_tol)
    w = torch.rand(want.shape, generator=_rng(77)) + 0.5 if weight is None else weight
    got, = torch.autograd.grad([loss], [x], [w.cuda()])
    wg = wgrad * w.double()[..., None]
    q, share, rest = parts["q"], parts["share"], parts["rest"][..., None]
    y = torch.nan_to_num(zc.double().abs() / temperature, posinf=0.0)
    y = torch.where(q > 0, y, torch.zeros_like(y))
    lse = torch.nan_to_num(parts["lse"].abs(), posinf=0.0)[..., None]
    norm = torch.nan_to_num(vc.double().abs(), posinf=0.0, neginf=0.0).amax(-1, keepdim=True)
    # the unlisted classes' gradient is (mass q_rest - r) e^{y - lse_rest}: the factor is off by u of its two terms, r <= 1
    tol = temperature * w.double().abs()[..., None] * U * ((16 + 3 * y + 4 * lse + terms) * (q * parts["mass"] + share * rest) + (16 + 6 * norm) * parts["target"])
    tol = tol + 4 * U * wg.abs() + _half_step(dtype, wg) + 1e-37
    assert got.dtype == x.dtype
    _near(got.movedim(dim, -1), wg, tol)
    sl, sg = eng.distill_step(zg, ig, vg, dim=dim, temperature=temperature, tail=tail, weight=w.cuda())
    zero = w == 0
    _near(sl, torch.where(zero, torch.zeros_like(want), want * w.double()), loss_tol * w.double().abs() + 2 * U * fin * w.double().abs() + 1e-37)
    _near(sg.movedim(dim, -1), torch.where(zero[..., None], torch.zeros_like(wg), wg), tol)
    ul, ug = eng.distill_step(zg, ig, vg, dim=dim, temperature=temperature, tail=tail)
    _near(ul, want, loss_tol)
    return loss, got


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("rows,classes,k", [
    (1, 1, 1), (3, 2, 1), (257, 21, 4), (5, 20, 20), (40, 64, 64), (70, 33, 100 // 4), (3, 65, 8), (9, 1001, 16), (5, 4096, 256), (2, 4097, 64), (40, 9001, 100),
    (600, 5003, 3), (1, 70001, 64), (2, 140000, 200)])
def test_distillation(eng, dtype, tail, rows, classes, k):
    z = _logits((rows, classes), rows + 3 * classes, dtype)
    idx, val = _teacher(z, k, 4)
    _check_distill(eng, z, idx, val, dtype, 1.0, tail)
    idx, val = _teacher(z, k, 5, torch.int64, pad=0.3, temperature=1.6)
    _check_distill(eng, z, idx, val, dtype, 1.6, tail)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("classes", [20, 300, 5000])
def test_distillation_lists_and_masks(eng, tail, classes):
    z = _logits((10, classes), classes, "f32")
    idx, val = _teacher(z, 6, 1)
    idx[0] = -1                                          # no used entry
    idx[1, 1:] = -1                                      # one
    idx[2, 1] = idx[2, 0]                                # a class named twice
    idx[2, 4] = idx[2, 5]
    val[3, 2:] = NEG                                     # listed with probability 0
    z[4] = NEG                                           # an empty student row
    z[5] = NEG                                           # all its mass on one class the teacher names
    z[5, idx[5, 0].item()] = 1.0
    val[5, 1:] = NEG
    z[6, :] = NEG                                        # its mass on the listed classes
    z[6, idx[6].long()] = torch.randn(6, generator=_rng(2))
    z[7, 0] = torch.finfo(torch.float32).min
    z[8, idx[8, 3].item()] = NEG                         # the teacher wants what the student forbids: +inf
    val[9] = NEG
    w = torch.rand((10,), generator=_rng(3)) + 0.1
    w[8] = 0.0
    z8 = z.clone()
    z8[8] = _logits((1, classes), 5, "f32")[0]
    _check_distill(eng, z8, idx, val, "f32", 1.3, tail, weight=w)
    loss, aux = eng.distill_loss(z.cuda(), idx.cuda(), val.cuda(), tail=tail)
    assert math.isinf(float(loss[8])) and float(loss[8]) > 0 and math.isinf(float(loss[4])) and float(loss[0]) == 0.0
    # an index that is no class, a NaN in the list or in the row: NaN there and nowhere else
    bad = idx.clone()
    bad[1, 0] = classes
    bv = val.clone()
    bv[2, 0] = float("nan")
    bz = z.clone()
    bz[3, classes - 1] = float("nan")
    loss2, aux2 = eng.distill_loss(bz.cuda(), bad.cuda(), bv.cuda(), tail=tail)
    keep = [0, 4, 5, 6, 7, 8, 9]
    assert torch.isnan(loss2[1:4]).all() and torch.equal(loss2[keep], loss[keep])
    ones = torch.ones(10, device="cuda")
    g = eng.distill_backward(bz.cuda(), bad.cuda(), bv.cuda(), aux2, ones, tail=tail)
    clean = eng.distill_backward(z.cuda(), idx.cuda(), val.cuda(), aux, ones, tail=tail)
    assert torch.isnan(g[1:4]).any(-1).all() and torch.equal(g[keep], clean[keep])
    # weight 0 hides them
    w = torch.ones(10, device="cuda")
    w[1:4] = 0.0
    w[4] = w[8] = 0.0
    sl, sg = eng.distill_step(bz.cuda(), bad.cuda(), bv.cuda(), tail=tail, weight=w)
    assert bool(torch.isfinite(sl).all()) and bool(torch.isfinite(sg).all()) and float(sg[1:5].abs().max()) == 0.0 and float(sl[1:5].abs().max()) == 0.0


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("tail", [False, True])
def test_distillation_layouts(eng, dtype, tail):
    z = _logits((2, 21, 4, 5, 6), 1, dtype)
    idx, val = _teacher(z, 4, 2, dim=1)
    _check_distill(eng, z, idx, val, dtype, 1.0, tail, dim=1)
    _check_distill(eng, z.cuda()[:, 1:], idx.clamp(max=19), val, dtype, 1.0, tail, dim=1)
    s = _logits((3, 6, 501), 3, dtype).cuda()[:, :-1]
    idx, val = _teacher(s.cpu(), 7, 4)
    _check_distill(eng, s, idx, val.bfloat16(), dtype, 1.0, tail)
    m = _logits((3, 400, 5), 5, dtype)
    idx, val = _teacher(m, 9, 6, dim=1)
    _check_distill(eng, m, idx, val, dtype, 2.0, tail, dim=1)
    u = _logits((4, 9004), 7, dtype).cuda()[:, 1:]
    idx, val = _teacher(u.cpu(), 33, 8)
    _check_distill(eng, u, idx.cuda().t().contiguous().t(), val, dtype, 1.0, tail)


def test_distillation_towards_the_own_distribution_is_zero(eng):
    z = _logits((4, 3000), 1, "f32").cuda()
    s = eng.token_logprobs(z, top=64, temperature=1.5)
    loss, grad = eng.distill_step(z, s.top_index, s.top_logprob, temperature=1.5, tail=True)
    # log p and log q differ by the rounding of the stored log probabilities
    assert float(loss.abs().max()) < 2.25 * U * 64 and float(grad.abs().max()) < 1.5 * U * 128


# ---- how the calls behave in a program -------------------------------------------------------------------------------------------------------

def _all_outputs(eng, z, tok, idx, val, w):
    s = eng.token_logprobs(z, tok, top=5)
    g = eng.token_logprobs_backward(z, tok, s.lse, s.entropy, w, w)
    loss, aux = eng.distill_loss(z, idx, val, tail=True)
    dg = eng.distill_backward(z, idx, val, aux, w, tail=True)
    return list(s) + [g, loss, dg] + list(eng.distill_step(z, idx, val, weight=w))


@pytest.mark.parametrize("rows,classes", [(300, 20), (40, 700), (2, 50000)])
def test_results_are_deterministic_and_ordered_on_the_current_stream(eng, rows, classes):
    z = _logits((rows, classes), 1, "bf16")
    idx, val = _teacher(z, 5, 2)
    d = [t.cuda() for t in (z, torch.randint(0, classes, (rows,), generator=_rng(1)), idx, val, torch.rand((rows,), generator=_rng(2)))]
    first = _all_outputs(eng, *d)
    side = torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.default_stream())
            filler = torch.zeros(1 << 26, device="cuda")
            for _ in range(4):
                filler += 1
            late = d[0].float().mul(1.0).to(torch.bfloat16)            # produced behind the filler on this stream
            again = _all_outputs(eng, late, *d[1:])
        torch.cuda.default_stream().wait_stream(side)
        for a, b in zip(first, again):
            assert torch.equal(a, b)


@pytest.mark.parametrize("rows,classes", [(300, 20), (40, 700), (2, 50000)])
def test_capture_and_replay(eng, rows, classes):
    """two graphs with different inputs, replayed in turn with eager work between"""
    def inputs(seed):
        z = _logits((rows, classes), seed, "bf16")
        idx, val = _teacher(z, 5, seed + 1)
        return [t.cuda() for t in (z, torch.randint(0, classes, (rows,), generator=_rng(seed)), idx, val, torch.rand((rows,), generator=_rng(2)))]
    a, b = inputs(1), inputs(50)
    want_a, want_b = _all_outputs(eng, *a), _all_outputs(eng, *b)
    graphs = []
    for d in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = _all_outputs(eng, *d)
        graphs.append((g, out))
    for i in range(4):
        for (g, out), want in zip(graphs, (want_a, want_b)):
            for o in out:
                o.zero_()
            g.replay()
            eager = _all_outputs(eng, *b)
            torch.cuda.synchronize()
            assert all(torch.equal(o, w) for o, w in zip(out, want)) and all(torch.equal(o, w) for o, w in zip(eager, want_b))
    # new values in the captured inputs
    a[0].copy_(b[0])
    a[1].copy_(b[1])
    a[2].copy_(b[2])
    a[3].copy_(b[3])
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(graphs[0][1], want_b))


def test_refusals_leave_no_error_behind(eng):
    from mica_amd._cabi import MicaHipError
    z = torch.zeros(3, 30, device="cuda")
    for call in (lambda: eng.token_logprobs(z, top=31), lambda: eng.token_logprobs(z.cpu()), lambda: eng.token_logprobs(z, torch.zeros(3, dtype=torch.int64)),
                 lambda: eng.token_logprobs(z, temperature=0.0), lambda: eng.distill_loss(z, torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, 2, device="cuda"))):
        with pytest.raises(MicaHipError):
            call()
    assert float(eng.token_logprobs(z).entropy[0]) == pytest.approx(math.log(30), abs=1e-5)


def test_candidates_residues_and_a_student_of_the_network(weights):
    """as a user strings them together: the network's amino-acid head scored at every voxel, residue fits at candidates, and one gradient
    step of a student towards the alternatives"""
    from mica_amd import clustering, scoring
    from mica_amd.model import MICA
    from mica_amd.synth import synth_density
    m = MICA(max_batch=1).to("cuda")
    m.load_state_dict(weights)
    x = torch.from_numpy(synth_density((1, 1, 16, 16, 16), 7)).cuda()
    aa = m.forward(x, None)[2]
    res = torch.randint(0, 20, (1, 16, 16, 16), generator=_rng(1))
    s = m.amino_acid_scores(x, None, res.cuda(), top=4)
    w = so.score(aa.cpu()[:, 1:].movedim(1, -1), res, 4)
    assert torch.equal(s.top_index.cpu().movedim(1, -1).long(), w["top_index"])
    assert float((s.logprob.cpu().double() - w["logprob"]).abs().max()) < 1e-5 and float((s.entropy.cpu().double() - w["entropy"]).abs().max()) < 1e-5
    e = m._engine((16, 16, 16))
    prof = torch.softmax(aa[0, 1:].reshape(20, -1)[:, :50], 0).t().cpu().numpy() * 0.3          # profiles are not normalised
    prof[3] = 0.0
    prof[3, 7] = 0.2
    r = clustering.residue_scores(e, prof, np.full(50, 7), top=2)
    norm = prof / prof.sum(1, keepdims=True)
    with np.errstate(divide="ignore"):
        want = np.log(norm[:, 7])
    assert np.abs(r.logprob.cpu().numpy() - want).max() < 1e-5 and float(r.entropy[3]) == 0.0 and r.top_index[3].tolist() == [7, 0]
    student = (torch.randn((1, 20, 16, 16, 16), generator=_rng(2))).cuda().requires_grad_()
    loss = scoring.distill_loss(e, student, s.top_index, s.top_logprob, dim=1, tail=True).mean()
    loss.backward()
    wl, wg, _ = so.distill(student.detach().cpu().movedim(1, -1), s.top_index.cpu().movedim(1, -1), s.top_logprob.cpu().movedim(1, -1), 1.0, True)
    assert abs(float(loss.detach()) - float(wl.mean())) < 1e-5
    assert float((student.grad.cpu().double() - wg.movedim(-1, 1) / 4096).abs().max()) < 1e-5 / 4096


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("classes", [7, 64, 300, 5000, 70001])
def test_rows_of_the_lowest_value_are_uniform_in_the_gradients_too(eng, dtype, classes):
    """a row masked with finfo.min throughout, or but for two classes: float32 log sums of it are the lowest value itself"""
    low = torch.finfo(DT[dtype]).min
    z = torch.full((3, classes), low).to(DT[dtype])
    z[1, ::2] = NEG
    z[2] = NEG
    z[2, [1, classes - 1]] = low
    tok = torch.tensor([1, 2, classes - 1])
    g = torch.tensor([1.0, -2.0, 0.5])
    for temperature in (1.0, 0.7, 0.9 if dtype == "f16" else 1.25):
        d = z.cuda()
        r = eng.token_logprobs(d, tok.cuda(), temperature=temperature)
        got = eng.token_logprobs_backward(d, tok.cuda(), r.lse, r.entropy, g.cuda(), g.cuda(), temperature=temperature)
        want = so.score_grad(z, tok, g, g, None, temperature)
        # f16: lse = -65504 + log C is rounded to a float32 of step 2^-8 (relative 2^-24), which the exponentials see in full
        rel = U * (64 + classes / 64) + (2.0 ** -8 if dtype == "f16" else 0.0)
        _near(got, want, rel * (want.abs() + 4.0 * g.abs()[:, None] / classes) * 4 + _half_step(dtype, want) + 1e-37)
        k = min(4, classes)
        idx = torch.arange(k).repeat(3, 1).int()
        val = torch.log(torch.tensor([0.4, 0.3, 0.1, 0.05])[:k]).repeat(3, 1)
        for tail in (False, True):
            if not tail:                                     # the list names classes the last two rows forbid: +inf there
                wl, wg, _ = so.distill(z[:1], idx[:1], val[:1], temperature, tail)
                zz, ii, vv, gg = d[:1], idx[:1].cuda(), val[:1].cuda(), g[:1]
            else:
                ii = torch.full_like(idx, -1)
                ii[0] = idx[0]
                ii[1, 0], ii[2, 0] = 1, classes - 1
                wl, wg, _ = so.distill(z, ii, val, temperature, tail)
                zz, ii, vv, gg = d, ii.cuda(), val.cuda(), g
            loss, aux = eng.distill_loss(zz, ii, vv, temperature=temperature, tail=tail)
            got = eng.distill_backward(zz, ii, vv, aux, gg.cuda(), temperature=temperature, tail=tail)
            want = wg * gg.double()[:, None]
            tol = U * (64 + classes / 64 + 8 * _log2c(classes)) * 4
            _near(loss, wl, tol * (1 + wl.abs()) * temperature ** 2)
            _near(got, want, tol * (want.abs() + 2.0 / classes) * temperature + _half_step(dtype, want) + 1e-37)
            sl, sg = eng.distill_step(zz, ii, vv, temperature=temperature, tail=tail, weight=gg.cuda())
            _near(sg, want, tol * (want.abs() + 2.0 / classes) * temperature + _half_step(dtype, want) + 1e-37)


def test_autograd_rules(eng):
    """written-to inputs and second derivatives are refused, not answered wrongly"""
    from mica_amd import scoring
    z = _logits((4, 300), 1, "f32").cuda()
    tok = torch.zeros(4, dtype=torch.int64, device="cuda")
    idx, val = _teacher(z.cpu(), 3, 2)
    for make in (lambda x: scoring.token_logprobs(eng, x, tok).logprob, lambda x: scoring.distill_loss(eng, x, idx.cuda(), val.cuda())):
        x = z.clone().requires_grad_()
        y = x * 1.0
        out = make(y).sum()
        with torch.no_grad():
            y.mul_(2.0)
        with pytest.raises(RuntimeError):
            out.backward()
        x = z.clone().requires_grad_()
        g, = torch.autograd.grad(make(x).sum(), x, create_graph=True)
        with pytest.raises(RuntimeError):
            g.sum().backward()
    r = scoring.token_logprobs(eng, z.clone().requires_grad_(), tok, top=2)
    assert not r.top_logprob.requires_grad and not r.top_index.requires_grad and r.lse.requires_grad


@pytest.mark.parametrize("rows,classes,dtype", [(260, 66003, "f32"), (257, 131080, "bf16")])
def test_many_rows_longer_than_one_block_takes(eng, rows, classes, dtype):
    """rows enough for a block each, but longer than its bits cover: still cut, and distill_step in two kernels"""
    z = _logits((rows, classes), 3, dtype)
    tok = torch.randint(0, classes, (rows,), generator=_rng(5))
    _check_score(eng, z, tok, 9)
    idx, val = _teacher(z, 12, 6)
    for tail in (False, True):
        _check_distill(eng, z, idx, val, dtype, 1.0, tail)


def test_c_entry_points_refuse_on_the_host(eng):
    """through the C ABI with a real context: refused with a message, nothing launched, the next call unharmed"""
    import ctypes as C
    from mica_amd import _cabi, scoring
    z = torch.randn((3, 40000), generator=_rng(1)).cuda()
    v = scoring.LogitsLayout(z, 1)
    f = torch.empty(3, device="cuda")
    tok = torch.zeros(3, dtype=torch.int64, device="cuda")
    need = eng.lib.mica_token_logprobs_ws(C.byref(v.desc), 0)
    ws = torch.empty(max(need, 16) + 16, dtype=torch.uint8, device="cuda")
    p = lambda t: t.data_ptr()
    assert need > 0
    ok = (eng._h, C.byref(v.desc), p(tok), 8, -100, 1.0, 0, p(f), p(f), p(f), None, None, p(ws), need, eng._raw_stream())
    bad = {1: None, 2: None, 3: 3, 5: 0.0, 6: 65, 7: None, 8: None, 9: None, 12: None, 13: need - 1}
    for at, value in bad.items():
        args = list(ok)
        args[at] = value
        assert eng.lib.mica_token_logprobs(*args) == _cabi.MICA_ERR_ARG, at
        assert b"mica_token_logprobs" in eng.lib.mica_last_error(eng._h)
    args = list(ok)
    args[12] += 8                                            # misaligned
    assert eng.lib.mica_token_logprobs(*args) == _cabi.MICA_ERR_ARG
    args = list(ok)
    args[6] = 3                                              # alternatives without a place to write them
    assert eng.lib.mica_token_logprobs(*args) == _cabi.MICA_ERR_ARG
    idx = torch.zeros((3, 2), dtype=torch.int32, device="cuda")
    val = torch.zeros((3, 2), device="cuda")
    for kw in (dict(k=0), dict(k=257), dict(index_bytes=2), dict(value_dtype=7), dict(d_index=None), dict(d_value=None)):
        d = dict(d_index=p(idx), d_value=p(val), index_bytes=4, value_dtype=0, k=2, tail=0)
        d.update(kw)
        lst = _cabi.MicaTopList(*[d[n] for n, _ in _cabi.MicaTopList._fields_])
        assert eng.lib.mica_distill_loss(eng._h, C.byref(v.desc), C.byref(lst), 1.0, p(f), None, p(ws), need, eng._raw_stream()) == _cabi.MICA_ERR_ARG
        assert b"mica_distill_loss" in eng.lib.mica_last_error(eng._h)
    lst = _cabi.MicaTopList(p(idx), p(val), 4, 0, 2, 0)
    assert eng.lib.mica_distill_backward(eng._h, C.byref(v.desc), C.byref(lst), 1.0, None, p(f), p(z), eng._raw_stream()) == _cabi.MICA_ERR_ARG
    assert eng.lib.mica_distill_step(eng._h, C.byref(v.desc), C.byref(lst), 1.0, None, p(f), None, p(ws), need, eng._raw_stream()) == _cabi.MICA_ERR_ARG
    assert eng.lib.mica_token_logprobs(*ok) == 0
    torch.cuda.synchronize()


def test_two_threads_share_an_engine(eng):
    """each on a stream of its own; the workspaces of their calls are their own as well"""
    import threading
    sets = []
    for seed in (1, 2):
        z = _logits((2, 60000), seed, "bf16")
        idx, val = _teacher(z, 5, seed)
        sets.append([t.cuda() for t in (z, torch.randint(0, 60000, (2,), generator=_rng(seed)), idx, val, torch.rand((2,), generator=_rng(2)))])
    want = [_all_outputs(eng, *s) for s in sets]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = _all_outputs(eng, *sets[i])
            torch.cuda.current_stream().synchronize()
            wrong.extend(not torch.equal(a, b) for a, b in zip(got, want[i]))
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(wrong) == 2 * len(want[0]) and not any(wrong)
