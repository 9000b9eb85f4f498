"""Class scoring and distillation of rows of any magnitude, on the GPU against float64 (oracle/score_oracle.py): rows masked with ordinary
large values (-1e4 ... -1e30), forced tokens, large common offsets, rows that hold NaN.

Softmax does not know a common offset, so the bounds here know none either: everything is relative to distances from the row's maximum m.
u = 2^-24 (half a step of float32, relative).  z - m, the rounding of T to float32, of 1 / T (or log2 e / T) and the product cost 4 u of
the distance |y - m|: 6 u is allowed.  A sum of C exponentials adds at most ~C / 64 terms one after the other per thread, each off by a few
u (the hardware's 2^x: 2 u): `terms` = 16 + C / 64 + 4 log2 C in units of u.  The log-sum-exp itself is of the row's magnitude: 4 u of it.
Results of fewer bits add half a step of their type."""
import math

import pytest
import torch

from oracle import score_oracle as so

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
NEG = float("-inf")
NAN = float("nan")


@pytest.fixture(scope="module")
def eng():
    from mica_amd.engine import Engine
    e = Engine(0, max_batch=1, tile_size=4)
    yield e
    e.close()


def _rng(seed):
    return torch.Generator().manual_seed(seed)


def _log2c(c):
    return math.log2(c) + 4.0


def _terms(c):
    return 16 + c / 64 + 4 * _log2c(c)


def _herr(c):
    """of the entropy: the same terms weighted once more with |log p|"""
    return U * (32 + c / 32 + 6 * _log2c(c) ** 2)


def _finite(t):
    return torch.nan_to_num(t, nan=0.0, posinf=0.0, neginf=0.0)


def _near(got, want, tol, what=""):
    """got against want, infinities and NaN at the same places; tol per element"""
    got = got.detach().cpu().double()
    want = want.double()
    assert got.shape == want.shape
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    inf = torch.isinf(want)
    assert torch.equal(torch.isinf(got), inf) and torch.equal(got[inf], want[inf]), what
    ok = ~(inf | torch.isnan(want))
    tol = torch.as_tensor(tol, dtype=torch.float64).expand(want.shape)
    over = ((got - want).abs() / tol)[ok]
    worst = float(over.max()) if bool(ok.any()) else 0.0
    assert worst <= 1.0, f"{what}: {worst} times the bound"


def _half_step(dtype, want):
    t = DT[dtype]
    if t == torch.float32:
        return U * want.abs() + 1e-37
    return torch.finfo(t).eps / 2 * want.abs() + (torch.finfo(t).smallest_normal * torch.finfo(t).eps)


def _values(dtype):
    if dtype == "f16":
        return [-1e4, -65504.0]
    return [-1e4, -65504.0, -1e6, -1e7, -1e9, -1e10, -1e12, -1e20, -1e30]


def _rows(classes, value, dtype, seed):
    """rows that hold `value` in different places, and one that does not"""
    g = _rng(seed)
    z = torch.randn((8, classes), generator=g) * 3.0
    half = classes // 2
    z[0] = value
    z[1, :half] = value                                      # whole threads see nothing but the value first
    keep = z[2, classes - 1].clone()
    z[2] = value
    z[2, classes - 1] = keep
    z[3, torch.rand((classes,), generator=g) < 0.6] = value
    z[4, half] = -value                                      # a forced class
    z[5] = -value
    z[6, :half] = value
    z[6, half:] = value * (1.0 - 2.0 ** -7)
    return z.to(DT[dtype])


def _tokens(classes):
    return torch.tensor([classes - 1, 0, classes - 1, classes // 3, classes // 2, 1, classes - 1, -100])


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("classes", [21, 65, 300, 5000, 70001])
@pytest.mark.parametrize("temperature", [0.1, 0.7, 1.0, 2.0])
def test_scores_of_rows_of_any_magnitude(eng, dtype, classes, temperature):
    tok = _tokens(classes)
    for value in _values(dtype):
        z = _rows(classes, value, dtype, classes)
        r = eng.token_logprobs(z.cuda(), tok.cuda(), top=5, temperature=temperature)
        w = so.score(z, tok, 5, temperature)
        what = f"value {value}"
        _near(r.lse, w["lse"], U * (_terms(classes) + 4 * w["lse"].abs()), what)
        _near(r.logprob, w["logprob"], U * (_terms(classes) + 6 * w["logprob"].abs()), what)
        _near(r.entropy, w["entropy"], _herr(classes), what)
        assert torch.equal(r.top_index.cpu().long(), w["top_index"]), what
        _near(r.top_logprob, w["top_logprob"], U * (_terms(classes) + 6 * w["top_logprob"].abs()), what)


def _check_distill(eng, z, idx, val, dtype, temperature, tail, weight, what=""):
    """loss, gradient and the one-call step, bounds by distances alone"""
    want, wgrad, p = so.distill(z, idx, val, temperature, tail)
    C = z.shape[-1]
    y = z.double() / temperature
    logq = so.log_softmax(y)[0]
    listed = torch.zeros(y.shape[:-1] + (C + 1,), dtype=torch.bool).scatter_(-1, torch.where(idx < 0, C, idx).long(), True)[..., :C]
    free = torch.where(listed, torch.full_like(y, NEG), y)
    mrest = free.amax(-1, keepdim=True)
    # of listed classes to the row's maximum, of the others to theirs; what has no probability has no error
    dist = torch.where(listed, (y - y.amax(-1, keepdim=True)).abs(), (y - torch.where(torch.isinf(mrest), torch.zeros_like(mrest), mrest)).abs())
    shown = torch.where(torch.exp(-dist) > 0, dist, torch.zeros_like(dist))
    lqr = torch.logsumexp(torch.where(listed, torch.full_like(y, NEG), logq), -1)
    lq = torch.maximum(_finite(p["lq"]).abs().amax(-1), torch.where(p["rest"] > 0, _finite(lqr).abs(), torch.zeros_like(lqr)))
    t = torch.where(idx < 0, torch.full_like(val, NEG), val).double()
    tmax = torch.zeros_like(t[..., :1]) if tail else t.amax(-1, keepdim=True)
    lt = _finite(t - tmax).abs().amax(-1, keepdim=True)
    mass = p["mass"][..., 0].clamp(min=1.0)
    loss_tol = temperature ** 2 * U * (_terms(C) + 6 * lq + 4 * lt[..., 0]) * mass + 2 * U * _finite(want).abs() + 1e-37
    d = [x.cuda() for x in (z, idx, val)]
    loss, aux = eng.distill_loss(*d, temperature=temperature, tail=tail)
    _near(loss, want, loss_tol, what)
    w = weight.double()[..., None]
    both = p["q"] * p["mass"] + p["share"] * p["rest"][..., None]
    tol = temperature * w.abs() * U * ((16 + 6 * shown + _terms(C)) * both + (16 + 6 * lt) * p["target"]) + _half_step(dtype, wgrad * w) + 1e-37
    got = eng.distill_backward(*d, aux, weight.cuda(), temperature=temperature, tail=tail)
    _near(got, wgrad * w, tol, what)
    sl, sg = eng.distill_step(*d, temperature=temperature, tail=tail, weight=weight.cuda())
    _near(sl, want * weight.double(), loss_tol * weight.double().abs() + 2 * U * _finite(want).abs() * weight.double().abs(), what)
    _near(sg, wgrad * w, tol, what)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("classes", [21, 65, 300, 5000, 70001])
@pytest.mark.parametrize("tail", [False, True])
def test_distillation_of_rows_of_any_magnitude(eng, dtype, classes, tail):
    g = _rng(classes)
    idx = torch.stack([torch.randperm(classes, generator=g)[:6] for _ in range(8)]).int()
    idx[:, 5] = -1
    idx[2, 0] = classes - 1
    idx[4, 0] = classes // 2
    for r in range(8):                                       # distinct again
        seen = set()
        for k in range(5):
            while int(idx[r, k]) in seen:
                idx[r, k] = (int(idx[r, k]) + 1) % classes
            seen.add(int(idx[r, k]))
    val = torch.log(torch.tensor([0.4, 0.3, 0.1, 0.05, 0.02, 0.9])).repeat(8, 1)
    weight = torch.rand((8,), generator=g) + 0.5
    for value in _values(dtype):
        z = _rows(classes, value, dtype, classes)
        for temperature in (0.1, 1.0, 2.0):
            _check_distill(eng, z, idx, val, dtype, temperature, tail, weight, f"value {value}, T {temperature}")


def test_a_call_of_few_rows_and_many_agree_on_masked_rows(eng):
    """cut into segments (each with a maximum of its own, some of masked classes only) or whole"""
    classes = 40000
    for value in (-1e9, -1e10, -1e20):
        z = torch.full((300, classes), value)
        z[:, 30000:30100] = torch.randn((300, 100), generator=_rng(1))
        z[1] = value
        a = eng.token_logprobs(z[:4].cuda(), torch.arange(4).cuda() + 30000, top=9)
        b = eng.token_logprobs(z.cuda(), torch.arange(300).cuda() % 100 + 30000, top=9)
        assert torch.equal(a.top_index, b.top_index[:4])
        for x, y in zip(a, b):
            assert float((x - y[:4]).abs().nan_to_num().max()) <= U * 2 * _terms(classes) + 4 * U * float(y[:4].abs().max()) and bool(torch.isfinite(x).all())
        w = so.score(z[:4], torch.arange(4) + 30000, 9)
        _near(a.logprob, w["logprob"], U * (_terms(classes) + 6 * w["logprob"].abs()))


# ---- gradients of the scores -----------------------------------------------------------------------------------------------------------------

def _grad_tol(z, dtype, want, gl, ge, gs, temperature):
    """p is off by 6 u of its distance and `terms` u of the sum, log p likewise, the entropy by its own bound; the token's 1 - p rounds twice.
    The hardware's 2^d is 0 below 2^-126, where p S < 2^-126: at most 2^-126 times what p is multiplied with is missing there."""
    C = z.shape[-1]
    w = so.score(z, temperature=temperature)
    p = torch.exp(w["logp"])
    y = z.double() / temperature
    dist = torch.where(p > 0, (y - y.amax(-1, keepdim=True)).abs(), torch.zeros_like(y))
    logp = torch.where(p > 0, w["logp"].abs(), torch.zeros_like(p))
    a = (gl.double().abs() + gs.double().abs())[..., None]
    e = ge.double().abs()[..., None]
    H = w["entropy"][..., None]
    own = U * (6 * dist + _terms(C))
    tol = p * (own * (a + e * (logp + H)) + e * (_herr(C) + own + 4 * U * (logp + H))) / temperature
    tol = tol + 2.0 ** -126 * (a + e * (logp + H)) / temperature
    return tol + 4 * U * gl.double().abs()[..., None] / temperature * (want.abs() > 0) + _half_step(dtype, want) + 1e-37


def _check_grad(eng, z, tok, dtype, gl, ge, gs, temperature, what=""):
    """through autograd, and the engine's call on the forward results alone"""
    from mica_amd import scoring
    used = torch.where(tok == -100, torch.zeros_like(gl), gl)
    want = so.score_grad(z, tok, gl, ge, gs, temperature)
    tol = _grad_tol(z, dtype, want, used, ge, gs, temperature)
    x = z.cuda().requires_grad_()
    r = scoring.token_logprobs(eng, x, tok.cuda(), temperature=temperature)
    got, = torch.autograd.grad([r.logprob, r.entropy, r.lse], [x], [gl.cuda(), ge.cuda(), gs.cuda()])
    _near(got, want, tol, what)
    alone = eng.token_logprobs_backward(z.cuda(), tok.cuda(), r.lse.detach(), r.entropy.detach(), gl.cuda(), ge.cuda(), gs.cuda(), temperature=temperature)
    _near(alone, want, tol, what)
    return got


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("classes", [7, 21, 65, 300, 5000, 70001])
def test_score_gradients_of_rows_of_any_magnitude(eng, dtype, classes):
    tok = _tokens(classes)
    g = _rng(classes)
    gl, ge, gs = (torch.randn((8,), generator=g) for _ in range(3))
    for value in _values(dtype):
        z = _rows(classes, value, dtype, classes)
        for temperature in (0.1, 1.0, 2.0):
            _check_grad(eng, z, tok, dtype, gl, ge, gs, temperature, f"value {value}, T {temperature}")


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("classes", [21, 300, 70001])
def test_score_gradients_of_rows_of_the_lowest_value_and_small_temperatures(eng, dtype, classes):
    low = torch.finfo(DT[dtype]).min
    z = torch.full((4, classes), low).to(DT[dtype])
    z[1, ::2] = NEG
    z[2] = NEG
    z[2, [1, classes - 1]] = low
    z[3] = 30.0
    z[3, 2] = 30.0625 if dtype == "f32" else 30.125
    tok = torch.tensor([1, 2, classes - 1, 2])
    g = torch.tensor([1.0, -2.0, 0.5, 1.5])
    for temperature in (1e-3, 0.7, 0.8, 1.25):
        _check_grad(eng, z, tok, dtype, g, g * 0.5, g * 0.25, temperature, f"T {temperature}")


@pytest.mark.parametrize("dtype,offset", [("f32", 2.0 ** 20), ("bf16", 128.0), ("f16", 1024.0)])
@pytest.mark.parametrize("classes", [21, 300, 5000])
def test_a_common_offset_changes_nothing(eng, dtype, offset, classes):
    """z and z + offset, both exact in the type"""
    from mica_amd import scoring
    g = _rng(classes)
    z = torch.randint(-4, 5, (6, classes), generator=g).float()
    assert torch.equal((z + offset).to(DT[dtype]).float(), z + offset) and torch.equal((z - offset).to(DT[dtype]).float(), z - offset)
    tok = torch.randint(0, classes, (6,), generator=g)
    gl, ge = torch.randn((6,), generator=g), torch.randn((6,), generator=g)
    zero = torch.zeros(6)
    outs = []
    for o in (0.0, offset, -offset):
        x = (z + o).to(DT[dtype]).cuda().requires_grad_()
        r = scoring.token_logprobs(eng, x, tok.cuda())
        grad, = torch.autograd.grad([r.logprob, r.entropy], [x], [gl.cuda(), ge.cuda()])
        outs.append((r.logprob.detach().cpu().double(), r.entropy.detach().cpu().double(), grad.cpu().double()))
    want = so.score_grad(z, tok, gl, ge, None)
    tol = _grad_tol(z, dtype, want, gl, ge, zero, 1.0)
    for lp, ent, grad in outs[1:]:
        _near(lp, outs[0][0], 2 * U * (_terms(classes) + 6 * outs[0][0].abs()))
        _near(ent, outs[0][1], 2 * _herr(classes))
        _near(grad, outs[0][2], 2 * tol)


def test_c_entry_points_want_the_maxima_and_sums(eng):
    """refused on the host, with a message; without a workspace rows are whole and a row's results do not depend on how many there are"""
    import ctypes as C
    from mica_amd import _cabi, scoring
    z = torch.randn((300, 40000), generator=_rng(1)).cuda()
    f = torch.empty((6, 300), device="cuda")

    def call(v, rows, entropy, lse, aux):
        return eng.lib.mica_token_logprobs_aux(eng._h, C.byref(v.desc), None, 0, -100, 1.0, 0, None, entropy.data_ptr(), lse.data_ptr(),
                                               None if aux is None else aux.data_ptr(), None, None, None, 0, eng._raw_stream())
    many, few = scoring.LogitsLayout(z, 1), scoring.LogitsLayout(z[:2], 1)
    assert call(few, 2, f[0], f[1], None) == _cabi.MICA_ERR_ARG and b"mica_token_logprobs_aux" in eng.lib.mica_last_error(eng._h)
    a, b = torch.zeros((2, 300), device="cuda"), torch.zeros((2, 2), device="cuda")
    assert call(many, 300, f[0], f[1], a) == 0 and call(few, 2, f[2], f[3], b) == 0
    assert torch.equal(a[:, :2], b) and torch.equal(f[0, :2], f[2, :2]) and torch.equal(a[0], z.amax(1))
    assert eng.lib.mica_token_logprobs_backward(eng._h, C.byref(few.desc), None, 0, -100, 1.0, None, f[0].data_ptr(), None, f[0].data_ptr(), None,
                                                z.data_ptr(), eng._raw_stream()) == _cabi.MICA_ERR_ARG
    assert b"mica_token_logprobs_backward" in eng.lib.mica_last_error(eng._h)


@pytest.mark.parametrize("classes", [21, 300])
def test_a_large_entropy_gradient_beside_masked_classes(eng, classes):
    """an entropy gradient scaled by 2^16 at T = 1e-4: finite at classes of probability 0 (the product with their log p is 0)"""
    z = torch.randn((3, classes), generator=_rng(classes)) * 1e-4
    z[0, ::2] = NEG
    z[1, ::2] = torch.finfo(torch.float32).min
    z[2, 1:] = NEG
    tok = torch.full((3,), -100)
    zero, ge = torch.zeros(3), torch.tensor([65536.0, -65536.0, 65536.0])
    _check_grad(eng, z, tok, "f32", zero, ge, zero, 1e-4)


# ---- teachers' lists ---------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("classes", [21, 65, 300, 5000, 70001])
@pytest.mark.parametrize("offset", [0.0, 1e4, 1e6, 1e8, -1e8, -1e30])
def test_a_constant_per_list_cancels(eng, classes, offset):
    """values of any common magnitude: what is left of their distances after the addition counts, in the loss and in both gradients"""
    g = _rng(classes)
    z = torch.randn((5, classes), generator=g) * 3.0
    idx = torch.stack([torch.randperm(classes, generator=g)[:5] for _ in range(5)]).int()
    idx[1, 4] = -1
    idx[2, 3] = idx[2, 0]
    val = torch.tensor([0.0, -1.0, -2.0, -3.0, -0.5]).repeat(5, 1) + offset
    val[3, 1] = NEG
    val[4, 1:] = NEG
    weight = torch.rand((5,), generator=g) + 0.5
    for temperature in (1.0, 1.7):
        _check_distill(eng, z, idx, val, "f32", temperature, False, weight, f"T {temperature}")


@pytest.mark.parametrize("classes", [20, 64, 65, 300, 5000, 70001])
@pytest.mark.parametrize("tail", [False, True])
def test_what_makes_the_loss_nan_makes_the_whole_gradient_nan(eng, classes, tail):
    """whatever the size and the entry point; and an empty row with a sound list keeps its loss of +inf and its gradient of 0"""
    g = _rng(classes)
    z = torch.randn((8, classes), generator=g)
    idx = torch.stack([torch.randperm(classes, generator=g)[:4] for _ in range(8)]).int()
    val = torch.log(torch.tensor([0.4, 0.3, 0.1, 0.05])).repeat(8, 1)
    z[0] = NAN
    z[1] = NEG
    idx[1, 2] = classes                                       # no class
    z[2] = NEG
    val[2, 1] = NAN
    val[3, 3] = NAN
    z[4, int(idx[4, 0])] = NAN
    val[4, 0] = NEG                                           # at a class that the list gives no probability
    idx[5, 0] = classes + 5
    z[6] = NEG
    nan = [0, 1, 2, 3, 4, 5]
    d = [t.cuda() for t in (z, idx, val)]
    ones = torch.ones(8, device="cuda")
    loss, aux = eng.distill_loss(*d, tail=tail)
    back = eng.distill_backward(*d, aux, ones, tail=tail)
    sl, sg = eng.distill_step(*d, tail=tail)
    for lo, gr in ((loss, back), (sl, sg)):
        assert torch.isnan(lo).nonzero()[:, 0].tolist() == nan
        assert bool(torch.isnan(gr[nan]).all()) and not bool(torch.isnan(gr[6:]).any())
        assert math.isinf(float(lo[6])) and float(lo[6]) > 0 and float(gr[6].abs().max()) == 0.0
    want, wgrad, _ = so.distill(z[7:], idx[7:], val[7:], 1.0, tail)
    assert float((loss[7:].cpu() - want).abs()) < U * 2 * _terms(classes) and float((back[7:].cpu() - wgrad).abs().max()) < U * 2 * _terms(classes)


@pytest.mark.parametrize("classes", [20, 64, 65, 300, 5000])
@pytest.mark.parametrize("tail", [False, True])
def test_a_masked_loss_has_gradient_zero_whatever_the_row_holds(eng, classes, tail):
    """through the loss's upstream gradient and through the step's weight, at both sides of 64 classes"""
    from mica_amd import scoring
    z = torch.randn((4, classes), generator=_rng(classes))
    idx = torch.arange(3).repeat(4, 1).int()
    val = torch.log(torch.tensor([0.4, 0.3, 0.1])).repeat(4, 1)
    z[0] = NAN
    idx[1, 0] = classes
    val[2, 0] = NAN
    mask = torch.tensor([0.0, 0.0, 0.0, 1.0]).cuda()
    x = z.cuda().requires_grad_()
    loss = scoring.distill_loss(eng, x, idx.cuda(), val.cuda(), tail=tail)
    torch.where(mask > 0, loss, torch.zeros_like(loss)).sum().backward()
    _, sg = eng.distill_step(z.cuda(), idx.cuda(), val.cuda(), tail=tail, weight=mask)
    for grad in (x.grad, sg):
        assert float(grad[:3].abs().max()) == 0.0 and bool(torch.isfinite(grad[3]).all()) and float(grad[3].abs().max()) > 0.0


# ---- what autograd keeps ------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("shape,dim,cut", [((3, 9, 501), 2, lambda x: x[:, :-1]), ((2, 21, 4, 4, 4), 1, lambda x: x[:, 1:]), ((3, 400, 5), 1, lambda x: x)])
def test_saved_logits_may_be_kept_on_the_host_and_are_freed(eng, shape, dim, cut):
    from mica_amd import scoring
    x = torch.randn(shape, generator=_rng(3)).cuda()
    z = cut(x)
    tok = torch.zeros(z.shape[:dim] + z.shape[dim + 1:], dtype=torch.int64, device="cuda")
    lists = z.shape[:dim] + (2,) + z.shape[dim + 1:]
    idx = torch.arange(2, device="cuda").view([2 if a == dim else 1 for a in range(len(lists))]).expand(lists).int()
    val = torch.full(lists, math.log(0.4), device="cuda")

    def grads(ctx):
        leaf = x.clone().requires_grad_()
        with ctx():
            a = scoring.token_logprobs(eng, cut(leaf * 1.0), tok, dim=dim)
            loss = (a.logprob + a.entropy).sum() + scoring.distill_loss(eng, cut(leaf * 1.0), idx, val, dim=dim, tail=True).sum()
        loss.backward()
        return loss, leaf.grad
    import contextlib
    _, want = grads(contextlib.nullcontext)
    _, got = grads(lambda: torch.autograd.graph.save_on_cpu(pin_memory=False))
    assert torch.equal(got, want)
    # a loss that is kept after its backward pass keeps no logits
    big = torch.randn((512, 16384), device="cuda").requires_grad_()
    before = torch.cuda.memory_allocated()
    kept = scoring.token_logprobs(eng, big * 1.0, torch.zeros(512, dtype=torch.int64, device="cuda")).logprob.sum()
    kept.backward()
    big.grad = None
    assert kept.grad_fn is not None and torch.cuda.memory_allocated() - before < 1 << 20
