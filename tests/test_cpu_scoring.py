"""Class scoring and distillation without a GPU: the oracle's gradients against differences, the view of a logits tensor that is handed
to the library, the library's own argument checks, and what the engine refuses."""
import ctypes as C
import gc
import threading
import weakref

import pytest
import torch

from mica_amd import _cabi, scoring
from mica_amd._cabi import MicaHipError
from oracle import score_oracle as so


def _z(shape, seed, scale=2.0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64) * scale


def _differences(f, z, h=1e-5):
    """central differences of a scalar function, element by element"""
    g = torch.zeros_like(z)
    flat, gf = z.view(-1), g.view(-1)
    for i in range(flat.numel()):
        v = float(flat[i])
        flat[i] = v + h
        hi = float(f(z))
        flat[i] = v - h
        lo = float(f(z))
        flat[i] = v
        gf[i] = (hi - lo) / (2 * h)
    return g


@pytest.mark.parametrize("temperature", [1.0, 0.6])
def test_oracle_score_gradient_equals_differences(temperature):
    z = _z((3, 7), 1)
    tok = torch.tensor([2, -100, 6])
    gl, ge, gs = _z((3,), 2), _z((3,), 3), _z((3,), 4)

    def f(x):
        s = so.score(x, tok, temperature=temperature)
        return (gl * s["logprob"] + ge * s["entropy"] + gs * s["lse"]).sum()
    want = _differences(f, z)
    got = so.score_grad(z, tok, gl, ge, gs, temperature)
    # central differences: h^2 / 6 times a third derivative of O(10), and 1e-16 / h
    assert float((want - got).abs().max()) < 1e-8


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("temperature", [1.0, 1.7])
def test_oracle_distill_gradient_equals_differences(tail, temperature):
    z = _z((4, 9), 5)
    idx = torch.tensor([[0, 3, 8], [5, 5, 1], [2, -1, -1], [-1, -1, -1]])
    val = torch.log(torch.tensor([[.5, .2, .1], [.3, .2, .4], [.6, .1, .1], [.2, .2, .2]], dtype=torch.float64))
    want = _differences(lambda x: so.distill(x, idx, val, temperature, tail)[0].sum(), z)
    assert float((want - so.distill(z, idx, val, temperature, tail)[1]).abs().max()) < 1e-8


def test_oracle_distillation_of_the_whole_distribution_is_the_divergence():
    z, t = _z((5, 6), 6), torch.log_softmax(_z((5, 6), 7), -1)
    kl = (torch.exp(t) * (t - torch.log_softmax(z, -1))).sum(-1)
    idx = torch.arange(6).expand(5, 6)
    for tail in (False, True):
        assert float((so.distill(z, idx, t, 1.0, tail)[0] - kl).abs().max()) < 1e-12


LIB = None


def _lib():
    global LIB
    if LIB is None:
        LIB = _cabi.load_library()
    return LIB


@pytest.mark.parametrize("make,dim,want", [
    (lambda: torch.zeros(2, 9, 100)[:, :-1], -1, (1, 2, 8, 100, 900, 100, 1)),                      # shifted next-token logits
    (lambda: torch.zeros(2, 21, 4, 4, 4)[:, 1:], 1, (0, 2, 64, 20, 1344, 1, 64)),                   # a head without its first class
    (lambda: torch.zeros(2, 21, 4, 4, 4), 1, (0, 2, 64, 21, 1344, 1, 64)),
    (lambda: torch.zeros(7), 0, (1, 1, 1, 7, 0, 0, 1)),
    (lambda: torch.zeros(5, 3, 20), 2, (1, 1, 15, 20, 0, 20, 1)),
    (lambda: torch.zeros(20, 15).t(), 1, (1, 1, 15, 20, 0, 1, 15)),                                 # few classes: any stride
    (lambda: torch.zeros(1, 20).expand(6, 20), 1, (1, 1, 6, 20, 0, 0, 1)),                          # a broadcast row
    (lambda: torch.zeros(6, 20, 1, 1), 1, (1, 1, 6, 20, 0, 20, 1)),
    (lambda: torch.zeros(4, 0, 30), 2, None),
])
def test_layout_describes_the_tensor_in_place(make, dim, want):
    t = make()
    v = scoring.LogitsLayout(t, dim)
    assert not v.moved and (v.base.data_ptr() == t.data_ptr())
    if want is None:
        assert v.rows == 0
        return
    d = v.desc
    assert (d.class_last, d.outer, d.inner, d.classes, d.stride_outer, d.stride_inner, d.stride_class) == want
    assert d.outer * d.inner == v.rows
    # every element is where the description says
    base = torch.arange(t.storage_offset() + sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1)
    ref = base.as_strided(t.shape, t.stride(), t.storage_offset()).movedim(dim, -1).reshape(-1, d.classes)
    for r in range(0, v.rows, max(1, v.rows // 5)):
        o, i = divmod(r, d.inner)
        for c in (0, d.classes - 1):
            assert int(ref[r, c]) == t.storage_offset() + o * d.stride_outer + i * d.stride_inner + c * d.stride_class


@pytest.mark.parametrize("make,dim,moved", [
    (lambda: torch.zeros(3, 100, 7), 1, True),                     # many classes in the middle: copied with the classes last
    (lambda: torch.zeros(2, 3, 4, 100)[:, :2, :3], 3, False),      # three row axes that do not join: copied
    (lambda: torch.zeros(4, 200)[:, ::2], 1, False),               # many classes at a stride
    (lambda: torch.zeros(2, 21, 4, 4, 8)[..., :5], 1, False),
])
def test_layout_copies_what_has_no_view(make, dim, moved):
    t = make()
    v = scoring.LogitsLayout(t, dim)
    assert v.moved == moved and v.base.data_ptr() != t.data_ptr() and v.base.is_contiguous()
    k = torch.zeros(v.with_axis(3))
    assert tuple(v.give(k).shape) == t.shape[:v.dim] + (3,) + t.shape[v.dim + 1:]


@pytest.mark.parametrize("make,dim", [
    (lambda: torch.zeros(3, 4, dtype=torch.float64), 1), (lambda: torch.zeros(3, 4, dtype=torch.int32), 1), (lambda: torch.zeros(3, 0), 1),
    (lambda: torch.zeros(3, 4), 2), (lambda: torch.zeros(3, 4), -3), (lambda: torch.zeros(()), 0), (lambda: [1.0, 2.0], 0),
    (lambda: torch.zeros(1, 1).expand(1 << 31, 1), 1),
])
def test_layout_refusals(make, dim):
    with pytest.raises(MicaHipError):
        scoring.LogitsLayout(make(), dim)


def _desc(**kw):
    d = dict(d_data=4096, dtype=0, class_last=1, outer=1, inner=4, classes=1000, stride_outer=0, stride_inner=1000, stride_class=1)
    d.update(kw)
    return _cabi.MicaLogits(*[d[f] for f, _ in _cabi.MicaLogits._fields_])


@pytest.mark.parametrize("kw", [dict(dtype=3), dict(dtype=-1), dict(classes=0), dict(classes=(1 << 28) + 1), dict(inner=-1), dict(outer=1 << 16, inner=1 << 15),
                                dict(outer=1 << 40), dict(stride_inner=-1), dict(stride_class=2), dict(class_last=0), dict(d_data=0), dict(d_data=4098),
                                dict(dtype=1, d_data=4097)])
def test_library_refuses_a_bad_view(kw):
    lib = _lib()
    assert lib.mica_token_logprobs_ws(C.byref(_desc()), 0) >= 0 and lib.mica_distill_ws(C.byref(_desc()), 1) >= 0
    assert lib.mica_token_logprobs_ws(C.byref(_desc(**kw)), 0) == _cabi.MICA_ERR_ARG
    assert lib.mica_distill_ws(C.byref(_desc(**kw)), 0) == _cabi.MICA_ERR_ARG


def test_library_workspace_and_null_context():
    lib = _lib()
    assert lib.mica_token_logprobs_ws(None, 0) == _cabi.MICA_ERR_ARG
    for top in (-1, 65, 21):
        assert lib.mica_token_logprobs_ws(C.byref(_desc(classes=20)), top) == _cabi.MICA_ERR_ARG
    assert lib.mica_token_logprobs_ws(C.byref(_desc(classes=20, stride_class=7)), 20) == 0
    few = _desc(inner=1, classes=1 << 20, stride_inner=1 << 20)
    assert 0 < lib.mica_token_logprobs_ws(C.byref(few), 0) < lib.mica_token_logprobs_ws(C.byref(few), 64)
    assert 0 < lib.mica_distill_ws(C.byref(few), 0) < lib.mica_distill_ws(C.byref(few), 1)
    assert lib.mica_token_logprobs_ws(C.byref(_desc(inner=0)), 5) == 0
    # a null context: refused before anything is touched
    assert lib.mica_token_logprobs(None, C.byref(_desc()), None, 0, -100, 1.0, 0, None, None, None, None, None, None, 0, None) == _cabi.MICA_ERR_ARG
    assert lib.mica_token_logprobs_backward(None, C.byref(_desc()), None, 0, -100, 1.0, None, None, None, None, None, None, None) == _cabi.MICA_ERR_ARG
    lst = _cabi.MicaTopList(4096, 4096, 4, 0, 3, 0)
    assert lib.mica_distill_loss(None, C.byref(_desc()), C.byref(lst), 1.0, None, None, None, 0, None) == _cabi.MICA_ERR_ARG
    assert lib.mica_distill_backward(None, C.byref(_desc()), C.byref(lst), 1.0, None, None, None, None) == _cabi.MICA_ERR_ARG
    assert lib.mica_distill_step(None, C.byref(_desc()), C.byref(lst), 1.0, None, None, None, None, 0, None) == _cabi.MICA_ERR_ARG


class _NoLibrary:
    def __getattr__(self, name):
        raise AssertionError(f"{name} was called")


@pytest.fixture
def eng():
    """An engine without a context on the CPU: whatever is not refused in Python fails the test."""
    from mica_amd.engine import Engine
    e = Engine.__new__(Engine)
    e.device, e.lib, e._h, e.call_lock = torch.device("cpu"), _NoLibrary(), None, threading.RLock()
    return e


def test_engine_refuses_bad_arguments(eng):
    z, tok = torch.zeros(4, 30), torch.zeros(4, dtype=torch.int64)
    bad = [dict(top=31), dict(top=-1), dict(top=65), dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=float("nan")),
           dict(temperature=float("inf")), dict(temperature=1e-5), dict(dim=2), dict(tokens=tok.float()), dict(tokens=tok[:3]), dict(tokens=tok[None]),
           dict(tokens=tok.to(torch.int16)), dict(tokens=[1, 2, 3, 4]), dict(logits=z.double()), dict(logits=z.to("meta")), dict(logits=None)]
    for kw in bad:
        args = dict(logits=z, tokens=tok)
        args.update(kw)
        with pytest.raises(MicaHipError):
            eng.token_logprobs(**args)
    row = torch.zeros(4)
    for kw in (dict(lse=None), dict(lse=row[:2]), dict(entropy=row.double()), dict(g_logprob=row.half()), dict(g_entropy=row[None]), dict(tokens=None)):
        args = dict(logits=z, tokens=tok, lse=row, entropy=row, g_logprob=row)
        args.update(kw)
        with pytest.raises(MicaHipError):
            eng.token_logprobs_backward(**args)


def test_engine_refuses_bad_teacher_lists(eng):
    z, idx, val = torch.zeros(4, 300), torch.zeros(4, 3, dtype=torch.int32), torch.zeros(4, 3)
    bad = [dict(teacher_index=idx.float()), dict(teacher_index=idx[:3]), dict(teacher_index=idx[0]), dict(teacher_logprob=val[:, :2]),
           dict(teacher_logprob=val.double()), dict(teacher_logprob=None), dict(teacher_index=None), dict(temperature=0.0), dict(dim=0),
           dict(teacher_index=torch.zeros(4, 0, dtype=torch.int32), teacher_logprob=torch.zeros(4, 0)),
           dict(teacher_index=torch.zeros(4, 257, dtype=torch.int32), teacher_logprob=torch.zeros(4, 257))]
    for kw in bad:
        args = dict(student=z, teacher_index=idx, teacher_logprob=val)
        args.update(kw)
        with pytest.raises(MicaHipError):
            eng.distill_loss(**args)
        with pytest.raises(MicaHipError):
            eng.distill_step(**args)
    with pytest.raises(MicaHipError):
        eng.distill_step(z, idx, val, weight=torch.zeros(4, dtype=torch.float16))
    with pytest.raises(MicaHipError):
        eng.distill_step(z, idx, val, weight=torch.zeros(1))
    aux = torch.zeros(4, 4)
    for kw in (dict(aux=aux[:3]), dict(aux=None), dict(g_loss=torch.zeros(3)), dict(g_loss=None)):
        args = dict(student=z, teacher_index=idx, teacher_logprob=val, aux=aux, g_loss=torch.zeros(4))
        args.update(kw)
        with pytest.raises(MicaHipError):
            eng.distill_backward(**args)


def test_engine_answers_an_empty_tensor_without_a_call(eng):
    s = eng.token_logprobs(torch.zeros(0, 5, 30), torch.zeros(0, 5, dtype=torch.int32), top=3)
    assert s.logprob.shape == (0, 5) and s.top_index.shape == (0, 5, 3) and s.top_index.dtype == torch.int32
    loss, aux = eng.distill_loss(torch.zeros(0, 300), torch.zeros(0, 3, dtype=torch.int32), torch.zeros(0, 3))
    assert loss.shape == (0,) and aux.shape == (4, 0)
    assert eng.distill_step(torch.zeros(0, 300), torch.zeros(0, 3, dtype=torch.int32), torch.zeros(0, 3))[1].shape == (0, 300)


def test_the_gradients_maxima_and_sums_are_checked(eng):
    """aux: one maximum and one sum per row of more than 64 classes, nothing for fewer"""
    z, tok, row = torch.zeros(4, 100), torch.zeros(4, dtype=torch.int64), torch.zeros(4)
    assert eng.logits_view(z, -1).score_aux().shape == (2, 4) and eng.logits_view(z[:, :64], -1).score_aux() is None
    for aux in (torch.zeros(4), torch.zeros(4, 2), torch.zeros(2, 4, dtype=torch.float64), torch.zeros(4, 2).t(), torch.zeros(2, 4, device="meta"), 1.0):
        with pytest.raises(MicaHipError):
            eng.token_logprobs(z, tok, aux=aux)
        with pytest.raises(MicaHipError):
            eng.token_logprobs_backward(z, tok, row, row, g_logprob=row, aux=aux)
    with pytest.raises(MicaHipError):
        eng.token_logprobs(z[:, :64], tok, aux=torch.zeros(2, 4))
    lib = _lib()
    assert lib.mica_token_logprobs_aux(None, C.byref(_desc()), None, 0, -100, 1.0, 0, None, None, None, None, None, None, None, 0, None) == _cabi.MICA_ERR_ARG


class _TorchEngine:
    """the engine's calls of the autograd functions, on the CPU: gradients read through the view that is handed to the library"""
    device = torch.device("cpu")

    def __init__(self):
        self.bases, self.call_lock = [], threading.RLock()

    def logits_view(self, logits, dim, name="logits"):
        v = scoring.LogitsLayout(logits, dim)
        self.bases.append(weakref.ref(v.base))
        return v

    def _rows(self, view):
        """the logits at the description's address alone: [outer, inner, classes]"""
        d = view.desc
        n = 1 + (d.outer - 1) * d.stride_outer + (d.inner - 1) * d.stride_inner + (d.classes - 1) * d.stride_class
        flat = torch.frombuffer((C.c_float * n).from_address(d.d_data), dtype=torch.float32)
        return flat.as_strided((d.outer, d.inner, d.classes), (d.stride_outer, d.stride_inner, d.stride_class)).double()

    def _give(self, g, view):
        return view.give((g if view.class_last else g.transpose(1, 2)).reshape(view.with_axis(view.classes)).to(view.dtype))

    def _scores(self, view, tokens, top, temperature, ignore_index, aux):
        lse = torch.logsumexp(self._rows(view), -1).reshape(view.rows_shape).float()
        return scoring.TokenScores(None if tokens is None else lse * 0, lse * 0, lse, None, None)

    def _score_gradient(self, view, tokens, aux, entropy, g_logprob, g_entropy, g_lse, temperature, ignore_index):
        z = self._rows(view)
        return self._give(torch.softmax(z, -1) * g_lse.reshape(z.shape[:2])[..., None], view)

    def distill_loss(self, student, index, logprob, dim, temperature, tail, view):
        lse = torch.logsumexp(self._rows(view), -1).reshape(view.rows_shape).float()
        return lse, torch.zeros(4, view.rows)

    def distill_backward(self, student, index, logprob, aux, g_loss, dim, temperature, tail, view):
        z = self._rows(view)
        return self._give(torch.softmax(z, -1) * g_loss.reshape(z.shape[:2])[..., None], view)


AUTOGRAD_LAYOUTS = [(lambda x: x, (6, 100), 1), (lambda x: x[:, 1:], (2, 21, 3, 4), 1), (lambda x: x, (3, 100, 5), 1), (lambda x: x[:, :-1], (3, 6, 90), 2),
                    (lambda x: x[..., ::2], (4, 200), 1)]


def _scoring_calls(engine, dim):
    idx, val = torch.zeros(1, dtype=torch.int64), torch.zeros(1)
    return (lambda y: scoring.token_logprobs(engine, y, None, dim=dim).lse, lambda y: scoring.distill_loss(engine, y, idx, val, dim=dim))


@pytest.mark.parametrize("cut,shape,dim", AUTOGRAD_LAYOUTS)
def test_logits_are_freed_with_the_backward_pass(cut, shape, dim):
    """a loss that the caller keeps keeps neither the logits nor a copy of them"""
    for which in (0, 1):
        engine = _TorchEngine()
        x = torch.randn(shape, generator=torch.Generator().manual_seed(1)).requires_grad_()
        y = cut(x * 1.0)
        ref = weakref.ref(y)
        loss = _scoring_calls(engine, dim)[which](y).sum()
        del y
        loss.backward()
        gc.collect()
        assert loss.grad_fn is not None and ref() is None and engine.bases[0]() is None
        want, = torch.autograd.grad(torch.logsumexp(cut(x * 1.0), dim).sum(), x)
        assert float((x.grad - want).abs().max()) < 1e-6


@pytest.mark.parametrize("cut,shape,dim", AUTOGRAD_LAYOUTS)
def test_the_backward_pass_reads_what_saved_tensor_hooks_give_back(cut, shape, dim):
    """packed elsewhere and given back at another address, with other strides"""
    for which in (0, 1):
        x = torch.randn(shape, generator=torch.Generator().manual_seed(2)).requires_grad_()
        given = []

        def unpack(t):
            given.append(t.clone(memory_format=torch.contiguous_format))
            return given[-1]
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().clone(memory_format=torch.contiguous_format), unpack):
            y = cut(x * 1.0)
            loss = _scoring_calls(_TorchEngine(), dim)[which](y).sum()
        with torch.no_grad():
            y.zero_()                                       # what was packed is what counts
        loss.backward()
        want, = torch.autograd.grad(torch.logsumexp(cut(x * 1.0), dim).sum(), x)
        assert given and float((x.grad - want).abs().max()) < 1e-6
