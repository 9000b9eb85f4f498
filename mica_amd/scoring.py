"""Scoring of class distributions and distillation from a teacher's top alternatives.

The network answers with a distribution over classes at every voxel (the amino-acid head: 21 logits, class 0 the background), and a caller
that traces a chain through it asks three things the softmax volume alone does not answer cheaply: how probable GIVEN residues are, how
sure the network is, and what the runners-up are.  A smaller network is then trained on exactly these runners-up.

    s = engine.token_logprobs(logits, residues, top=3, dim=1)        # s.logprob, s.entropy, s.lse, s.top_logprob, s.top_index
    loss = scoring.distill_loss(engine, student, s.top_index, s.top_logprob, dim=1, tail=True)      # per row, in an autograd graph
    loss, grad = engine.distill_step(student, s.top_index, s.top_logprob, dim=1, weight=w)          # without one

`token_logprobs` and `distill_loss` of this module are the differentiable forms of the engine's calls; the class axis may be any axis of
float32, bfloat16 or float16 logits: the last one of a language model's [B, S, C], axis 1 of a head's NCDHW logits, or a slice of either."""
from __future__ import annotations

import math
import typing

import torch

from . import _cabi
from ._cabi import MicaHipError

COL_MAX = 64                # up to so many classes are read at any stride (kernels_score.hip)
MAX_TOP = 64                # alternatives per row
MAX_LIST = 256              # entries of a teacher's list
INTS = (torch.int32, torch.int64)
DTYPES = {torch.float32: _cabi.MICA_F32, torch.bfloat16: _cabi.MICA_BF16, torch.float16: _cabi.MICA_F16}


class TokenScores(typing.NamedTuple):
    """logprob (None without tokens), entropy, lse: float32, the logits' shape without the class axis; top_logprob float32 and top_index
    int32 (None if top = 0): the logits' shape with K at the class axis."""
    logprob: torch.Tensor | None
    entropy: torch.Tensor
    lse: torch.Tensor
    top_logprob: torch.Tensor | None
    top_index: torch.Tensor | None


def _collapse(sizes, strides):
    """Adjacent axes that one stride describes become one: -> [(size, stride)] without axes of size 1."""
    out = []
    for n, s in zip(sizes, strides):
        if n == 1:
            continue
        if out and out[-1][1] == s * n:
            out[-1] = (out[-1][0] * n, s)
        else:
            out.append((n, s))
    return out


class LogitsLayout:
    """How a logits tensor is handed to the library: the view (`desc`), the tensor it points into (`base`: the logits themselves, or a
    copy where no view fits), and the shapes of what comes back.  `moved`: the copy has the class axis last, results are laid out like
    it and returned as views with the axis where the caller has it."""
    __slots__ = ("dim", "shape", "classes", "rows_shape", "rows", "base", "moved", "class_last", "desc", "dtype", "strides", "device")

    def __init__(self, logits: torch.Tensor, dim: int):
        dtype = DTYPES.get(logits.dtype) if isinstance(logits, torch.Tensor) else None
        if dtype is None:
            raise MicaHipError(f"logits: expected a float32, bfloat16 or float16 tensor, got {getattr(logits, 'dtype', type(logits))}")
        shape = tuple(logits.shape)
        if not shape or not -len(shape) <= dim < len(shape):
            raise MicaHipError(f"dim {dim} is no axis of logits of shape {shape}")
        self.dim = dim = dim % len(shape)
        self.shape, self.dtype, self.device = shape, logits.dtype, logits.device
        self.classes = classes = shape[dim]
        self.rows_shape = rows_shape = shape[:dim] + shape[dim + 1:]
        self.rows = rows = math.prod(rows_shape)
        if not 1 <= classes <= 1 << 28:
            raise MicaHipError(f"logits: 1 to 2^28 classes expected along axis {dim}, got {classes}")
        if rows >= 1 << 31:
            raise MicaHipError(f"logits: fewer than 2^31 rows expected, got {rows}")
        self.base, self.moved = logits, False
        if dim == len(shape) - 1 and logits.is_contiguous():
            outer, inner, self.class_last, sc = (1, 0), (rows, classes if rows > 1 else 0), True, 1
        else:
            view = self._view(logits, dim)
            if view is None:
                if classes > COL_MAX and dim != len(shape) - 1:
                    self.base, self.moved = logits.movedim(dim, -1).contiguous(), True
                    view = self._view(self.base, len(shape) - 1)
                else:
                    self.base = logits.contiguous()
                    view = self._view(self.base, dim)
            outer, inner, self.class_last, sc = view
        self.strides = self.base.stride()
        self.desc = _cabi.MicaLogits(self.base.data_ptr(), dtype, self.class_last, outer[0], inner[0], classes, outer[1], inner[1], sc)

    def release(self):
        """-> the tensor the view points into, for autograd to keep: the layout stays behind with sizes and strides alone"""
        base, self.base = self.base, None
        return base

    def over(self, base):
        """this layout of `base`, a tensor of release()'s values: that tensor itself, or what a saved-tensor hook made of it"""
        if base.data_ptr() == self.desc.d_data and base.stride() == self.strides:
            return self
        v = LogitsLayout(base, base.dim() - 1 if self.moved else self.dim)
        v.dim, v.shape, v.rows_shape, v.moved = self.dim, self.shape, self.rows_shape, self.moved
        return v

    @staticmethod
    def _view(t, dim):
        """-> ((outer, stride), (inner, stride), class_last, class stride), or None where the library has no view of t."""
        n, s = t.shape, t.stride()
        before, after = _collapse(n[:dim], s[:dim]), _collapse(n[dim + 1:], s[dim + 1:])
        sc = s[dim] if n[dim] > 1 else 1
        if not after:
            if n[dim] > COL_MAX and sc != 1 or len(before) > 2:
                return None
            before = [(1, 0)] * (2 - len(before)) + before
            return before[0], before[1], True, sc
        if n[dim] > COL_MAX or len(before) > 1 or len(after) > 1:
            return None
        return (before or [(1, 0)])[0], after[0], False, sc

    def score_aux(self):
        """what token_logprobs hands to its backward pass: maximum and sum of every row; None for few classes, which a thread sums again"""
        return torch.empty((2, self.rows), dtype=torch.float32, device=self.device) if self.classes > COL_MAX else None

    def with_axis(self, k):
        """shape with k entries at the class axis, as the library lays it out"""
        return self.rows_shape + (k,) if self.moved else self.shape[:self.dim] + (k,) + self.shape[self.dim + 1:]

    def give(self, t):
        """a result of that shape, with the axis where the caller has it"""
        return t.movedim(-1, self.dim) if self.moved else t

    def take(self, t):
        """a list the caller passes, as the library reads it"""
        return (t.movedim(self.dim, -1) if self.moved else t).contiguous()


def check_temperature(t):
    t = float(t)
    if not 1e-4 <= t <= 1e4:
        raise MicaHipError(f"temperature must be in [1e-4, 1e4], got {t}")
    return t


def check_ints(t, name, shape, device):
    if not isinstance(t, torch.Tensor) or t.dtype not in INTS or t.shape != shape or t.device != device:
        got = f"{t.dtype} {tuple(t.shape)} on {t.device}" if isinstance(t, torch.Tensor) else type(t)
        raise MicaHipError(f"{name}: expected an int32 or int64 tensor of shape {tuple(shape)} on {device}, got {got}")
    return t


def check_floats(t, name, shape, device, dtypes=(torch.float32,)):
    if not isinstance(t, torch.Tensor) or t.dtype not in dtypes or t.shape != shape or t.device != device:
        got = f"{t.dtype} {tuple(t.shape)} on {t.device}" if isinstance(t, torch.Tensor) else type(t)
        raise MicaHipError(f"{name}: expected a {' / '.join(str(d) for d in dtypes)} tensor of shape {tuple(shape)} on {device}, got {got}")
    return t


def top_list(layout: LogitsLayout, index, value, tail, device):
    """-> (the library's description of a teacher's list, the tensors it points into)"""
    if not isinstance(index, torch.Tensor) or index.dim() != len(layout.shape):
        raise MicaHipError(f"teacher_index: expected a tensor of {len(layout.shape)} axes, the list at axis {layout.dim}")
    k = index.shape[layout.dim]
    if not 1 <= k <= MAX_LIST:
        raise MicaHipError(f"teacher_index: 1 to {MAX_LIST} entries per row expected, got {k}")
    shape = layout.shape[:layout.dim] + (k,) + layout.shape[layout.dim + 1:]
    check_ints(index, "teacher_index", shape, device)
    check_floats(value, "teacher_logprob", shape, device, DTYPES)
    index, value = layout.take(index), layout.take(value)
    return _cabi.MicaTopList(index.data_ptr(), value.data_ptr(), index.element_size(), DTYPES[value.dtype], k, int(bool(tail))), (index, value)


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, engine, tokens, top, dim, temperature, ignore_index):
        view = engine.logits_view(logits, dim)
        aux = view.score_aux()
        with engine.call_lock:
            r = engine._scores(view, tokens, top, temperature, ignore_index, aux)
        # every tensor through save_for_backward: torch frees them after the backward pass, refuses one over logits that were written since,
        # and lets hooks keep them elsewhere
        ctx.save_for_backward(view.release(), r.entropy, tokens, aux)
        ctx.call = engine, view, float(temperature), ignore_index
        if r.top_index is not None:
            ctx.mark_non_differentiable(r.top_logprob, r.top_index)
        ctx.set_materialize_grads(False)
        return tuple(r)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_logprob, g_entropy, g_lse, *_):
        if g_logprob is None and g_entropy is None and g_lse is None:
            return (None,) * 7
        base, entropy, tokens, aux = ctx.saved_tensors
        engine, view, temperature, ignore_index = ctx.call
        with engine.call_lock:
            grad = engine._score_gradient(view.over(base), tokens, aux, entropy, g_logprob, g_entropy, g_lse, temperature, ignore_index)
        return grad, None, None, None, None, None, None


def token_logprobs(engine, logits, tokens=None, top: int = 0, dim: int = -1, temperature: float = 1.0, ignore_index: int = -100) -> TokenScores:
    """Engine.token_logprobs in an autograd graph: logprob, entropy and lse are differentiable (once), the alternatives are not."""
    return TokenScores(*_TokenLogprobs.apply(logits, engine, tokens, top, dim, temperature, ignore_index))


class _DistillLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, student, engine, index, logprob, dim, temperature, tail):
        view = engine.logits_view(student, dim, "student")
        loss, aux = engine.distill_loss(student, index, logprob, dim, temperature, tail, view)
        ctx.save_for_backward(view.release(), index, logprob, aux)
        ctx.call = engine, view, dim, temperature, tail
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_loss):
        base, index, logprob, aux = ctx.saved_tensors
        engine, view, dim, temperature, tail = ctx.call
        return (engine.distill_backward(base, index, logprob, aux, g_loss, dim, temperature, tail, view.over(base)), None, None, None, None, None, None)


def distill_loss(engine, student, teacher_index, teacher_logprob, dim: int = -1, temperature: float = 1.0, tail: bool = False) -> torch.Tensor:
    """Engine.distill_loss in an autograd graph: the per-row loss, differentiable (once) in the student's logits; the teacher's list is a
    constant."""
    return _DistillLoss.apply(student, engine, teacher_index, teacher_logprob, dim, temperature, tail)
