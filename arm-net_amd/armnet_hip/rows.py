"""Row operators: layer norm, log probabilities of score rows, distillation from a teacher's listed scores.

A row is the last dimension of a tensor: a sample's features in front of a projection, or its scores over the classes / ids
behind one.  `layer_norm` stands beside the training BatchNorm (it needs no batch statistics: a batch of one, a sharded
server), `score_logprobs` and `distill_loss` beside the sparse map over a row of scores: what a row answers, and what a
student learns from a teacher's answer.  Device tensors run the HIP kernels (float32, bfloat16, float16; fp32 arithmetic),
host tensors the same formulas on ATen ops.  All three are differentiable once, by a backward pass; an input with a
forward-mode tangent is refused, and so are, on the device, a call while a trace is recorded (torch.jit.trace, make_fx) and a
tensor without memory.
"""
from typing import NamedTuple, Optional

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import host_ops, native
from .block import IdStatus, _id_mode

_FLOATS = (torch.float32, torch.bfloat16, torch.float16)


def _place(what, first, *others):
    """True on the device, False on the host; tensors in different places raise"""
    for name, t in others:
        if t is not None and t.device != first.device:
            raise native.ArmnetNativeError(f"{what} is on {first.device}, {name} on {t.device}: move them to one device")
    return first.is_cuda


def _float_rows(x, what):
    if x.dim() < 1 or x.shape[-1] < 1:
        raise native.ArmnetNativeError(f"{what}: expected rows in the last dimension, got the shape {list(x.shape)}")
    if x.dtype not in _FLOATS and not (x.dtype == torch.float64 and not x.is_cuda):
        raise native.ArmnetNativeError(f"{what}: expected float32, bfloat16 or float16, got {x.dtype}")


def _temperature(t):
    if isinstance(t, bool) or not isinstance(t, (int, float)) or not 1e-6 <= t <= 1e6:
        raise native.ArmnetNativeError(f"temperature: expected a number in [1e-6, 1e6], got {t!r}")
    return float(t)


def _poll(status, devices):
    for d in devices:
        if d.type == "cuda":
            torch.cuda.synchronize(d)
    status.raise_if_set()


# ---- layer norm ----------------------------------------------------------------------------------------------------------

class _HostLayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, st = host_ops.layer_norm_fwd(x, weight, bias, eps)
        ctx.save_for_backward(x, weight, st)
        p = weight if weight is not None else bias
        ctx.p_dtype = None if p is None else p.dtype
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, st = ctx.saved_tensors
        return host_ops.layer_norm_bwd(x, dy, weight, st, *ctx.needs_input_grad[:3], ctx.p_dtype) + (None,)


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension of x [.., D], in x's type.

    weight, bias: [D] or None, both of one type (float32 parameters beside 16-bit activations are fine).  Leading strides are
    taken as they are where two describe them; y is dense.  Differentiable in x, weight and bias; the parameters' gradients are
    summed in a fixed order."""
    _float_rows(x, "x")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is not None and (tuple(p.shape) != (x.shape[-1],) or (p.dtype not in _FLOATS and p.dtype != x.dtype)):
            raise native.ArmnetNativeError(f"{name}: expected [{x.shape[-1]}] float32, bfloat16 or float16, got "
                                           f"{list(p.shape)} {p.dtype}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise native.ArmnetNativeError(f"weight and bias are of different types ({weight.dtype}, {bias.dtype})")
    if not eps >= 0:
        raise native.ArmnetNativeError(f"eps: expected a number >= 0, got {eps!r}")
    on_device = _place("x", x, ("weight", weight), ("bias", bias))
    weight = weight if weight is None or weight.is_contiguous() else weight.contiguous()
    bias = bias if bias is None or bias.is_contiguous() else bias.contiguous()
    if on_device:
        return native.rows().layer_norm(x, weight, bias, float(eps))
    return _HostLayerNormFn.apply(x, weight, bias, float(eps))


class HipLayerNorm(nn.LayerNorm):
    """nn.LayerNorm (same constructor, parameters and state_dict keys) on layer_norm()"""

    def forward(self, x):
        k = len(self.normalized_shape)
        if tuple(x.shape[-k:]) != tuple(self.normalized_shape):
            raise native.ArmnetNativeError(f"expected a tensor that ends in {list(self.normalized_shape)}, got {list(x.shape)}")
        w, b = self.weight, self.bias
        if k == 1:
            return layer_norm(x, w, b, self.eps)
        y = layer_norm(x.flatten(-k), None if w is None else w.flatten(), None if b is None else b.flatten(), self.eps)
        return y.view(x.shape)


# ---- log probabilities ---------------------------------------------------------------------------------------------------

class ScoreLogprobs(NamedTuple):
    """what score_logprobs() returns; None for what was not asked for"""
    logp: Optional[torch.Tensor]          # of the given ids, their shape, float32
    entropy: Optional[torch.Tensor]       # per row, float32
    top_logp: Optional[torch.Tensor]      # [.., top_k], best first, float32
    top_ids: Optional[torch.Tensor]       # [.., top_k], int64


class _HostScoreLogprobsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, X, ids, temperature, top_k, entropy):
        logp, ent, tl, ti = host_ops.score_logprobs_fwd(X, ids, temperature, top_k, entropy)
        ctx.save_for_backward(X, ids, ent)
        ctx.temperature = temperature
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(*(t for t in (tl, ti) if t is not None))
        return logp, ent, tl, ti

    @staticmethod
    @once_differentiable
    def backward(ctx, g_logp, g_entropy, _tl, _ti):
        X, ids, ent = ctx.saved_tensors
        dx = None
        if g_logp is not None or g_entropy is not None:
            dx = host_ops.score_logprobs_bwd(X, ids, ctx.temperature, ent, g_logp, g_entropy)
        return (dx,) + (None,) * 4


def _row_ids(ids, lead, name):
    """ids as [.., n] for rows of the shape `lead`, and whether they came as one per row"""
    if ids.dtype not in (torch.int64, torch.int32):
        raise native.ArmnetNativeError(f"{name} must be int64 or int32, got {ids.dtype}")
    one = ids.dim() == len(lead)
    if not 0 <= ids.dim() - len(lead) <= 1 or (ids.shape if one else ids.shape[:-1]) != lead:
        raise native.ArmnetNativeError(f"{name}: expected {list(lead)} or {list(lead) + ['n']}, got {list(ids.shape)}")
    ids = ids.unsqueeze(-1) if one else ids
    if ids.shape[-1] > native.MAX_ROW_IDS:
        raise native.ArmnetNativeError(f"{name}: at most {native.MAX_ROW_IDS} ids a row, got {ids.shape[-1]}")
    return ids.contiguous(), one


def score_logprobs(X, ids=None, temperature=1.0, top_k=0, entropy=False, check_ids=True, status=None):
    """What rows of scores X [.., C] say, p = softmax(X / temperature): ScoreLogprobs(logp, entropy, top_logp, top_ids).

    ids       [..] or [.., n] (n <= 1024), int64 / int32: logp has their shape.  A negative id is an empty slot: log p 0 and no
              gradient.  An id >= C is an IndexError — check_ids / status as for the embedding lookup (deferred to the owner's
              next call with a `status`, else before this call returns); its log p is NaN
    top_k     0 .. min(64, C): the largest scores' log p and ids, best first, ties to the lowest id
    entropy   -sum p log p per row

    A score of -inf is masked: it is no alternative (slots past the last unmasked score: -inf and -1).  A row of nothing but
    -inf: log p -inf, entropy 0, gradient 0.  A row with a NaN or +inf: NaN, alternatives -1.  A row of empty slots (padding) whose
    entropy has no gradient or 0: gradient 0, whatever it holds.  Differentiable in X through logp
    and entropy (not through top_logp: pass top_ids as ids for that)."""
    _float_rows(X, "X")
    t = _temperature(temperature)
    if isinstance(top_k, bool) or not isinstance(top_k, int) or not 0 <= top_k <= min(native.MAX_ROW_TOP, X.shape[-1]):
        raise native.ArmnetNativeError(f"top_k: expected 0 .. {min(native.MAX_ROW_TOP, X.shape[-1])}, got {top_k!r}")
    one = False
    if ids is not None:
        ids, one = _row_ids(ids, X.shape[:-1], "ids")
    on_device = _place("X", X, ("ids", ids))
    word = sync = None
    if ids is not None and on_device:
        status, sync = _id_mode(check_ids, status)
        word = None if status is None else status.word()
    elif ids is not None:
        host_ops._check_ids(ids, X.shape[-1], check_ids)
    if on_device:
        out = native.rows().score_logprobs(X, ids, t, top_k, bool(entropy), word)
    else:
        out = _HostScoreLogprobsFn.apply(X, ids, t, top_k, bool(entropy))
    if sync:
        status.poll(X.device)
    return ScoreLogprobs(out[0].squeeze(-1) if one else out[0], *out[1:])


class HipScoreLogprobs(nn.Module):
    """score_logprobs() with its settings and the deferred report of ids out of range: check_ids = True raises IndexError at the
    next call or at poll(), "sync" before the call returns, False never (models.layers.Embedding has the same switch)"""

    def __init__(self, temperature=1.0, top_k=0, entropy=False):
        super().__init__()
        self.temperature, self.top_k, self.entropy = _temperature(temperature), top_k, entropy
        self.check_ids = True
        self._id_status, self._where = IdStatus(), set()

    def poll(self):
        """synchronise and raise IndexError if a call so far met an id past its row"""
        _poll(self._id_status, self._where)

    def forward(self, X, ids=None):
        self._where.add(X.device)
        return score_logprobs(X, ids, self.temperature, self.top_k, self.entropy, self.check_ids, self._id_status)


# ---- distillation --------------------------------------------------------------------------------------------------------

class _HostDistillFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, X, ids, teacher, temperature):
        ctx.save_for_backward(X, ids, teacher)
        ctx.temperature = temperature
        return host_ops.distill_fwd(X, ids, teacher, temperature)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        X, ids, teacher = ctx.saved_tensors
        return host_ops.distill_bwd(X, ids, teacher, ctx.temperature, g), None, None, None


def distill_loss(X, top_ids, top_scores, temperature=1.0, check_ids=True, status=None):
    """The distillation loss of every row of a student's scores X [.., C] from a teacher's listed ones:

        q = softmax(top_scores / T) over the row's listed ids,  p = softmax(X / T) over the whole row,
        loss = T^2 * sum_k q_k (log q_k - log p[top_ids_k])                                    [..], float32

    top_ids, top_scores: [.., k], k <= 1024; a negative id is an empty slot, an id >= C an IndexError (check_ids / status as for
    score_logprobs()).  score_logprobs(teacher_scores, top_k=k) gives both: its top_logp are the teacher's scores up to a
    constant that q does not see (at temperature 1).  A row without a teacher: loss and gradient 0, whatever X holds there.  An id that is listed
    twice counts twice.  A student's row of nothing but -inf: loss +inf, gradient 0.  Differentiable in X; the teacher is a
    constant (top_scores that require a gradient raise)."""
    _float_rows(X, "X")
    t = _temperature(temperature)
    ids, one = _row_ids(top_ids, X.shape[:-1], "top_ids")
    if one or ids.shape[-1] < 1:
        raise native.ArmnetNativeError(f"top_ids: expected {list(X.shape[:-1]) + ['k']}, got {list(top_ids.shape)}")
    if top_scores.shape != ids.shape or (top_scores.dtype not in _FLOATS and top_scores.dtype != X.dtype):
        raise native.ArmnetNativeError(f"top_scores: expected float32, bfloat16 or float16 of top_ids' shape {list(ids.shape)}, "
                                       f"got {list(top_scores.shape)} {top_scores.dtype}")
    if top_scores.requires_grad and torch.is_grad_enabled():
        raise native.ArmnetNativeError("top_scores requires a gradient: the teacher is a constant of this loss (detach it)")
    teacher = top_scores.contiguous()
    on_device = _place("X", X, ("top_ids", ids), ("top_scores", teacher))
    word = sync = None
    if on_device:
        status, sync = _id_mode(check_ids, status)
        word = None if status is None else status.word()
    else:
        host_ops._check_ids(ids, X.shape[-1], check_ids)
    if on_device:
        loss = native.rows().distill_loss(X, ids, teacher, t, word)
    else:
        loss = _HostDistillFn.apply(X, ids, teacher, t)
    if sync:
        status.poll(X.device)
    return loss


class HipDistillLoss(nn.Module):
    """distill_loss() with its temperature, a reduction over all rows ("mean", "sum" or "none") and the deferred report of ids
    out of range (check_ids, poll(): see HipScoreLogprobs)"""

    def __init__(self, temperature=1.0, reduction="mean"):
        super().__init__()
        if reduction not in ("mean", "sum", "none"):
            raise native.ArmnetNativeError(f"reduction: expected 'mean', 'sum' or 'none', got {reduction!r}")
        self.temperature, self.reduction = _temperature(temperature), reduction
        self.check_ids = True
        self._id_status, self._where = IdStatus(), set()

    def poll(self):
        """synchronise and raise IndexError if a call so far met an id past its row"""
        _poll(self._id_status, self._where)

    def forward(self, X, top_ids, top_scores):
        self._where.add(X.device)
        loss = distill_loss(X, top_ids, top_scores, self.temperature, self.check_ids, self._id_status)
        return loss if self.reduction == "none" else getattr(loss, self.reduction)()
