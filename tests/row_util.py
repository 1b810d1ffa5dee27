"""Row operators in 64 bits from their definitions, and what fp32 arithmetic with one rounding at the end may be off by.

U = 2^-24 is half a step of fp32.  A sum of n terms in any order is off by at most (its longest chain of additions) * U * the
sum of the terms' magnitudes; `chain(n)` bounds that length for the kernels: a row's sum runs over at least 64 threads (a
wave), then over a tree; a product, a subtraction or an exponential adds a few U."""
import ctypes
import math

import torch

U = 2.0 ** -24


def half_step(dtype, ref):
    """half a step of `dtype` at the values `ref` (subnormal numbers have a fixed step)"""
    f = torch.finfo(dtype)
    return ref.abs() * (f.eps / 2) * (1 + 1e-6) + f.smallest_normal * f.eps / 2


def chain(n):
    return math.ceil(n / 64) + 24


def norm_ref(x, w, b, eps):
    """y, mean, rstd, h in float64"""
    x = x.double()
    mean = x.mean(-1, keepdim=True)
    var = ((x - mean) ** 2).mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    h = (x - mean) * rstd
    y = h
    if w is not None:
        y = y * w.double()
    if b is not None:
        y = y + b.double()
    return y, mean, rstd, h


def norm_tol(x, w, b, eps, dtype):
    """y: the mean is off by chain U mean|x|, a centred value by that and U |x|, the rest is relative"""
    y, mean, rstd, h = norm_ref(x, w, b, eps)
    n = chain(x.shape[-1])
    size = x.double().abs().mean(-1, keepdim=True)
    wd = torch.ones_like(h) if w is None else w.double().abs().expand_as(h)
    bd = torch.zeros_like(h) if b is None else b.double().abs().expand_as(h)
    slack = n * U * ((size + x.double().abs()) * rstd * wd + 4 * h.abs() * wd + bd)
    return y, half_step(dtype, y) + slack


def norm_grad_ref(x, w, eps, dy):
    """dx, dw, db in float64 and, for each, the sums of magnitudes that its rounding errors are relative to"""
    _, mean, rstd, h = norm_ref(x, w, None, eps)
    dy = dy.double()
    g = dy if w is None else dy * w.double()
    m1, m2 = g.mean(-1, keepdim=True), (g * h).mean(-1, keepdim=True)
    dx = rstd * (g - m1 - h * m2)
    # h itself is off by chain U times `k` (values far from 0 lose digits when they are centred)
    k = (x.double().abs().mean(-1, keepdim=True) + x.double().abs()) * rstd + 4 * h.abs()
    a1 = g.abs().mean(-1, keepdim=True)
    a2 = (g.abs() * (h.abs() + k)).mean(-1, keepdim=True)
    sx = rstd * (g.abs() + a1 + (h.abs() + k) * a2 + k * m2.abs())
    flat = lambda t: t.reshape(-1, t.shape[-1])      # noqa: E731
    return (dx, flat(dy * h).sum(0), flat(dy).sum(0)), (sx, flat(dy.abs() * (h.abs() + k)).sum(0), flat(dy).abs().sum(0))


def log_p(x, t):
    """log softmax(x / t) in float64: -inf everywhere in a row of nothing but -inf, NaN in one with a NaN or +inf"""
    z = x.double() / t
    m = z.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    s = torch.exp(z - m).sum(-1, keepdim=True)
    lp = (z - m) - torch.log(s)
    return torch.where(s == 0, torch.full_like(lp, -math.inf), lp)


def scores_ref(x, ids, t, top):
    lp = log_p(x, t)
    c = x.shape[-1]
    p = torch.exp(lp)
    ent = -torch.where(p == 0, torch.zeros_like(p), p * lp).sum(-1)
    logp = None
    if ids is not None:
        logp = lp.gather(-1, ids.long().clamp(0, c - 1))
        logp = torch.where(ids >= c, torch.full_like(logp, math.nan), torch.where(ids < 0, torch.zeros_like(logp), logp))
    # largest first, the lowest id among equals: sort by id, then stably by value
    order = torch.sort(x.double() + 0.0, dim=-1, descending=True, stable=True).indices[..., :top]
    tl = lp.gather(-1, order)
    order = torch.where((x.gather(-1, order) > -math.inf) & ~torch.isnan(tl), order, torch.full_like(order, -1))
    f32 = lambda v: None if v is None else v.float().double()        # results are fp32: what lies past its range is infinite    # noqa: E731
    return lp, f32(logp), f32(ent), f32(tl), order


def logp_tol(logp, x, t):
    """log p = z - log S: each part is off by a few U of its size, log S by what its sum's relative error is"""
    n = chain(x.shape[-1]) + z_size(x, t)
    return U * (n + 8 * torch.where(torch.isfinite(logp), logp.abs(), torch.zeros_like(logp)) + 8 * math.log(x.shape[-1] + 1))


def scores_grad_ref(x, ids, t, g, gh):
    """the gradient in X and the sum of magnitudes that its rounding errors are relative to"""
    lp = log_p(x, t)
    c = x.shape[-1]
    p = torch.exp(lp)
    live = (p > 0).any(-1, keepdim=True) | torch.isnan(p).any(-1, keepdim=True)
    d, size = torch.zeros_like(p), torch.zeros_like(p)
    if g is not None:
        gm = torch.where((ids >= 0) & (ids < c) & live, g.double(), torch.zeros((), dtype=torch.float64))
        at = ids.long().clamp(0, c - 1)
        d = (-p * gm.sum(-1, keepdim=True)).scatter_add(-1, at, gm)
        size = (p * gm.abs().sum(-1, keepdim=True)).scatter_add(-1, at, gm.abs())
    if gh is not None:
        ent = -torch.where(p == 0, torch.zeros_like(p), p * lp).sum(-1, keepdim=True)
        d = d - gh.double().unsqueeze(-1) * torch.where(p == 0, torch.zeros_like(p), p * (lp + ent))
        size = size + gh.double().abs().unsqueeze(-1) * torch.where(p == 0, torch.zeros_like(p), p * (lp.abs() + ent))
    return d / t, size / t


def z_size(x, t):
    """how far a row's scores reach below its largest, in units of the temperature: exponentials are off by that many U"""
    z = x.double() / t
    z = torch.where(torch.isfinite(z), z, torch.zeros_like(z))
    return (z.amax(-1, keepdim=True) - z.amin(-1, keepdim=True)).clamp(max=200.0)


def teacher_ref(ids, ts, t):
    s = torch.where(ids < 0, torch.full((), -math.inf, dtype=torch.float64), ts.double())
    lq = log_p(s, t)
    return lq, torch.exp(lq)


def distill_ref(x, ids, ts, t):
    """loss per row and the sum of magnitudes of its terms"""
    lp = log_p(x, t).gather(-1, ids.long().clamp(0, x.shape[-1] - 1))
    lq, q = teacher_ref(ids, ts, t)
    term = torch.where(q == 0, torch.zeros_like(q), q * (lq - lp))
    size = torch.where(q == 0, torch.zeros_like(q), q * (lq.abs() + torch.where(torch.isfinite(lp), lp.abs(), torch.zeros_like(lp)) + 1))
    return t * t * term.sum(-1), t * t * size.sum(-1)


def distill_grad_ref(x, ids, ts, t, g):
    p = torch.exp(log_p(x, t))
    live = (p > 0).any(-1, keepdim=True)
    _, q = teacher_ref(ids, ts, t)
    told = (q.sum(-1, keepdim=True) > 0).double()
    q = torch.where((ids >= 0) & live, q, torch.zeros_like(q))
    at = ids.long().clamp(0, x.shape[-1] - 1)
    gt = g.double().unsqueeze(-1) * t
    return gt * (p * told).scatter_add(-1, at, -q), gt.abs() * (p * told).scatter_add(-1, at, q)


def close(got, ref, tol):
    """non-finite values in the same places, the rest within tol"""
    got, ref = got.detach().double().cpu(), ref.detach().double().cpu()
    tol = tol.detach().double().cpu().expand_as(ref) if torch.is_tensor(tol) else torch.full_like(ref, tol)
    fine = torch.isfinite(ref)
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), "NaN in other places"
    inf = ~fine & ~torch.isnan(ref)
    assert torch.equal(got[inf], ref[inf]) and bool(torch.isfinite(got[fine]).all()), "infinities in other places"
    if fine.any():
        over = (got - ref).abs()[fine] - tol[fine]
        i = int(over.argmax())
        assert float(over.max()) <= 0, f"off by {float((got - ref).abs()[fine][i]):.3g}, {float(tol[fine][i]):.3g} allowed, at {float(ref[fine][i]):.6g}"


def declare_row_calls(lib):
    """argument types of the row operators' C entries, so that plain numbers and addresses can be passed"""
    i, l, f, p = ctypes.c_int, ctypes.c_int64, ctypes.c_float, ctypes.c_void_p
    view = [l, l, l, l, l, i, p]                        # rows, inner, outer_stride, row_stride, last dimension, type, x
    ids = [f, l, p, i]                                  # temperature, ids of a row, ids, their type
    for name, args, res in (
            ("armnet_layer_norm_fwd", view + [i, p, p, f, p, p, p, p], i),
            ("armnet_layer_norm_bwd_ws_bytes", [l, l], l),
            ("armnet_layer_norm_bwd", view + [p, i, p, p, p, p, p, p, p, l, p], i),
            ("armnet_score_ws_bytes", [l, l, i], l),
            ("armnet_score_logprobs_fwd", view + ids + [i, p, p, p, p, p, p, l, p, p], i),
            ("armnet_score_logprobs_bwd", view + ids + [p, p, p, p, p, p], i),
            ("armnet_distill_fwd", view + ids + [i, p, p, p, p, l, p, p], i),
            ("armnet_distill_bwd", view + ids + [i, p, p, p, p, p], i)):
        fn = getattr(lib, name)
        fn.argtypes, fn.restype = args, res
