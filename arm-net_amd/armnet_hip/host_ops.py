"""The module surface on HOST tensors: the reference's ATen op chain, for a model that was never moved to the GPU.

The reference's model runs wherever its tensors are (`models/model_utils.py:86` calls `.cuda()` only if a device is
available; `train.py:103-106`).  This file is the branch `ARMNetModel.arm_block`, `models.layers.Embedding` and
`utils.entmax.entmax_bisect` take when BOTH the parameters and the batch are CPU tensors: plain torch ops in the
reference's order — in-place clamp, embedding x value, key projection, gates,
the 50-step bisection of `utils/entmax.py:29-68` with tensor-tensor `pow`, value weighting, einsum + exp — differentiable
by autograd (the sparse map through `block._EntmaxFn`, whose backward is `entmax.py:70-80`).

It is a DEVICE DISPATCH, not a fallback: device tensors never come here (a missing / unloadable HIP library, or a model
and a batch on different devices, still raise), nothing here touches `oracle/`, and `bench.py` times it as the
`cpu_baseline.aten_chain` leg next to the GPU number."""
import torch
import torch.nn.functional as Fn


def on_host(*tensors):
    """True when every tensor lives in host memory (the reference's CPU path); mixed placements are the caller's error"""
    return all(not t.is_cuda for t in tensors)


def note_host_branch(owner):
    """A model that was never moved to the GPU runs the reference's ATen chain on the host — the reference's own device
    semantics (model_utils.py:86), but orders of magnitude slower than the HIP path.  On a box that HAS a GPU that is most
    likely a forgotten `.cuda()`: say so once per model (`model.allow_host = True` or
    ARMNET_ALLOW_HOST=1 silences it).  On a box without a GPU there is nothing to warn about."""
    if getattr(owner, "_host_noted", False) or getattr(owner, "allow_host", False):
        return
    owner._host_noted = True
    import os
    if torch.cuda.is_available() and not os.environ.get("ARMNET_ALLOW_HOST"):
        import warnings
        warnings.warn(f"{type(owner).__name__}: model and batch are in host memory — running the reference's ATen op chain on "
                      "the CPU, not the HIP kernels (this box has a GPU: call model.cuda() and move the batch, or set "
                      "model.allow_host = True to silence this)", RuntimeWarning, stacklevel=3)


def clamp_vals_(vals):
    """armnet_1h.py:81 / armnet.py:82: x['value'].clamp_(0.001, 1.) in place"""
    return vals.clamp_(0.001, 1.0)


def embedding(ids, vals, table):
    """layers.py:15-21: table[ids] * vals.unsqueeze(2); out-of-range ids raise torch's own IndexError"""
    x = Fn.embedding(ids, table)
    return x if vals is None else x * vals.unsqueeze(-1)


def entmax_bisect(X, alpha, dim=-1, n_iter=50, ensure_sum_one=True):
    """utils/entmax.py:29-68 statement for statement on ATen ops (softmax when alpha == 1, as armnet_1h.py:12 builds it):
    alpha as a broadcast TENSOR (the reference's `pow` is tensor-tensor), tau_lo = max - 1, tau_hi = max - (1/d)^(alpha-1),
    n_iter halvings keeping the side on which f has the sign of f_lo, p of the LAST tau_m, renormalised."""
    moved = dim % X.dim() != X.dim() - 1
    if torch.is_tensor(alpha) and alpha.numel() != 1:
        # entmax.py:31-36: a tensor alpha, already expanded to X's shape with extent 1 along `dim`
        Xm = X.movedim(dim, -1) if moved else X
        al = (alpha.movedim(dim, -1) if moved else alpha).to(Xm.dtype)
    else:
        if float(alpha) == 1.0:
            return torch.softmax(X, dim=dim)
        Xm = X.movedim(dim, -1) if moved else X
        al = torch.full((1,) * Xm.dim(), float(alpha), dtype=Xm.dtype, device=Xm.device).expand(*Xm.shape[:-1], 1)
    d = Xm.shape[-1]
    am1 = al - 1
    inv = 1 / am1
    Xs = Xm * am1
    mx = Xs.max(dim=-1, keepdim=True).values
    tau_lo = mx - 1.0
    tau_hi = mx - (1.0 / d) ** am1
    f_lo = torch.clamp(Xs - tau_lo, min=0).pow(inv).sum(-1, keepdim=True) - 1
    dm = tau_hi - tau_lo
    p = None
    for _ in range(n_iter):
        dm = dm / 2
        tau_m = tau_lo + dm
        p = torch.clamp(Xs - tau_m, min=0).pow(inv)
        f_m = p.sum(-1, keepdim=True) - 1
        tau_lo = torch.where((f_m * f_lo) >= 0, tau_m, tau_lo)
    if p is None:                                               # n_iter == 0: the reference fails on the unbound p_m too
        raise ValueError("entmax_bisect needs n_iter >= 1")
    if ensure_sum_one:
        p = p / p.sum(-1, keepdim=True)
    return p.movedim(-1, dim) if dim % X.dim() != X.dim() - 1 else p


def arm_block(variant_one_head, ids, vals, table, bilinear_w, query, values, alpha, n_iter=50):
    """rows a2..a8 of SURVEY.md §8a on host tensors -> the pre-BatchNorm exponential neurons [B, K*H, E].
    `vals` is clamped in place.  one head: bilinear_w [D,E] (nn.Linear weight), query [H,D], values [H,F];
    multi-head: bilinear_w [K,E,D], query [K,H,D], values [K,H,F]."""
    from .block import entmax_forward
    clamp_vals_(vals)                                                           # armnet_1h.py:81 / armnet.py:82
    x = embedding(ids, vals, table)                                             # layers.py:20-21
    scale = query.shape[-1] ** -0.5
    if variant_one_head:                                                        # armnet_1h.py:30-34, 85-86
        keys = Fn.linear(x, bilinear_w)
        gates = torch.einsum("bfe,oe->bof", keys, query) * scale
        p = entmax_forward(gates, alpha, dim=-1, n_iter=n_iter)
        w = torch.einsum("bof,of->bof", p, values)
        return torch.exp(torch.einsum("bfe,bof->boe", x, w))
    gates = torch.einsum("bfx,kxy,koy->bkof", x, bilinear_w, query) * scale    # armnet.py:33-36, 86-88
    p = entmax_forward(gates, alpha, dim=-1, n_iter=n_iter)
    w = torch.einsum("bkof,kof->bkof", p, values)
    z = torch.exp(torch.einsum("bfe,bkof->bkoe", x, w))
    return z.reshape(z.shape[0], -1, z.shape[-1])                               # 'b k o e -> b (k o) e'


# ---- row operators on host tensors: the formulas of csrc/layer_norm.hip and csrc/score_rows.hip on ATen ops, in float32 or
# ---- wider, rounded once to the tensors' type

def _wide(x):
    return x if x.dtype == torch.float64 else x.float()


def layer_norm_fwd(x, weight, bias, eps):
    """y and the statistics [2, .., 1]: mean, 1 / standard deviation"""
    xw = _wide(x)
    mean = xw.mean(-1, keepdim=True)
    xc = xw - mean
    rstd = 1.0 / torch.sqrt((xc * xc).mean(-1, keepdim=True) + eps)
    y = xc * rstd
    if weight is not None:
        y = y * _wide(weight)
    if bias is not None:
        y = y + _wide(bias)
    return y.to(x.dtype), torch.stack((mean, rstd))


def layer_norm_bwd(x, dy, weight, st, need_dx, need_dw, need_db, p_dtype):
    mean, rstd = st
    dyw, h = _wide(dy), (_wide(x) - mean) * rstd
    g = dyw if weight is None else dyw * _wide(weight)
    dx = (rstd * (g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True))).to(x.dtype) if need_dx else None
    d = x.shape[-1]
    dw = (dyw * h).reshape(-1, d).sum(0).to(p_dtype) if need_dw else None
    db = dyw.reshape(-1, d).sum(0).to(p_dtype) if need_db else None
    return dx, dw, db


def _log_softmax_rows(x, temperature):
    """log p of every score; -inf everywhere in a row of nothing but -inf; NaN in a row with a NaN or +inf"""
    m = x.amax(-1, keepdim=True)
    low = torch.full_like(m, torch.finfo(x.dtype).min)
    z = (x - torch.where(m == -float("inf"), low, m)) / temperature
    s = torch.exp(z).sum(-1, keepdim=True)
    return torch.where(s == 0, torch.full_like(z, -float("inf")), z - torch.log(s))


def _check_ids(ids, c, check):
    if check and bool((ids >= c).any()):
        raise IndexError("index out of range in self")


def _at_ids(lp, ids):
    """lp[.., ids]; 0 for an empty slot (a negative id), NaN past the row"""
    c = lp.shape[-1]
    v = lp.gather(-1, ids.long().clamp(0, c - 1))
    v = torch.where(ids >= c, torch.full_like(v, float("nan")), v)
    return torch.where(ids < 0, torch.zeros_like(v), v)


def score_logprobs_fwd(X, ids, temperature, top_k, entropy):
    lp = _log_softmax_rows(_wide(X), temperature)
    logp = None if ids is None else _at_ids(lp, ids)
    ent = None
    if entropy:
        p = torch.exp(lp)
        ent = -torch.where(p == 0, torch.zeros_like(p), p * lp).sum(-1)
    tl = ti = None
    if top_k:
        # a stable sort keeps the lowest id first among equals; -0 and 0 are equals
        ti = torch.sort(_wide(X), dim=-1, descending=True, stable=True).indices[..., :top_k]
        tl = lp.gather(-1, ti)
        ti = torch.where(X.gather(-1, ti) > -float("inf"), ti, torch.full_like(ti, -1))
        ti = torch.where(torch.isnan(tl), torch.full_like(ti, -1), ti)
    return logp, ent, tl, ti


def score_logprobs_bwd(X, ids, temperature, entropy, g_logp, g_entropy):
    x = _wide(X)
    lp = _log_softmax_rows(x, temperature)
    p = torch.exp(lp)
    dz = torch.zeros_like(p)
    live = (lp > -float("inf")).any(-1, keepdim=True) | torch.isnan(lp).any(-1, keepdim=True)
    if g_logp is not None:
        ok = (ids >= 0) & (ids < x.shape[-1]) & live
        g = torch.where(ok, g_logp.to(p.dtype), torch.zeros((), dtype=p.dtype))
        dz = torch.where(ok.any(-1, keepdim=True), -p * g.sum(-1, keepdim=True), torch.zeros_like(p))    # padding: 0, whatever it holds
        dz = dz.scatter_add(-1, ids.long().clamp(0, x.shape[-1] - 1), g)
    if g_entropy is not None:
        t = torch.where(p == 0, torch.zeros_like(p), p * (lp + entropy.to(p.dtype).unsqueeze(-1)))
        gh = g_entropy.to(p.dtype).unsqueeze(-1)
        dz = dz - torch.where(gh == 0, torch.zeros_like(t), gh * t)
    return (dz / temperature).to(X.dtype)


def _teacher(ids, teacher, temperature, dtype):
    """(log q, q) over the listed slots; q = 0 in empty ones and in rows without a teacher"""
    t = torch.where(ids < 0, torch.full((), -float("inf"), dtype=dtype), teacher.to(dtype))
    lq = _log_softmax_rows(t, temperature)
    return lq, torch.exp(lq)


def distill_fwd(X, ids, teacher, temperature):
    x = _wide(X)
    lp = _at_ids(_log_softmax_rows(x, temperature), ids)
    lq, q = _teacher(ids, teacher, temperature, x.dtype)
    return temperature ** 2 * torch.where(q == 0, torch.zeros_like(q), q * (lq - lp)).sum(-1)


def distill_bwd(X, ids, teacher, temperature, g_loss):
    x = _wide(X)
    c = x.shape[-1]
    lp = _log_softmax_rows(x, temperature)
    p = torch.exp(lp)
    live = (lp > -float("inf")).any(-1, keepdim=True) | torch.isnan(lp).any(-1, keepdim=True)
    _, q = _teacher(ids, teacher, temperature, x.dtype)
    told = q.sum(-1, keepdim=True)
    told = torch.where(told > 0, torch.ones_like(told), told)
    d = torch.where(told == 0, torch.zeros_like(p), p * told).scatter_add(-1, ids.long().clamp(0, c - 1),
                               torch.where((ids >= 0) & (ids < c) & live, -q, torch.zeros_like(q)))
    return (d * (g_loss.to(x.dtype) * temperature).unsqueeze(-1)).to(X.dtype)
