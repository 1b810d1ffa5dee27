"""The row operators of armnet_hip, as they are measured: layer norm, log probabilities of score rows, distillation.

Every operator works on rows: `N` rows of `D` values (layer norm) or of `C` scores, one per id (the other two).
`listed()` names the cases, `prepare()` makes a case's inputs from a seed, `run()` makes one pass — in plain tensor
operations, or with `own` set through armnet_hip's entry points —, `exact()` is the definition in 64 bits and `work()` what a
pass has to read, write and compute.

    norm     y = (x - mean) / sqrt(var + eps) * weight + bias over the last dimension; a training pass returns y and the
             gradients of x, weight and bias.
    scores   p = softmax(X / T).  Per row: log p of the given ids (a negative id is an empty slot: 0), the entropy of p, the
             `top` largest scores' log p and ids (ties: the lowest id; slots past the last unmasked score hold -inf and -1).
             A row without any score above -inf has log p = -inf, entropy 0 and gradient 0.
    distill  q = softmax of the teacher's listed scores / T (a negative id is an empty slot);
             loss = T^2 * sum_k q_k (log q_k - log p[id_k]) per row, and its gradient in X.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-5


def listed():
    return [
        # eight requests' 512 exponential neurons (32 neurons x 16) normalised before the head: the time of a call
        {"name": "norm_serve_8x512_f32", "op": "norm", "n": 8, "d": 512, "type": "f32", "train": False, "pad": 0},
        # the training batch of the Criteo-shaped block, the norm in BatchNorm's place in front of the head
        {"name": "norm_train_65536x512_f32", "op": "norm", "n": 65536, "d": 512, "type": "f32", "train": True, "pad": 0},
        # a wide block (256 neurons x 16) in 16 bits
        {"name": "norm_train_16384x4096_bf16", "op": "norm", "n": 16384, "d": 4096, "type": "bf16", "train": True, "pad": 0},
        # odd sizes, rows that are part of wider ones (an ensemble's two branches side by side)
        {"name": "norm_fwd_10007x2049_f16_part", "op": "norm", "n": 10007, "d": 2049, "type": "f16", "train": False, "pad": 51},
        # one request against the whole id space of the headline table: the best twenty ids
        {"name": "scores_1x1000000_f32_top20", "op": "scores", "n": 1, "c": 1000000, "type": "f32", "ids": 1, "top": 20,
         "entropy": True, "train": False, "temp": 1.0, "masked": 0.01},
        # a batch of requests against the same id space
        {"name": "scores_256x1000000_bf16_top50", "op": "scores", "n": 256, "c": 1000000, "type": "bf16", "ids": 1, "top": 50,
         "entropy": True, "train": False, "temp": 0.7, "masked": 0.0},
        # training a classifier on the large batch: log probability of the label, with an entropy bonus
        {"name": "scores_train_65536x1001_f32", "op": "scores", "n": 65536, "c": 1001, "type": "f32", "ids": 1, "top": 0,
         "entropy": True, "train": True, "temp": 1.0, "masked": 0.0},
        # lists of a hundred candidates out of Frappe's ids, padded lists, ids that are not on offer masked
        {"name": "scores_train_4096x5382_bf16_list", "op": "scores", "n": 4096, "c": 5382, "type": "bf16", "ids": 100, "top": 0,
         "entropy": False, "train": True, "temp": 1.5, "masked": 0.1},
        # a small student step
        {"name": "distill_64x5382_f32_k16", "op": "distill", "n": 64, "c": 5382, "type": "f32", "k": 16, "temp": 2.0},
        # Frappe's ids, a large batch, odd list length
        {"name": "distill_8191x5382_f16_k7", "op": "distill", "n": 8191, "c": 5382, "type": "f16", "k": 7, "temp": 4.0},
        # a large id space, long lists
        {"name": "distill_2048x131072_bf16_k64", "op": "distill", "n": 2048, "c": 131072, "type": "bf16", "k": 64, "temp": 1.0},
    ]


def _spread(rng, lo, hi):
    """a whole number between lo and hi, spread evenly over its logarithm"""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "scores", "distill"])
    dt = rng.choice(["f32", "bf16", "f16"])
    if op == "norm":
        d = _spread(rng, 8, 16384)
        return {"op": op, "n": _spread(rng, 1, min(131072, 60_000_000 // d)), "d": d, "type": dt,
                "train": rng.random() < 0.6, "pad": rng.choice([0, 0, 0, 3, 8])}
    c = _spread(rng, 2, 1000000)
    n = _spread(rng, 1, min(131072, 200_000_000 // c))
    if op == "scores":
        return {"op": op, "n": n, "c": c, "type": dt, "ids": rng.choice([1, 1, _spread(rng, 2, 200)]),
                "top": rng.choice([0, _spread(rng, 1, min(64, c))]), "entropy": rng.random() < 0.5,
                "train": rng.random() < 0.5, "temp": rng.choice([1.0, 1.0, 0.6, 2.5]), "masked": rng.choice([0.0, 0.0, 0.2])}
    return {"op": op, "n": n, "c": c, "type": dt, "k": _spread(rng, 1, min(c, 200)), "temp": rng.choice([1.0, 2.0, 5.0])}


def _scores_like(n, c, dt, gen):
    """scores as a head gives them: a spread of a few units, a few large ones per row"""
    x = torch.randn(n, c, generator=gen, device="cuda", dtype=torch.float32).mul_(2.0)
    if c >= 64:
        top = torch.randint(0, c, (n, 4), generator=gen, device="cuda")
        x.scatter_add_(1, top, 6.0 * torch.rand(n, 4, generator=gen, device="cuda"))
    return x.to(dt)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt, n = TYPES[case["type"]], case["n"]
    if case["op"] == "norm":
        d = case["d"]
        # exponential neurons: positive, a mean of about one, and of another scale in every row
        base = torch.randn(n, d + case["pad"], generator=gen, device="cuda").mul_(0.5)
        base = (base + 1.0 + torch.rand(n, 1, generator=gen, device="cuda")).to(dt)
        s = {"x": base[:, :d], "w": 1.0 + 0.1 * torch.randn(d, generator=gen, device="cuda"),
             "b": 0.1 * torch.randn(d, generator=gen, device="cuda")}
        if case["train"]:
            s["x"].requires_grad_(True), s["w"].requires_grad_(True), s["b"].requires_grad_(True)
            s["dy"] = torch.randn(n, d, generator=gen, device="cuda").to(dt)
        return dict(s, case=case)
    c = case["c"]
    x = _scores_like(n, c, dt, gen)
    if case["op"] == "scores":
        ids = torch.randint(0, c, (n, case["ids"]), generator=gen, device="cuda")
        if case["ids"] > 1:          # lists of different lengths: the rest of a row is empty
            length = torch.randint(1, case["ids"] + 1, (n, 1), generator=gen, device="cuda")
            ids = torch.where(torch.arange(case["ids"], device="cuda") < length, ids, torch.full_like(ids, -1))
        if case["masked"]:
            off = torch.rand(n, c, generator=gen, device="cuda") < case["masked"]
            off.scatter_(1, ids.clamp(min=0), False)
            x.masked_fill_(off, -math.inf)
            if n > 2:
                x[n // 2] = -math.inf        # nothing on offer
                ids[n // 2] = -1
        s = {"x": x, "ids": ids, "case": case}
        if case["train"]:
            x.requires_grad_(True)
            s["g"] = torch.randn(n, case["ids"], generator=gen, device="cuda") / case["ids"]
            s["gh"] = 0.1 * torch.randn(n, generator=gen, device="cuda")
        return s
    # the teacher agrees with the student in part: its list holds distinct ids, its scores are its own
    k = case["k"]
    start = torch.randint(0, c, (n, 1), generator=gen, device="cuda")
    step = max(1, c // k)
    ids = (start + step * torch.arange(k, device="cuda")) % c
    length = torch.randint(1, k + 1, (n, 1), generator=gen, device="cuda")
    if n > 2:
        length[n // 2] = 0               # a row that the teacher says nothing about
    ids = torch.where(torch.arange(k, device="cuda") < length, ids, torch.full_like(ids, -1))
    teacher = torch.randn(n, k, generator=gen, device="cuda").mul_(2.0).sort(dim=1, descending=True).values + 5.0
    return {"x": x.requires_grad_(True), "ids": ids, "teacher": teacher,
            "g": torch.rand(n, generator=gen, device="cuda") / n * 64.0, "case": case}


# ---- the plain forms -----------------------------------------------------------------------------------------------------

def _norm_plain(s):
    case = s["case"]
    x = s["x"].detach().float()
    mean = x.mean(1, keepdim=True)
    xc = x - mean
    rstd = 1.0 / torch.sqrt((xc * xc).mean(1, keepdim=True) + EPS)
    xhat = xc * rstd
    y = (xhat * s["w"].detach() + s["b"].detach()).to(s["x"].dtype)
    if not case["train"]:
        return y
    dy = s["dy"].float()
    g = dy * s["w"].detach()
    dx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
    return y, dx.to(s["x"].dtype), (dy * xhat).sum(0), dy.sum(0)


def _log_p(x, temp):
    """(x - max) / T and the logarithm of the sum of its exponentials; rows without a score have 0 for both"""
    m = x.amax(1, keepdim=True)
    some = m > -math.inf
    z = torch.where(some, x - torch.where(some, m, torch.zeros_like(m)), torch.full_like(x, -math.inf)) / temp
    e = torch.exp(z)
    total = e.sum(1, keepdim=True)
    return z, e, torch.where(some, total, torch.ones_like(total)), some


def _best(x, top):
    """the `top` largest of each row and their ids, ties to the lowest id: whole-number keys that order like (value, -id)"""
    bits = (x.float() + 0.0).view(torch.int32).long()
    order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
    key = order * (1 << 31) + ((1 << 31) - 1 - torch.arange(x.shape[1], device=x.device))
    at = (1 << 31) - 1 - torch.topk(key, top, dim=1).values.remainder(1 << 31)
    return x.gather(1, at), at


def _scores_plain(s):
    case = s["case"]
    x = s["x"].detach()
    temp, ids = case["temp"], s["ids"]
    z, e, total, some = _log_p(x.float(), temp)
    log_total = torch.log(total)
    here = ids >= 0
    at = ids.clamp(min=0)
    logp = torch.where(here, z.gather(1, at) - log_total, torch.zeros_like(log_total))
    out = {"logp": logp}
    p = e / total if case["entropy"] or case["train"] else None
    if case["entropy"]:
        plogp = torch.where(p > 0, p * (z - log_total), torch.zeros_like(p))
        entropy = out["entropy"] = -plogp.sum(1)
    if case["top"]:
        value, best = _best(x, case["top"])
        live = value.float() > -math.inf
        out["top_ids"] = torch.where(live, best, torch.full_like(best, -1))
        out["top_logp"] = torch.where(live, z.gather(1, best) - log_total, torch.full_like(value.float(), -math.inf))
    if case["train"]:
        g = torch.where(here & some, s["g"], torch.zeros_like(s["g"]))
        dz = -p * g.sum(1, keepdim=True)
        if case["entropy"]:
            dz = dz - s["gh"][:, None] * (plogp + p * entropy[:, None])
        dz = dz.scatter_add(1, at, g)
        out["dx"] = (dz / temp).to(x.dtype)
    return out


def _distill_plain(s):
    case = s["case"]
    x, temp, ids = s["x"].detach(), case["temp"], s["ids"]
    z, e, total, _ = _log_p(x.float(), temp)
    here = ids >= 0
    t = torch.where(here, s["teacher"], torch.full_like(s["teacher"], -math.inf))
    zt, et, total_t, _ = _log_p(t, temp)
    q = et / total_t
    at = ids.clamp(min=0)
    logp = z.gather(1, at) - torch.log(total)
    loss = temp * temp * torch.where(q > 0, q * (zt - torch.log(total_t) - logp), torch.zeros_like(q)).sum(1)
    g = s["g"][:, None] * temp
    any_q = here.any(1, keepdim=True)
    dx = torch.where(any_q, e / total * g, torch.zeros_like(g)).scatter_add(1, at, -(q * g))
    return loss, dx.to(x.dtype)


# ---- the framework's own -------------------------------------------------------------------------------------------------

def _entry(case):
    """what a user's program makes once: the function or the module that it calls on every batch"""
    import os
    import sys
    package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "arm-net_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    import armnet_hip
    if case["op"] == "norm":
        return armnet_hip.layer_norm
    if case["op"] == "scores":
        return armnet_hip.HipScoreLogprobs(temperature=case["temp"], top_k=case["top"], entropy=case["entropy"])
    return armnet_hip.HipDistillLoss(temperature=case["temp"], reduction="none")


def _own(s):
    case = s["case"]
    call = s.get("call") or s.setdefault("call", _entry(case))
    if case["op"] == "norm":
        if not case["train"]:
            with torch.no_grad():
                return call(s["x"], s["w"], s["b"], EPS)
        y = call(s["x"], s["w"], s["b"], EPS)
        return (y.detach(), *torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["dy"]))
    if case["op"] == "scores":
        r = call(s["x"], s["ids"])
        out = {"logp": r.logp.detach()}
        if case["entropy"]:
            out["entropy"] = r.entropy.detach()
        if case["top"]:
            out["top_ids"], out["top_logp"] = r.top_ids, r.top_logp
        if case["train"]:
            outs, grads = ((r.logp, r.entropy), (s["g"], s["gh"])) if case["entropy"] else ((r.logp,), (s["g"],))
            out["dx"], = torch.autograd.grad(outs, s["x"], grads)
        return out
    loss = call(s["x"], s["ids"], s["teacher"])
    dx, = torch.autograd.grad(loss, s["x"], s["g"])
    return loss.detach(), dx


def run(state):
    if own:
        return _own(state)
    return {"norm": _norm_plain, "scores": _scores_plain, "distill": _distill_plain}[state["case"]["op"]](state)


# ---- the definition in 64 bits -------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].detach().double()
    if case["op"] == "norm":
        var, mean = torch.var_mean(x, dim=1, unbiased=False, keepdim=True)
        sd = torch.sqrt(var + EPS)
        h = (x - mean) / sd
        w = s["w"].detach().double()
        y = h * w + s["b"].detach().double()
        if not case["train"]:
            return y
        dy = s["dy"].double()
        a = dy * w
        # the projection of a onto what is orthogonal to the constants and to h
        dx = (a - a.sum(1, keepdim=True) / case["d"] - h * ((a * h).sum(1, keepdim=True) / case["d"])) / sd
        return y, dx, torch.sum(dy * h, dim=0), torch.sum(dy, dim=0)
    temp, n = case["temp"], case["n"]
    live = (x > -math.inf).any(1)
    x[~live] = 0.0
    lp = torch.log_softmax(x / temp, dim=1)
    lp[~live] = -math.inf
    p = torch.exp(lp)
    rows = torch.arange(n, device=x.device)[:, None]
    ids = s["ids"]
    if case["op"] == "scores":
        out = {"logp": torch.where(ids >= 0, lp[rows, ids.clamp(min=0)], torch.zeros((), dtype=torch.float64, device=x.device))}
        entropy = torch.special.entr(p).sum(1)
        if case["entropy"]:
            out["entropy"] = entropy
        if case["top"]:
            out["top_ids"] = None
            out["top_logp"] = torch.topk(lp, case["top"], dim=1).values
        if case["train"]:
            g = torch.where((ids >= 0) & live[:, None], s["g"], torch.zeros_like(s["g"])).double()
            d = torch.zeros_like(p).index_put((rows.expand_as(ids), ids.clamp(min=0)), g, accumulate=True)
            d = d - p * g.sum(1, keepdim=True)
            if case["entropy"]:
                d = d + s["gh"].double()[:, None] * (torch.special.entr(p) - p * entropy[:, None])
            out["dx"] = d / temp
        return out
    told = (ids >= 0).any(1)
    q = torch.softmax(s["teacher"].double().masked_fill(ids < 0, -math.inf) / temp, dim=1)
    q[~told] = 0.0
    given = torch.where(ids >= 0, lp[rows, ids.clamp(min=0)], torch.zeros((), dtype=torch.float64, device=x.device))
    loss = temp ** 2 * (torch.special.xlogy(q, q) - q * given).sum(1)
    full = torch.zeros_like(p).index_put((rows.expand_as(ids), ids.clamp(min=0)), q, accumulate=True)
    return loss, temp * (s["g"].double() * told)[:, None] * (p - full)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------

def work(case):
    n, b = case["n"], SIZE[case["type"]]
    if case["op"] == "norm":
        d = case["d"]
        if case["train"]:            # x and dy in, y and dx out; weight and bias in, their gradients out; about 17 operations a value
            return {"bytes": 4 * n * d * b + 16 * d, "flops": 17 * n * d}
        return {"bytes": 2 * n * d * b + 8 * d, "flops": 8 * n * d}
    c = case["c"]
    if case["op"] == "scores":
        out = n * case["ids"] * (8 + 4) + (4 * n if case["entropy"] else 0) + n * case["top"] * 12
        if case["train"]:            # the gradient out, the outputs' gradients in
            out += n * c * b + 4 * n * case["ids"] + (4 * n if case["entropy"] else 0)
        return {"bytes": n * c * b + out, "flops": n * c * (6 + (2 if case["entropy"] else 0) + (6 if case["train"] else 0))}
    return {"bytes": 2 * n * c * b + n * case["k"] * 12 + 8 * n, "flops": 11 * n * c}
