"""The row operators' HIP kernels against their definitions in 64 bits (row_util derives what they may be off by)."""
import math

import pytest
import torch

from armnet_hip import HipDistillLoss, HipLayerNorm, HipScoreLogprobs, distill_loss, layer_norm, native, score_logprobs
from row_util import (U, chain, close, distill_grad_ref, distill_ref, half_step, logp_tol, norm_grad_ref, norm_tol,
                      scores_grad_ref, scores_ref, z_size)

pytestmark = pytest.mark.gpu
DEV = "cuda"
INF = math.inf
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]


def gen(seed=0):
    return torch.Generator().manual_seed(seed)


def rnd(*shape, seed=0):
    return torch.randn(shape, generator=gen(seed))


# ---- layer norm ----------------------------------------------------------------------------------------------------------

NORM_SHAPES = [(1, 1), (5, 2), (1, 8), (9, 10), (3, 33), (70, 64), (4, 100), (17, 257), (33, 512), (3, 1000), (2, 2049), (6, 4096),
               (2, 5001), (1, 16384), (2, 40003), (3, 2, 5, 24)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", NORM_SHAPES)
def test_layer_norm(shape, dtype):
    d = shape[-1]
    x = (rnd(*shape) * 0.5 + 1.5).to(dtype)
    for w, b in ((1 + 0.1 * rnd(d, seed=1), 0.1 * rnd(d, seed=2)), (rnd(d, seed=1).to(dtype), None), (None, rnd(d).to(dtype)), (None, None)):
        y, tol = norm_tol(x, w, b, 1e-5, dtype)
        got = layer_norm(x.to(DEV), None if w is None else w.to(DEV), None if b is None else b.to(DEV))
        assert got.dtype == dtype and got.is_contiguous()
        close(got, y, tol)


def norm_gradients(x, w, b, dy, dtype, got=None, eps=1e-5):
    """the kernels' dx, dw, db against the formula's"""
    if got is None:
        xd = x.to(DEV).requires_grad_(True)
        ps = [p.to(DEV).requires_grad_(True) for p in (w, b) if p is not None]
        it = iter(ps)
        y = layer_norm(xd, next(it) if w is not None else None, next(it) if b is not None else None, eps)
        got = list(torch.autograd.grad(y, [xd] + ps, dy.to(DEV)))
    (dx, dw, db), (sx, sw, sb) = norm_grad_ref(x, w, eps, dy)
    n, rows = chain(x.shape[-1]), x.numel() // x.shape[-1]
    close(got[0], dx, half_step(dtype, dx) + 2 * n * U * sx)
    r = chain(rows) + 64 + rows // 256       # rows one after the other in a chunk, then the chunks
    k = 1
    if w is not None:
        close(got[k], dw, half_step(w.dtype, dw) + (r + n) * U * sw)
        k += 1
    if b is not None:
        close(got[k], db, half_step(b.dtype, db) + r * U * sb)
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", NORM_SHAPES + [(700, 16), (3000, 130), (513, 512), (600, 2050), (300, 9001)])
def test_layer_norm_gradients(shape, dtype):
    d = shape[-1]
    x, dy = (rnd(*shape) * 0.5 + 1.5).to(dtype), rnd(*shape, seed=3).to(dtype)
    norm_gradients(x, 1 + 0.1 * rnd(d, seed=1), 0.1 * rnd(d, seed=2), dy, dtype)
    norm_gradients(x, None, None, dy, dtype)
    norm_gradients(x, rnd(d, seed=1).to(dtype), None, dy, dtype)
    norm_gradients(x, None, rnd(d, seed=1).to(dtype), dy, dtype)


@pytest.mark.parametrize("x_type", TYPES)
@pytest.mark.parametrize("w_type", TYPES)
@pytest.mark.parametrize("d", [3, 40, 1001, 20001])
def test_layer_norm_parameters_of_another_type(x_type, w_type, d):
    x, dy = (rnd(9, d) + 1).to(x_type), rnd(9, d, seed=3).to(x_type)
    w, b = (1 + 0.1 * rnd(d, seed=1)).to(w_type), (0.1 * rnd(d, seed=2)).to(w_type)
    y, tol = norm_tol(x, w, b, 1e-5, x_type)
    close(layer_norm(x.to(DEV), w.to(DEV), b.to(DEV)), y, tol)
    norm_gradients(x, w, b, dy, x_type)


def test_layer_norm_only_the_gradients_that_are_wanted():
    x, w, b = rnd(40, 48).to(DEV), rnd(48, seed=1).to(DEV), rnd(48, seed=2).to(DEV)
    full = torch.autograd.grad(layer_norm(x.requires_grad_(True), w.requires_grad_(True), b.requires_grad_(True)).sin().sum(), (x, w, b))
    for k in range(3):
        ts = [t.detach().requires_grad_(i == k) for i, t in enumerate((x, w, b))]
        g, = torch.autograd.grad(layer_norm(*ts).sin().sum(), ts[k])
        assert torch.equal(g, full[k])


@pytest.mark.parametrize("dtype", TYPES)
def test_layer_norm_takes_rows_where_they_are(dtype):
    base = (rnd(6, 5, 83) + 2).to(dtype).to(DEV)
    w, b = rnd(82, seed=1).to(DEV), rnd(82, seed=2).to(DEV)
    views = [base[..., 1:], base[:, 1:, :-1], base[::2, :, 1:], base.transpose(0, 1)[..., 1:], base[:, 2, 1:], base[2, 2, 1:],
             base[0, 0, 1:].expand(4, 82), base[..., 1:].transpose(0, 1)[1:]]
    for v in views:
        y, tol = norm_tol(v.cpu(), w.cpu(), b.cpu(), 1e-5, dtype)
        close(layer_norm(v, w, b), y, tol)
        dy = rnd(*v.shape, seed=4).to(dtype)
        leaf = v.detach().requires_grad_(True)
        norm_gradients(v.cpu(), w.cpu(), b.cpu(), dy, dtype, torch.autograd.grad(
            layer_norm(leaf, w.requires_grad_(True), b.requires_grad_(True)), (leaf, w, b), dy.to(DEV)))
    y = layer_norm(base[..., 1:].requires_grad_(True))
    y.sum().backward()                                           # an expanded upstream gradient


@pytest.mark.parametrize("dtype", TYPES)
def test_layer_norm_rows_do_not_mix(dtype):
    """constant, far off, not finite: each row for itself"""
    x = rnd(8, 200)
    x[1] = 3.25
    x[2] = 0
    x[3] += 1000 if dtype != BF16 else 60
    x[4] *= 1e-4
    x[5, 7] = math.nan
    x[6, 9] = INF
    x = x.to(dtype)
    y, tol = norm_tol(x, None, None, 1e-5, dtype)
    got = layer_norm(x.to(DEV))
    close(got[:5], y[:5], tol[:5])
    close(got[7], y[7], tol[7])
    assert got[5].isnan().all() and not got[6].isfinite().any()


def test_layer_norm_many_and_no_rows():
    x = rnd(70001, 10).to(DEV)
    y, tol = norm_tol(x.cpu(), None, None, 1e-5, F32)
    close(layer_norm(x), y, tol)
    w = torch.ones(10, device=DEV, requires_grad=True)
    e = torch.zeros(0, 10, device=DEV, requires_grad=True)
    g = torch.autograd.grad(layer_norm(e, w).sum(), (e, w))
    assert g[0].shape == (0, 10) and g[1].eq(0).all()


def test_layer_norm_gradient_against_differences():
    x, w, v = rnd(7, 40) + 1, rnd(40, seed=1), rnd(7, 40, seed=2)
    xd = x.to(DEV).requires_grad_(True)
    f = lambda a: (layer_norm(a.to(DEV), w.to(DEV)).double() * torch.arange(1., 41., device=DEV)).sum()      # noqa: E731
    g, = torch.autograd.grad((layer_norm(xd, w.to(DEV)) * torch.arange(1., 41., device=DEV)).sum(), xd)
    h = 2.0 ** -7
    diff = (f(x + h * v) - f(x - h * v)) / (2 * h)
    # both sides carry fp32 results: 16 U sum|y c| / h; the difference is off by h^2 times a third derivative (order sum |y c|)
    size = float((layer_norm(x.to(DEV), w.to(DEV)).abs() * torch.arange(1., 41., device=DEV)).sum())
    assert abs(float(diff) - float((g.double().cpu() * v).sum())) <= 16 * U * size / h + 20 * h * h * size / 40


# ---- log probabilities ---------------------------------------------------------------------------------------------------

def check_scores(x, ids, t, top, dtype=None, entropy=True):
    """forward of rows x (on the host) against the definition"""
    _, logp, ent, tl, ti = scores_ref(x, ids, t, top)
    r = score_logprobs(x.to(DEV), None if ids is None else ids.to(DEV), t, top, entropy, check_ids=False)
    if ids is not None:
        close(r.logp, logp, logp_tol(logp, x, t))
    if entropy:
        close(r.entropy, ent, 4 * logp_tol(ent.unsqueeze(-1), x, t).squeeze(-1))
    if top:
        assert torch.equal(r.top_ids.cpu(), ti)
        tl = torch.where(ti < 0, torch.where(torch.isnan(tl), tl, torch.full_like(tl, -INF)), tl)
        close(r.top_logp, tl, logp_tol(tl, x, t))
    return r


SCORE_SHAPES = [(1, 1), (3, 2), (300, 7), (5, 64), (2, 65), (4, 127), (3, 513), (2, 1000), (5, 1001), (3, 4096), (2, 5382), (2, 20011),
                (1, 131072), (1, 300007), (3, 262145), (2, 3, 50)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SCORE_SHAPES)
def test_scores(shape, dtype):
    c = shape[-1]
    x = (rnd(*shape) * 3).to(dtype)
    ids = torch.randint(0, c, shape[:-1] + (5,), generator=gen(1))
    ids[..., 1] = -1
    ids[..., 2] = c - 1
    check_scores(x, ids, 1.0, min(c, 20))
    check_scores(x, ids[..., :1].int(), 0.7, min(c, 64), entropy=False)
    check_scores(x, None, 2.0, min(c, 1))
    check_scores(x, ids, 2.0, 0, entropy=False)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_in_slices(dtype):
    """more slices than the launch has blocks; the last slice shorter than the alternatives"""
    x = (rnd(700, 20001) * 3).to(dtype)
    ids = torch.randint(0, 20001, (700, 2), generator=gen(1))
    check_scores(x, ids, 1.0, 9)
    check_scores(x[:3, :8197], ids[:3].clamp(max=8196), 0.9, 64)


def test_lists_of_no_ids():
    x = rnd(4, 30).to(DEV).requires_grad_(True)
    r = score_logprobs(x, torch.zeros(4, 0, dtype=torch.int64, device=DEV), entropy=True)
    assert r.logp.shape == (4, 0)
    g, = torch.autograd.grad((r.logp.sum(), r.entropy.sum()), x)
    want, = torch.autograd.grad(score_logprobs(x, entropy=True).entropy.sum(), x)
    assert torch.equal(g, want)


@pytest.mark.parametrize("c", [30, 3000])
def test_a_masked_answer_is_a_lesson(c):
    """alternatives that are not there come as empty slots"""
    teacher = rnd(5, c)
    teacher[1, 3:] = -INF
    teacher[2] = -INF
    told = score_logprobs(teacher.to(DEV), top_k=8)
    x = rnd(5, c, seed=1)
    check_distill(x, told.top_ids.cpu(), told.top_logp.cpu(), 1.5, torch.ones(5), F32)
    assert distill_loss(x.to(DEV), told.top_ids, told.top_logp)[2] == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("c", [11, 300, 5000, 140001])
def test_scores_masks_and_what_is_not_finite(c, dtype):
    x = (rnd(9, c) * 3).to(dtype)
    low = torch.finfo(dtype).min
    x[1, 2:c - 2] = -INF                                         # a few on offer
    x[2] = -INF                                                  # none
    x[3] = low                                                   # masks of the type's lowest value: all
    x[4, 1:] = low                                               # ... all but one
    x[5, c // 2] = math.nan
    x[6, c - 1] = INF
    x[7] = -INF
    x[7, c - 3] = 1.5                                            # one on offer
    ids = torch.stack([torch.arange(9) % c, torch.full((9,), c - 1), torch.full((9,), -1), torch.full((9,), c - 3)], 1)
    r = check_scores(x, ids, 1.0, min(c, 10))
    assert r.entropy[2] == 0 and r.entropy[7] == 0 and r.top_ids[7].tolist() == [c - 3] + [-1] * (min(c, 10) - 1)
    check_scores(x, ids, 0.5, min(c, 50))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("c", [40, 700, 9000, 200003])
def test_alternatives_with_ties(c, dtype):
    """equal scores: the lowest ids, whatever part of the row they are in"""
    few = torch.randint(0, 3, (4, c), generator=gen()).to(dtype)
    check_scores(few, None, 1.0, min(c, 33))
    check_scores(torch.zeros(2, c, dtype=dtype), None, 1.0, min(c, 64))
    z = torch.zeros(1, c, dtype=dtype)
    z[0, ::2] = -0.0
    check_scores(z, None, 1.0, min(c, 17))
    up = torch.linspace(-4, 4, c).to(dtype)
    check_scores(torch.stack([up, up.flip(0)]), None, 1.0, min(c, 40))
    one = torch.full((2, c), -2.0, dtype=dtype)                  # the best lie next to each other
    one[0, c // 2:c // 2 + 20] = torch.linspace(0, 2, 20).to(dtype)
    one[1, ::256] = 1.0
    check_scores(one, None, 1.0, min(c, 24))


@pytest.mark.parametrize("dtype", TYPES)
def test_alternatives_in_a_pattern(dtype):
    """the large scores recur at a fixed distance: a few threads meet all of them"""
    c = 300001
    n = 128 // torch.finfo(dtype).bits
    at = torch.arange(c)
    for period in (1024, 2048, 4096, 64 * n):
        x = torch.randint(-50, 0, (2, c), generator=gen()).float()
        big = (at % period) < n
        x[0, big] = torch.arange(int(big.sum())).float() % 1000 / 4
        x[1, big] = 7.0
        for top in (1, 9, 64):
            check_scores(x.to(dtype), None, 1.0, top)


def score_gradients(x, ids, t, g, gh, dtype, got):
    dx, size = scores_grad_ref(x, ids, t, g, gh)
    n = 2 * chain(x.shape[-1]) + 4 * z_size(x, t) + 16
    close(got, dx, half_step(dtype, dx) + n * U * size)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SCORE_SHAPES)
def test_score_gradients(shape, dtype):
    c = shape[-1]
    x = (rnd(*shape) * 3).to(dtype)
    ids = torch.randint(0, c, shape[:-1] + (6,), generator=gen(1))
    ids[..., 1] = -1
    ids[..., 2] = ids[..., 0]                                    # the same id twice
    ids[..., 5] = c - 1
    g, gh = rnd(*ids.shape, seed=2), rnd(*shape[:-1], seed=3)
    for t, use_g, use_h in ((1.0, True, True), (0.6, True, False), (2.0, False, True)):
        xd = x.to(DEV).requires_grad_(True)
        r = score_logprobs(xd, ids.to(DEV), t, entropy=True, check_ids=False)
        outs = [o for o, u in ((r.logp, use_g), (r.entropy, use_h)) if u]
        ups = [o.to(DEV) for o, u in ((g, use_g), (gh, use_h)) if u]
        got, = torch.autograd.grad(outs, xd, ups)
        assert got.dtype == dtype
        score_gradients(x, ids, t, g if use_g else None, gh if use_h else None, dtype, got)
    xd = x.to(DEV).requires_grad_(True)                          # one id a row, its own shape
    got, = torch.autograd.grad(score_logprobs(xd, ids[..., 0].to(DEV), 1.0, check_ids=False).logp, xd, g[..., 0].to(DEV))
    score_gradients(x, ids[..., :1], 1.0, g[..., :1], None, dtype, got)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("c", [12, 900, 20001])
def test_score_gradients_masks(c, dtype):
    x = (rnd(6, c) * 2).to(dtype)
    x[1, 3:] = -INF
    x[2] = -INF
    x[3] = torch.finfo(dtype).min
    x[4, 5] = math.nan
    ids = torch.tensor([[0, 1], [2, c - 1], [3, -1], [4, 4], [1, 2], [-1, -1]])
    g, gh = rnd(6, 2, seed=2), rnd(6, seed=3)
    xd = x.to(DEV).requires_grad_(True)
    r = score_logprobs(xd, ids.to(DEV), 1.0, entropy=True, check_ids=False)
    got, = torch.autograd.grad((r.logp, r.entropy), xd, (g.to(DEV), gh.to(DEV)))
    score_gradients(x, ids, 1.0, g, gh, dtype, got)
    assert got[2].eq(0).all() and got[4].isnan().all() and not got[[0, 1, 3, 5]].isnan().any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,c", [(70001, 2), (40007, 10), (20001, 33), (9001, 64), (6001, 100), (5003, 250), (4999, 2050), (4100, 5382)])
def test_many_rows(n, c, dtype):
    """several rows a wave, a wave a row, more rows than the launch has waves"""
    x = (rnd(n, c) * 2).to(dtype)
    x[n - 1, c // 2:] = -INF
    x[7] = -INF
    ids = torch.randint(-1, c, (n, 2), generator=gen(1))
    check_scores(x, ids, 1.0, min(c, 7))
    check_scores(x, ids[:, :1], 0.8, 0)
    xd = x.to(DEV).requires_grad_(True)
    g, gh = rnd(n, 2, seed=2), rnd(n, seed=3)
    r = score_logprobs(xd, ids.to(DEV), 1.0, entropy=True)
    got, = torch.autograd.grad((r.logp, r.entropy), xd, (g.to(DEV), gh.to(DEV)))
    score_gradients(x, ids, 1.0, g, gh, dtype, got)
    lesson_ids, ts, up = lesson((n,), c, 3)
    x[7] = 0
    check_distill(x, lesson_ids, ts, 2.0, up, dtype)


@pytest.mark.parametrize("n", [64, 65, 200, 1024])
def test_long_lists_of_ids(n):
    """every slot of a long list, most ids several times"""
    x = rnd(3, 150)
    ids = torch.randint(-1, 150, (3, n), generator=gen(1))
    g = rnd(3, n, seed=2)
    xd = x.to(DEV).requires_grad_(True)
    r = score_logprobs(xd, ids.to(DEV), check_ids=False)
    _, logp, _, _, _ = scores_ref(x, ids, 1.0, 1)
    close(r.logp, logp, logp_tol(logp, x, 1.0))
    got, = torch.autograd.grad(r.logp, xd, g.to(DEV))
    dx, size = scores_grad_ref(x, ids, 1.0, g, None)
    close(got, dx, half_step(F32, dx) + (n + 2 * chain(150) + 4 * z_size(x, 1.0)) * U * size)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,c", [(5, 1500), (9000, 600), (7, 6001), (3, 50001)])
@pytest.mark.parametrize("n", [63, 65, 129, 1000, 1024])
def test_long_lists_of_ids_on_longer_rows(n, rows, c, dtype):
    """ids that are alone, several times, everywhere or nowhere in the list; the same bits again"""
    rows = rows if n < 1000 else min(rows, 40)
    x = rnd(rows, c).to(dtype)
    ids = torch.randint(-1, c, (rows, n), generator=gen(1))
    ids[1, ::2] = c - 1
    ids[2] = 7
    ids[-1, :n // 2] = torch.arange(n // 2) * 5 % c              # neighbours in the list are neighbours in the row
    if rows > 3:
        ids[3] = -1
        ids[4] = torch.randint(0, 9, (n,), generator=gen(4))
    g = rnd(rows, n, seed=2)
    xd = x.to(DEV).requires_grad_(True)
    logp = score_logprobs(xd, ids.to(DEV), check_ids=False).logp
    got, = torch.autograd.grad(logp, xd, g.to(DEV), retain_graph=True)
    dx, size = scores_grad_ref(x, ids, 1.0, g, None)
    close(got, dx, half_step(dtype, dx) + (n + 2 * chain(c) + 4 * z_size(x, 1.0)) * U * size)
    for _ in range(3):
        again, = torch.autograd.grad(logp, xd, g.to(DEV), retain_graph=True)
        assert torch.equal(again, got)


@pytest.mark.parametrize("dtype", TYPES)
def test_scores_take_rows_where_they_are(dtype):
    base = (rnd(4, 5, 301) * 2).to(dtype).to(DEV)
    for v in (base[..., 1:], base[:, 1:, :-1], base[:, :-1], base.transpose(0, 1)[..., 3:], base[1, 2, 1:], base[0, :1, 1:].expand(3, 300),
              base[..., ::2], base.transpose(1, 2)):
        c = v.shape[-1]
        ids = torch.randint(0, c, v.shape[:-1], generator=gen(1))
        r = score_logprobs(v, ids.to(DEV), 1.0, 3, True)
        vc = v.cpu().contiguous()
        _, logp, ent, _, ti = scores_ref(vc, ids.unsqueeze(-1), 1.0, 3)
        assert r.logp.shape == ids.shape
        close(r.logp.unsqueeze(-1), logp, logp_tol(logp, vc, 1.0))
        close(r.entropy, ent, 4 * logp_tol(ent.unsqueeze(-1), vc, 1.0).squeeze(-1))
        assert torch.equal(r.top_ids.cpu(), ti)
        leaf = v.detach().requires_grad_(True)
        g = rnd(*ids.shape, seed=5)
        got, = torch.autograd.grad(score_logprobs(leaf, ids.to(DEV)).logp, leaf, g.to(DEV))
        score_gradients(vc, ids.unsqueeze(-1), 1.0, g.unsqueeze(-1), None, dtype, got)


def test_extreme_temperatures():
    x = rnd(4, 50)
    ids = torch.randint(0, 50, (4, 2), generator=gen(1))
    for t in (1e-6, 1e-3, 1e3, 1e6):
        check_scores(x, ids, t, 5)


# ---- distillation --------------------------------------------------------------------------------------------------------

def lesson(lead, c, k, seed=0):
    ids = torch.randint(0, c, lead + (k,), generator=gen(seed + 1))
    length = torch.randint(0, k + 1, lead + (1,), generator=gen(seed + 2))
    ids = torch.where(torch.arange(k) < length, ids, torch.full_like(ids, -1))
    return ids, rnd(*lead, k, seed=seed + 3) * 2 + 4, torch.rand(lead, generator=gen(seed + 4))


def check_distill(x, ids, ts, t, g, dtype):
    xd = x.to(DEV).requires_grad_(True)
    loss = distill_loss(xd, ids.to(DEV), ts.to(DEV), t, check_ids=False)
    ref, size = distill_ref(x, ids, ts, t)
    n = chain(x.shape[-1]) + chain(ids.shape[-1]) + ids.shape[-1] + z_size(x, t).squeeze(-1) + z_size(ts, t).squeeze(-1) + 16
    assert loss.dtype == F32
    close(loss, ref, n * U * size + 1e-30)
    got, = torch.autograd.grad(loss, xd, g.to(DEV))
    dx, size = distill_grad_ref(x, ids, ts, t, g)
    close(got, dx, half_step(dtype, dx) + 2 * n.unsqueeze(-1) * U * size)
    assert got.dtype == dtype
    with torch.no_grad():
        assert torch.equal(distill_loss(xd, ids.to(DEV), ts.to(DEV), t, check_ids=False), loss)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,k", [((1, 1), 1), ((3, 2), 4), ((200, 7), 3), ((5, 64), 64), ((4, 127), 5), ((3, 1001), 100),
                                     ((2, 5382), 16), ((2, 20011), 1024), ((1, 300007), 64), ((3, 262145), 7), ((2, 3, 50), 9)])
def test_distillation(shape, k, dtype):
    x = (rnd(*shape) * 2).to(dtype)
    ids, ts, g = lesson(shape[:-1], shape[-1], k)
    for t, tt in ((1.0, F32), (3.0, BF16), (0.5, F16)):
        check_distill(x, ids, ts.to(tt), t, g, dtype)
    check_distill(x, ids.int(), ts, 1.0, g, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("c", [9, 700, 30001])
def test_distillation_edges(c, dtype):
    x = (rnd(7, c)).to(dtype)
    x[1, 3:] = -INF
    x[2] = -INF
    x[4] = torch.finfo(dtype).min
    ids = torch.tensor([[0, 0, 0], [1, 2, -1], [3, 4, -1], [-1, -1, -1], [5, 6, 7], [1, 2, 3], [8, 8, 2]])
    ts = rnd(7, 3, seed=1)
    ts[5] = -INF                                                 # listed, but without weight
    ts[6, 1] = -INF
    g = torch.rand(7, generator=gen(2)) + 0.5
    xd = x.to(DEV).requires_grad_(True)
    loss = distill_loss(xd, ids.to(DEV), ts.to(DEV), 2.0)
    got, = torch.autograd.grad(loss, xd, g.to(DEV))
    assert loss[2] == INF and loss[3] == 0 and loss[5] == 0
    assert got[2].eq(0).all() and got[3].eq(0).all() and got[5].eq(0).all()
    keep = [0, 1, 3, 4, 5, 6]
    check_distill(x[keep], ids[keep], ts[keep], 2.0, g[keep], dtype)
    x[0, 1] = math.nan
    ts[1, 0] = math.nan
    xd = x.to(DEV).requires_grad_(True)
    loss = distill_loss(xd, ids.to(DEV), ts.to(DEV), 2.0)
    got, = torch.autograd.grad(loss, xd, g.to(DEV))
    assert loss.isnan().tolist() == [True, True] + [False] * 5 and got[:2].isnan().all() and not got[2:].isnan().any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("c", [9, 40, 700, 5382, 40003])
@pytest.mark.parametrize("device", ["cpu", DEV])
def test_padding_has_gradient_zero(c, dtype, device):
    """rows that nothing is asked of may hold anything"""
    x = rnd(6, c).to(dtype)
    x[3] = math.nan
    x[4, 1] = INF
    x[5] = torch.finfo(dtype).max
    ids = torch.tensor([[0, 1], [2, -1], [c - 1, 0], [-1, -1], [-1, -2], [-5, -1]], device=device)
    ts = rnd(6, 2, seed=1).to(device)
    xd = x.to(device).requires_grad_(True)
    up = torch.tensor([1.0, 2.0, 0.5, 0.0, 0.0, 0.0], device=device)
    r = score_logprobs(xd, ids, entropy=True)
    for outs, ups in (((r.logp,), (torch.ones(6, 2, device=device),)), ((r.logp, r.entropy), (torch.ones(6, 2, device=device), up))):
        got, = torch.autograd.grad(outs, xd, ups, retain_graph=True)
        assert got[3:].eq(0).all() and got[:3].isfinite().all() and got[:3].ne(0).any(-1).all()
    loss = distill_loss(xd, ids, ts, 1.5)
    got, = torch.autograd.grad(loss, xd, torch.ones(6, device=device))
    assert loss[3:].eq(0).all() and got[3:].eq(0).all() and got[:3].isfinite().all() and got[:3].ne(0).any(-1).all()


def test_distillation_takes_rows_where_they_are():
    base = rnd(4, 6, 120).to(DEV)
    for v in (base[:, 1:, 3:], base.transpose(0, 1), base[1, 0, 1:]):
        ids, ts, g = lesson(v.shape[:-1], v.shape[-1], 6)
        leaf = v.detach().requires_grad_(True)
        loss = distill_loss(leaf, ids.to(DEV), ts.to(DEV), 1.5)
        got, = torch.autograd.grad(loss, leaf, g.to(DEV))
        same = v.contiguous().requires_grad_(True)
        want = distill_loss(same, ids.to(DEV), ts.to(DEV), 1.5)
        assert torch.equal(loss, want) and torch.equal(got, torch.autograd.grad(want, same, g.to(DEV))[0])


def test_gradients_against_differences():
    """a directional derivative of the kernels' own forward; fp32 results: 2^-24 of the loss over the step, and the step squared"""
    x, v = rnd(6, 90) * 2, rnd(6, 90, seed=7)
    ids, ts, _ = lesson((6,), 90, 8)
    pick = torch.randint(0, 90, (6, 3), generator=gen(9))

    def f(a):
        a = a.to(DEV)
        r = score_logprobs(a, pick.to(DEV), 1.3, entropy=True)
        return distill_loss(a, ids.to(DEV), ts.to(DEV), 1.3).double().sum() + r.logp.double().sum() + r.entropy.double().sum()

    xd = x.to(DEV).requires_grad_(True)
    r = score_logprobs(xd, pick.to(DEV), 1.3, entropy=True)
    g, = torch.autograd.grad(distill_loss(xd, ids.to(DEV), ts.to(DEV), 1.3).sum() + r.logp.sum() + r.entropy.sum(), xd)
    h = 2.0 ** -8
    size = float(r.logp.abs().sum() + r.entropy.sum()) + float(distill_ref(x, ids, ts, 1.3)[1].sum())
    diff = float((f(x + h * v) - f(x - h * v)) / (2 * h))
    assert abs(diff - float((g.double().cpu() * v).sum())) <= 64 * U * size / h + 10 * h * h * size


# ---- reports, streams, graphs, large tensors -----------------------------------------------------------------------------

def test_an_id_past_the_row_is_an_index_error():
    x, ids = rnd(4, 10).to(DEV), torch.tensor([[0], [10], [3], [2]], device=DEV)
    for call in (lambda: score_logprobs(x, ids), lambda: distill_loss(x, ids, torch.zeros(4, 1, device=DEV))):
        with pytest.raises(IndexError):
            call()
    m = HipScoreLogprobs(top_k=2)
    r = m(x, ids)
    with pytest.raises(IndexError):
        m.poll()
    assert r.logp.isnan().flatten().tolist() == [False, True, False, False]
    m(x, ids)
    torch.cuda.synchronize()
    with pytest.raises(IndexError):                              # deferred: at the next call
        m(x, ids.clamp(max=9))
    m(x, ids.clamp(max=9))
    m.poll()
    d = HipDistillLoss()
    d(x, ids, torch.zeros(4, 1, device=DEV))
    with pytest.raises(IndexError):
        d.poll()
    # its gradient leaves the other rows alone
    xd = x.clone().requires_grad_(True)
    g, = torch.autograd.grad(score_logprobs(xd, ids, check_ids=False).logp.nan_to_num().sum(), xd)
    close(g[[0, 2, 3]], scores_grad_ref(x.cpu()[[0, 2, 3]], ids.cpu()[[0, 2, 3]], 1.0, torch.ones(3, 1), None)[0], 1e-5)


def test_mixed_places_are_refused():
    x, ids = rnd(3, 8).to(DEV), torch.zeros(3, 2, dtype=torch.int64)
    for call in (lambda: score_logprobs(x, ids), lambda: distill_loss(x, ids.to(DEV), torch.zeros(3, 2)),
                 lambda: layer_norm(x, torch.ones(8)), lambda: layer_norm(x.double()), lambda: score_logprobs(x.double())):
        with pytest.raises(native.ArmnetNativeError):
            call()


def test_the_same_bits_every_time():
    x = rnd(2000, 333).to(DEV).requires_grad_(True)
    w, b = rnd(333, seed=1).to(DEV).requires_grad_(True), rnd(333, seed=2).to(DEV).requires_grad_(True)
    big = (rnd(2, 200001) * 3).to(DEV).requires_grad_(True)
    ids, ts, _ = lesson((2,), 200001, 40)

    def once():
        y = layer_norm(x, w, b)
        r = score_logprobs(big, ids.to(DEV), 1.0, 30, True)
        loss = distill_loss(big, ids.to(DEV), ts.to(DEV))
        return [y, *r, loss, *torch.autograd.grad((y.sin().sum(), r.entropy.sum(), r.logp.sum(), loss.sum()), (x, w, b, big))]

    first = once()
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(first, once()))


def test_on_another_stream():
    x = rnd(64, 4096).to(DEV).requires_grad_(True)
    w = torch.ones(4096, device=DEV, requires_grad=True)
    ids = torch.randint(0, 4096, (64, 3), generator=gen()).to(DEV)

    def chain_of(x):
        y = layer_norm(x, w)
        r = score_logprobs(y, ids, 1.0, 4, True)
        loss = distill_loss(y, r.top_ids, r.top_logp.detach() * 0.5)
        return [r.logp, r.entropy, r.top_ids, loss, *torch.autograd.grad((r.logp.sum(), loss.sum()), (x, w))]

    want = chain_of(x)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = chain_of(x)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("c", [500, 150001])
def test_captured_and_replayed(c):
    """forward and gradients in one graph; replays on new inputs, eager work between them"""
    n, k = 6, 9
    x = rnd(n, c).to(DEV).requires_grad_(True)
    w = torch.ones(c, device=DEV, requires_grad=True)
    ids, ts, _ = lesson((n,), c, k)
    ids, ts = ids.to(DEV), ts.to(DEV)
    scores, distill = HipScoreLogprobs(1.2, 5, True), HipDistillLoss(2.0, "none")

    def step():
        y = layer_norm(x, w)
        r = scores(y, ids)
        loss = distill(y, ids, ts)
        return [y, *r, loss, *torch.autograd.grad((r.logp.sum(), r.entropy.sum(), loss.sum()), (x, w))]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()                                                   # the report's word exists before the capture
    torch.cuda.current_stream().wait_stream(s)
    graphs = []
    for _ in range(2):                                           # two graphs: each has a workspace of its own
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    for i in range(4):
        with torch.no_grad():
            x.copy_(rnd(n, c, seed=20 + i))
        want = [t.clone() for t in step()]
        for g, out in graphs:
            for t in out:
                t.detach().zero_() if t.is_floating_point() else t.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))
    scores.poll(), distill.poll()


def test_rows_past_32_bits():
    """element offsets beyond 2^32: the last rows of a large tensor and of a view with a large stride"""
    c = 1 << 20
    n = 4100                                                     # 4.3e9 elements
    x = torch.zeros(n, c, device=DEV, dtype=BF16)
    rows = [0, 2047, 2048, 4095, 4096, n - 1]
    x[rows] = (rnd(len(rows), c) * 2).to(BF16).to(DEV)
    ids = torch.randint(0, c, (n, 1), generator=gen(1))
    x.requires_grad_(True)
    r = score_logprobs(x, ids.to(DEV), 1.0, 3, True)
    part = x.detach()[rows].cpu()
    _, logp, ent, _, ti = scores_ref(part, ids[rows], 1.0, 3)
    close(r.logp[rows], logp, logp_tol(logp, part, 1.0))
    assert torch.equal(r.top_ids[rows].cpu(), ti)
    assert r.top_ids[1].tolist() == [0, 1, 2] and abs(float(r.entropy[1]) - math.log(c)) < 1e-4
    g, = torch.autograd.grad(r.logp, x, torch.ones(n, 1, device=DEV))
    score_gradients(part, ids[rows], 1.0, torch.ones(len(rows), 1), None, BF16, g[rows])
    del g
    y = layer_norm(x.detach())
    ref, tol = norm_tol(part, None, None, 1e-5, BF16)
    close(y[rows], ref, tol)
    del y
    v = x.detach().view(2, n // 2, c)[:, :3, 5:]                 # rows 2e9 elements apart
    ref, tol = norm_tol(v.cpu(), None, None, 1e-5, BF16)
    close(layer_norm(v), ref, tol)


def test_two_devices():
    if torch.cuda.device_count() < 2:
        pytest.skip("one GPU")
    x = rnd(3, 100).to("cuda:1")
    y, tol = norm_tol(x.cpu(), None, None, 1e-5, F32)
    close(layer_norm(x), y, tol)
    check = score_logprobs(x, torch.zeros(3, dtype=torch.int64, device="cuda:1"), top_k=2)
    assert check.top_ids.device == x.device


# ---- together ------------------------------------------------------------------------------------------------------------

def test_norm_projection_scores_and_distillation_together():
    """a block's neurons -> layer norm -> projection -> scores; a teacher's best ids teach a student; serving gives log p"""
    from models.armnet_1h import ARMNetModel
    torch.manual_seed(3)
    F, E, H, nfeat, B, C, K = 10, 8, 6, 500, 33, 77, 12
    block = ARMNetModel(F, nfeat, E, 1.7, H, E, 1, 16, 0.0, False, 1, 16).eval().cuda()
    ids, vals = torch.randint(0, nfeat, (B, F), device=DEV), torch.rand(B, F, device=DEV)
    with torch.no_grad():
        feat = block.arm_block(ids, vals).reshape(B, H * E)
    norm, teacher, student = HipLayerNorm(H * E).cuda(), torch.nn.Linear(H * E, C).cuda(), torch.nn.Linear(H * E, C).cuda()
    scores, loss_fn = HipScoreLogprobs(top_k=K, entropy=True), HipDistillLoss(temperature=2.0)
    with torch.no_grad():
        told = scores(teacher(norm(feat)) * 4)
    loss = loss_fn(student(norm(feat)), told.top_ids, told.top_logp)
    loss.backward()
    scores.poll(), loss_fn.poll()
    # the same in 64 bits
    f, wt, bt = feat.cpu().double(), teacher.weight.detach().cpu().double(), teacher.bias.detach().cpu().double()
    ws, bs = (p.detach().cpu().double().requires_grad_(True) for p in (student.weight, student.bias))
    gamma, beta = (p.detach().cpu().double().requires_grad_(True) for p in (norm.weight, norm.bias))
    h = (f - f.mean(1, keepdim=True)) / torch.sqrt(f.var(1, unbiased=False, keepdim=True) + norm.eps)
    n = h * gamma + beta
    lt = torch.log_softmax((n.detach() @ wt.t() + bt) * 4, 1)
    best = torch.sort(lt, dim=1, descending=True, stable=True)
    assert torch.equal(told.top_ids.cpu(), best.indices[:, :K])
    torch.testing.assert_close(told.top_logp.cpu().double(), best.values[:, :K], rtol=1e-4, atol=1e-4)
    q = torch.softmax(best.values[:, :K] / 2, 1)
    lp = torch.log_softmax((n @ ws.t() + bs) / 2, 1).gather(1, best.indices[:, :K])
    want = (4 * (q * (q.log() - lp)).sum(1)).mean()
    want.backward()
    torch.testing.assert_close(loss.detach().cpu().double(), want.detach(), rtol=1e-5, atol=1e-6)
    for got, ref in ((student.weight.grad, ws.grad), (student.bias.grad, bs.grad), (norm.weight.grad, gamma.grad), (norm.bias.grad, beta.grad)):
        torch.testing.assert_close(got.cpu().double(), ref, rtol=1e-4, atol=1e-5 * float(ref.abs().max()))


def test_saved_tensors_that_were_moved():
    """hooks that keep the saved tensors elsewhere: the backward takes them where they come back, dense"""
    base = rnd(12, 300).to(DEV)
    x = base[:, 3:].detach().requires_grad_(True)                # a view with a stride of its own
    w = rnd(297, seed=1).to(DEV).requires_grad_(True)
    ids, ts, _ = lesson((12,), 297, 5)
    ids, ts = ids.to(DEV), ts.to(DEV)

    def grads(out):
        return torch.autograd.grad(out, (x, w), torch.ones_like(out), allow_unused=True)

    calls = [lambda: layer_norm(x, w), lambda: score_logprobs(x, ids, 1.3, entropy=True).logp,
             lambda: score_logprobs(x, entropy=True).entropy, lambda: distill_loss(x, ids, ts, 2.0)]
    for call in calls:
        want = grads(call())
        with torch.autograd.graph.save_on_cpu():
            moved = call()
        junk = [torch.full_like(base, 7.0) for _ in range(3)]    # whatever freed memory is taken again
        got = grads(moved)
        del junk
        for a, b in zip(got, want):
            assert (a is None) == (b is None) and (a is None or torch.equal(a, b))


def test_second_backward_of_one_graph():
    x = rnd(9, 200).to(DEV).requires_grad_(True)
    ids, ts, g = lesson((9,), 200, 4)
    loss = distill_loss(x, ids.to(DEV), ts.to(DEV))
    a, = torch.autograd.grad(loss, x, g.to(DEV), retain_graph=True)
    b, = torch.autograd.grad(loss, x, 2 * g.to(DEV))
    assert torch.equal(2 * a, b)
    y = layer_norm(x)
    first, = torch.autograd.grad(y, x, torch.ones_like(y), create_graph=True)
    with pytest.raises(RuntimeError):
        first.sum().backward()                                   # differentiable once
    with torch.no_grad():
        x.add_(1)
    with pytest.raises(RuntimeError, match="modified"):
        y2 = layer_norm(x)
        with torch.no_grad():
            x.add_(1)
        y2.sum().backward()
