"""The row operators' kernels over more rows than a launch has places for: every group goes on to further rows, with its registers and
its LDS as the row before left them.  Row counts go by the device's compute units (the launches do), and the last round is ragged.
What a row says is also compared with a call of its own, bit for bit: it must not depend on which rows came before."""
import math

import pytest
import torch

from armnet_hip import distill_loss, layer_norm, score_logprobs
from row_util import (U, chain, close, distill_grad_ref, distill_ref, half_step, logp_tol, norm_grad_ref, norm_tol, scores_grad_ref,
                      scores_ref, z_size)

pytestmark = pytest.mark.gpu
DEV = "cuda"
INF = math.inf
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]


def rows_of(per_cu, more=7):
    return int(torch.cuda.get_device_properties(0).multi_processor_count * per_cu) + more


def rnd(*shape, seed=0):
    return torch.randn(shape, generator=torch.Generator(DEV).manual_seed(seed), device=DEV)


def ids_of(n, k, c, seed=1, low=-1):
    return torch.randint(low, c, (n, k), generator=torch.Generator(DEV).manual_seed(seed), device=DEV)


# rows a compute unit takes at once, forward: 512 of 10 values, 32 or 64 of 130, 32 of 512, 8 or 32 of 1000, 4 or 8 of 2049, 2 or 4 of
# 4100, 2 of 9001; backward: 256 of 10 values and fewer of longer rows
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("per_cu,d", [(547, 10), (547, 3), (79, 130), (36, 512), (36, 1000), (10, 2049), (5, 4100), (3, 9001)])
def test_layer_norm(per_cu, d, dtype):
    n = rows_of(per_cu)
    x, dy = (rnd(n, d) * 0.5 + 1.5).to(dtype), rnd(n, d, seed=3).to(dtype)
    w, b = 1 + 0.1 * rnd(d, seed=1), 0.1 * rnd(d, seed=2)
    x.requires_grad_(True), w.requires_grad_(True), b.requires_grad_(True)
    y = layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    with torch.no_grad():
        ref, tol = norm_tol(x, w, b, 1e-5, dtype)
        close(y, ref, tol)
        (rx, rw, rb), (sx, sw, sb) = norm_grad_ref(x, w, 1e-5, dy)
        m, r = chain(d), chain(n) + 64 + n // 256                # rows one after the other in a chunk, then the chunks
        close(dx, rx, half_step(dtype, rx) + 2 * m * U * sx)
        close(dw, rw, half_step(F32, rw) + (r + m) * U * sw)
        close(db, rb, half_step(F32, rb) + r * U * sb)
    for part in (slice(0, 9), slice(n - 9, n), slice(n // 2, n // 2 + 9)):
        xs = x[part].detach().requires_grad_(True)
        ys = layer_norm(xs, w, b)
        assert torch.equal(ys, y[part]) and torch.equal(torch.autograd.grad(ys, xs, dy[part])[0], dx[part])


def check(x, k, t, top, dtype, own=True):
    """rows x [n, c] (on the device): what they say, its gradient, the loss and its gradient"""
    n, c = x.shape
    x[n - 1, c // 2:] = -INF
    x[n // 3] = -INF
    ids = ids_of(n, k, c)
    g, gh = rnd(n, k, seed=2), rnd(n, seed=3)
    xd = x.detach().requires_grad_(True)
    r = score_logprobs(xd, ids, t, top, True)
    dx, = torch.autograd.grad((r.logp, r.entropy), xd, (g, gh))
    plain = score_logprobs(x, ids, t, 0, False).logp             # other kernels where alternatives have their own
    lengths = torch.arange(k, device=DEV) < torch.randint(0, k + 1, (n, 1), generator=torch.Generator(DEV).manual_seed(4), device=DEV)
    listed = torch.where(lengths, ids.clamp(min=0), torch.full_like(ids, -1))
    ts, up = rnd(n, k, seed=5) * 2 + 4, rnd(n, seed=6).abs()
    x2 = x.clone()
    x2[n // 3] = 0
    xe = x2.requires_grad_(True)
    live = torch.where(torch.arange(n, device=DEV) == n - 1, torch.zeros(1, device=DEV), up)    # (a masked id has loss +inf)
    listed[n - 1] = -1
    loss = distill_loss(xe, listed, ts, t)
    de, = torch.autograd.grad(loss, xe, live)
    step = max(1, (1 << 25) // c)                                # the definition, some rows at a time
    for i in range(0, n, step):
        s = slice(i, min(n, i + step))
        xs = x[s]
        _, logp, ent, tl, ti = scores_ref(xs, ids[s], t, max(top, 1))
        close(r.logp[s], logp, logp_tol(logp, xs, t))
        close(plain[s], logp, logp_tol(logp, xs, t))
        close(r.entropy[s], ent, 4 * logp_tol(ent.unsqueeze(-1), xs, t).squeeze(-1))
        if top:
            assert torch.equal(r.top_ids[s], ti)
            close(r.top_logp[s], torch.where(ti < 0, torch.full_like(tl, -INF), tl), logp_tol(tl, xs, t))
        ref, size = scores_grad_ref(xs, ids[s], t, g[s], gh[s])
        close(dx[s], ref, half_step(dtype, ref) + (2 * chain(c) + 4 * z_size(xs, t) + 16 + k) * U * size)
        xs = x2.detach()[s]
        ref, size = distill_ref(xs, listed[s], ts[s], t)
        m = chain(c) + chain(k) + k + z_size(xs, t).squeeze(-1) + z_size(ts[s], t).squeeze(-1) + 16
        close(loss[s], ref, m * U * size + 1e-30)
        ref, size = distill_grad_ref(xs, listed[s], ts[s], t, live[s])
        close(de[s], ref, half_step(dtype, ref) + 2 * m.unsqueeze(-1) * U * size)


# rows a compute unit takes at once: 512 (of up to 16 or 32 scores), 256 or 128 (up to 64), 128 (up to 256 or 512)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("per_cu,c,top", [(547, 7, 0), (547, 7, 2), (547, 7, 6), (547, 3, 3), (300, 33, 4), (300, 64, 8), (300, 64, 50),
                                          (157, 100, 5), (157, 250, 4), (157, 250, 0)])
def test_short_rows(per_cu, c, top, dtype):
    check((rnd(rows_of(per_cu), c) * 2).to(dtype), 3, 1.0, top, dtype)


# a wave a row: 32 rows (24 with alternatives); a block a row: 8 (6); rows in slices: as many slices
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("per_cu,c,top,k", [(36, 1001, 20, 3), (36, 1001, 0, 70), (36, 600, 64, 2), (36, 5382, 9, 5), (10, 5382, 20, 3),
                                            (10, 5382, 0, 100), (2.9, 30001, 0, 4), (3.3, 65537, 20, 2)])
def test_long_rows(per_cu, c, top, k, dtype):
    check((rnd(rows_of(per_cu), c) * 2).to(dtype), k, 1.3, top, dtype)


@pytest.mark.parametrize("n,c,k", [((1 << 22) + 1001, 520, 70), ((1 << 20) + 501, 2050, 3)])
def test_gradients_of_more_rows_than_a_launch_has_blocks(n, c, k):
    """a wave, and a block a row: the list and its table in LDS again and again"""
    x = torch.empty(n, c, device=DEV, dtype=BF16)
    for i in range(0, n, 1 << 19):
        x[i:i + (1 << 19)] = (rnd(min(1 << 19, n - i), c, seed=i) * 2).to(BF16)
    ids = ids_of(n, k, c)
    ids[::3, 1] = ids[::3, 0]
    g = rnd(n, k, seed=2)
    xd = x.requires_grad_(True)
    logp = score_logprobs(xd, ids).logp
    got, = torch.autograd.grad(logp, xd, g)
    for i in range(0, n, 1 << 19):                               # calls that fit a launch
        s = slice(i, min(n, i + (1 << 19)))
        xs = x.detach()[s].requires_grad_(True)
        part = score_logprobs(xs, ids[s]).logp
        if s.stop - i >= 4096:                                   # (fewer rows have kernels of their own, which sum in another order)
            assert torch.equal(part, logp[s]) and torch.equal(torch.autograd.grad(part, xs, g[s])[0], got[s])
    for s in (slice(0, 300), slice((1 << 20) - 150, (1 << 20) + 150), slice(n - 300, n)):
        xs = x.detach()[s]
        ref = scores_ref(xs, ids[s], 1.0, 1)[1]
        close(logp[s], ref, logp_tol(ref, xs, 1.0))
        ref, size = scores_grad_ref(xs, ids[s], 1.0, g[s], None)
        close(got[s], ref, half_step(BF16, ref) + (2 * chain(c) + 4 * z_size(xs, 1.0) + 16 + k) * U * size)
