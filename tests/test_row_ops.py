"""Row operators on host tensors, their refusals and the C entries' argument checks (no GPU)."""
import copy
import math

import pytest
import torch

from armnet_hip import HipDistillLoss, HipLayerNorm, HipScoreLogprobs, distill_loss, layer_norm, native, score_logprobs
from row_util import close, declare_row_calls, distill_ref, logp_tol, norm_tol, scores_ref

Error = native.ArmnetNativeError
INF = math.inf


def gen(seed=0):
    return torch.Generator().manual_seed(seed)


# ---- host formulas -------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(1, 1), (3, 2), (5, 33), (2, 3, 17)])
def test_layer_norm_on_host(dtype, shape):
    x = (torch.randn(shape, generator=gen()) + 3).to(dtype)
    w, b = torch.randn(shape[-1], generator=gen(1)), torch.randn(shape[-1], generator=gen(2))
    for ww, bb in ((w, b), (w, None), (None, b), (None, None)):
        y, tol = norm_tol(x, ww, bb, 1e-5, dtype)
        close(layer_norm(x, ww, bb), y, tol)


def test_layer_norm_gradients_on_host():
    x = torch.randn(4, 7, generator=gen(), dtype=torch.float64, requires_grad=True)
    w = torch.randn(7, generator=gen(1), dtype=torch.float64, requires_grad=True)
    b = torch.randn(7, generator=gen(2), dtype=torch.float64, requires_grad=True)
    assert torch.autograd.gradcheck(lambda *a: layer_norm(*a), (x, w, b))
    assert torch.autograd.gradcheck(lambda a: layer_norm(a), (x,))
    assert torch.autograd.gradcheck(lambda a, c: layer_norm(a, None, c), (x, b))


def test_layer_norm_module():
    for shape in (6, (3, 5)):
        a, b = HipLayerNorm(shape), torch.nn.LayerNorm(shape)
        assert list(a.state_dict()) == list(b.state_dict())
        with torch.no_grad():
            for p in a.parameters():
                p.normal_(generator=gen())
        b.load_state_dict(a.state_dict())
        x = torch.randn(4, *a.normalized_shape, generator=gen(3))
        k = len(a.normalized_shape)
        y, tol = norm_tol(x.flatten(-k), b.weight.flatten(), b.bias.flatten(), 1e-5, torch.float32)
        close(a(x).flatten(-k), y, tol)
        with pytest.raises(Error, match="ends in"):
            a(torch.zeros(4, 7))
    assert HipLayerNorm(6, elementwise_affine=False)(torch.ones(2, 6)).eq(0).all()


def masked_rows():
    x = torch.randn(7, 11, generator=gen()) * 3
    x[1, 2:9] = -INF
    x[2] = -INF
    x[3] = torch.finfo(torch.float32).min
    x[4, 1:] = torch.finfo(torch.float32).min
    x[5, 3] = math.nan
    x[6, 4] = INF
    ids = torch.tensor([[0, 10, 5], [0, 2, -1], [3, -1, 3], [1, 1, 2], [0, 1, 2], [0, 3, -1], [4, 0, -7]])
    return x, ids


@pytest.mark.parametrize("t", [1.0, 0.3, 4.0])
def test_scores_on_host(t):
    x, ids = masked_rows()
    r = score_logprobs(x, ids, t, top_k=5, entropy=True)
    _, logp, ent, tl, ti = scores_ref(x, ids, t, 5)
    close(r.logp, logp, logp_tol(logp, x, t))
    close(r.entropy, ent, 4 * logp_tol(ent.unsqueeze(-1), x, t).squeeze(-1))
    close(r.top_logp, tl, logp_tol(tl, x, t))
    assert torch.equal(r.top_ids, ti)
    assert r.entropy[2] == 0 and r.logp[2, 0] == -INF and r.logp[2, 1] == 0
    assert abs(float(r.entropy[3]) - math.log(11)) < 1e-5


def test_score_gradients_on_host():
    x = torch.randn(3, 6, generator=gen(), dtype=torch.float64)
    x = x.requires_grad_(True)
    ids = torch.tensor([[0, 0, 5], [-1, 2, 2], [-1, -1, -1]])
    assert torch.autograd.gradcheck(lambda a: score_logprobs(a, ids, 0.7, entropy=True)[:2], (x,))
    assert torch.autograd.gradcheck(lambda a: score_logprobs(a, ids[:, 0], 2.0).logp, (x,))
    assert torch.autograd.gradcheck(lambda a: score_logprobs(a, entropy=True).entropy, (x,))
    r = score_logprobs(x, ids, top_k=2)
    assert r.logp.requires_grad and not r.top_logp.requires_grad and not r.top_ids.requires_grad


def test_distill_on_host():
    x = torch.randn(4, 9, generator=gen())
    ids = torch.tensor([[0, 3, 8], [2, 2, -1], [-1, -1, -1], [1, -1, 5]])
    ts = torch.randn(4, 3, generator=gen(1))
    ts[3, 2] = -INF
    for t in (1.0, 3.0):
        ref, size = distill_ref(x, ids, ts, t)
        close(distill_loss(x, ids, ts, t), ref, 64 * 2.0 ** -24 * (size + 1))
    assert distill_loss(x, ids, ts)[2] == 0
    xd = x.double().requires_grad_(True)
    assert torch.autograd.gradcheck(lambda a: distill_loss(a, ids, ts.double(), 2.0), (xd,))
    loss = distill_loss(torch.full((1, 9), -INF, requires_grad=True), ids[:1], ts[:1])
    assert loss.item() == INF
    for reduction in ("mean", "sum"):
        got = HipDistillLoss(2.0, reduction)(x, ids, ts)
        torch.testing.assert_close(got, getattr(distill_loss(x, ids, ts, 2.0), reduction)())


def test_a_teachers_answer_is_a_students_lesson_on_host():
    """the teacher's logp differ from its scores by a constant per row: the same q"""
    teacher, x = torch.randn(5, 20, generator=gen()), torch.randn(5, 20, generator=gen(1))
    r = score_logprobs(teacher, top_k=6)
    raw = teacher.gather(-1, r.top_ids)
    for t in (1.0, 2.5):
        a, b = distill_loss(x, r.top_ids, r.top_logp, t), distill_loss(x, r.top_ids, raw, t)
        close(a, b, 64 * 2.0 ** -24 * (distill_ref(x, r.top_ids, raw, t)[1] + 1))


# ---- refusals ------------------------------------------------------------------------------------------------------------

def test_layer_norm_refuses():
    x = torch.zeros(2, 4)
    for bad, word in ((dict(x=torch.zeros(2, 4, dtype=torch.int64)), "float32"), (dict(x=torch.tensor(1.0)), "rows"),
                      (dict(x=torch.zeros(2, 0)), "rows"), (dict(x=x, weight=torch.zeros(3)), "weight"),
                      (dict(x=x, weight=torch.zeros(4, 1)), "weight"), (dict(x=x, bias=torch.zeros(4, dtype=torch.int32)), "bias"),
                      (dict(x=x, weight=torch.zeros(4), bias=torch.zeros(4).half()), "different"), (dict(x=x, eps=-1.0), "eps"),
                      (dict(x=x, eps=math.nan), "eps"), (dict(x=x, weight=torch.zeros(4, device="meta")), "move them")):
        with pytest.raises(Error, match=word):
            layer_norm(**bad)
    with pytest.raises(RuntimeError, match="once_differentiable|twice|does not require grad"):
        xr = torch.randn(2, 4, requires_grad=True)
        g, = torch.autograd.grad(layer_norm(xr).pow(2).sum(), xr, create_graph=True)
        g.sum().backward()


def test_scores_refuse():
    x, i = torch.zeros(2, 5), torch.zeros(2, dtype=torch.int64)
    for bad, word in ((dict(X=x.long(), ids=i), "float32"), (dict(X=torch.tensor(1.0)), "rows"), (dict(X=torch.zeros(2, 0)), "rows"),
                      (dict(X=x, ids=i.float()), "int64"), (dict(X=x, ids=torch.zeros(3, dtype=torch.int64)), "ids"),
                      (dict(X=x, ids=torch.zeros(2, 1, 1, dtype=torch.int64)), "ids"),
                      (dict(X=x, ids=torch.zeros(2, 1025, dtype=torch.int64)), "1024"),
                      (dict(X=x, ids=torch.tensor(0)), "ids"), (dict(X=x, top_k=6), "top_k"), (dict(X=x, top_k=-1), "top_k"),
                      (dict(X=torch.zeros(2, 99), top_k=65), "top_k"), (dict(X=x, top_k=1.0), "top_k"),
                      (dict(X=x, temperature=0.0), "temperature"), (dict(X=x, temperature=-1.0), "temperature"),
                      (dict(X=x, temperature=math.nan), "temperature"), (dict(X=x, temperature=1e7), "temperature"),
                      (dict(X=x, temperature=torch.tensor(1.0)), "temperature"),
                      (dict(X=x, ids=i.to("meta")), "move them")):
        with pytest.raises(Error, match=word):
            score_logprobs(**bad)
    with pytest.raises(IndexError):
        score_logprobs(x, torch.tensor([0, 5]))
    assert score_logprobs(x, torch.tensor([0, 5]), check_ids=False).logp.isnan().tolist() == [False, True]
    with pytest.raises(Error, match="temperature"):
        HipScoreLogprobs(temperature=0)


def test_distill_refuses():
    x, i, t = torch.zeros(2, 5), torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 3)
    for bad, word in (((x.int(), i, t), "float32"), ((x, i[:, 0], t), "top_ids"), ((x, i, t[:, :2]), "top_scores"),
                      ((x, i, t.int()), "top_scores"), ((x, i[:, :0], t[:, :0]), "top_ids"), ((x, i.float(), t), "int64"),
                      ((x, i, t, 0.0), "temperature"), ((x, i, t.requires_grad_(True)), "constant"),
                      ((x, i.to("meta"), t.detach()), "move them")):
        with pytest.raises(Error, match=word):
            distill_loss(*bad)
    with pytest.raises(IndexError):
        distill_loss(x, i + 5, t.detach())
    with pytest.raises(Error, match="reduction"):
        HipDistillLoss(reduction="max")


def test_modules_can_be_copied():
    for m in (HipScoreLogprobs(2.0, 3, True), HipDistillLoss(2.0, "sum")):
        c = copy.deepcopy(m)
        assert c._id_status is not m._id_status and c.temperature == 2.0 and not list(c.state_dict())


def test_empty_batches_on_host():
    x = torch.zeros(0, 5, requires_grad=True)
    assert layer_norm(x).shape == (0, 5)
    r = score_logprobs(x, torch.zeros(0, 3, dtype=torch.int64), top_k=2, entropy=True)
    assert [tuple(v.shape) for v in r] == [(0, 3), (0,), (0, 2), (0, 2)]
    assert distill_loss(x, torch.zeros(0, 3, dtype=torch.int64), torch.zeros(0, 3)).shape == (0,)


# ---- the C entries -------------------------------------------------------------------------------------------------------

def test_c_entries_check_their_arguments():
    if torch.cuda.is_available():
        pytest.skip("made-up addresses: only where nothing can be launched")
    lib = native.load()
    declare_row_calls(lib)
    bad, unsup, ok = native.ERR_BAD_ARG, native.ERR_UNSUPPORTED, native.OK
    P = 1 << 20                                                  # an address that is never used: no call below launches
    view = lambda rows=4, d=8, ty=0, x=P: (rows, 0, 0, d, d, ty, x)      # noqa: E731
    fwd = lib.armnet_layer_norm_fwd
    assert fwd(*view(rows=-1), 0, None, None, 1e-5, P, None, None, None) == bad
    assert fwd(*view(d=0), 0, None, None, 1e-5, P, None, None, None) == bad
    assert fwd(*view(ty=3), 0, None, None, 1e-5, P, None, None, None) == bad
    assert fwd(*view(), 7, None, None, 1e-5, P, None, None, None) == bad
    assert fwd(*view(), 0, None, None, -1.0, P, None, None, None) == bad
    assert fwd(*view(), 0, None, None, 1e-5, P, P, None, None) == bad          # mean without rstd
    assert fwd(*view(), 0, None, None, 1e-5, None, None, None, None) == bad
    assert fwd(*view(rows=1 << 31), 0, None, None, 1e-5, P, None, None, None) == unsup
    assert fwd(*view(d=1 << 31), 0, None, None, 1e-5, P, None, None, None) == unsup
    assert fwd(*view(rows=0, x=None), 0, None, None, 1e-5, None, None, None, None) == ok
    bwd = lib.armnet_layer_norm_bwd
    need = lib.armnet_layer_norm_bwd_ws_bytes(100000, 8)                        # parameter gradients of many rows: a workspace
    assert need > 0 and bwd(*view(rows=100000), P, 0, None, P, P, P, P, None, None, 0, None) == bad
    assert bwd(*view(rows=100000), P, 0, None, P, P, P, P, None, P, need - 1, None) == bad
    assert bwd(*view(rows=100000), P, 0, None, P, P, P, P, None, None, need, None) == bad
    assert bwd(*view(), None, 0, None, P, P, P, None, None, None, 0, None) == bad
    assert bwd(*view(rows=0, x=None), None, 0, None, None, None, None, None, None, None, 0, None) == ok
    assert lib.armnet_layer_norm_bwd_ws_bytes(-1, 8) == -1 and lib.armnet_layer_norm_bwd_ws_bytes(4, 0) == -1
    sc = lib.armnet_score_logprobs_fwd
    tail = (P, None, None, None, None, None, 0, None, None)
    assert sc(*view(), 0.0, 1, P, 0, 0, *tail) == bad
    assert sc(*view(), 1.0, -1, P, 0, 0, *tail) == bad
    assert sc(*view(), 1.0, 1, None, 0, 0, *tail) == bad
    assert sc(*view(), 1.0, 1, P, 2, 0, *tail) == bad
    assert sc(*view(), 1.0, 1, P, 0, 9, *tail) == bad                           # more alternatives than scores
    assert sc(*view(), 1.0, 1, P, 0, 1, *tail) == bad                           # nowhere to put them
    assert sc(*view(), 1.0, 1025, P, 0, 0, *tail) == unsup
    assert sc(*view(d=100), 1.0, 1, P, 0, 65, *tail) == unsup
    assert sc(*view(rows=0, x=None), 1.0, 0, None, 0, 0, *tail) == ok
    assert lib.armnet_score_ws_bytes(-1, 8, 0) == -1 and lib.armnet_score_ws_bytes(1, 8, -1) == -1
    big = lib.armnet_score_ws_bytes(1, 1 << 20, 64)
    if big:                                                                     # a split row needs its workspace
        assert sc(*view(rows=1, d=1 << 20), 1.0, 1, P, 0, 64, P, None, P, P, None, P, big - 1, None, None) == bad
    assert lib.armnet_score_logprobs_bwd(*view(), 1.0, 1, P, 0, P, None, P, P, P, None) == bad    # g_entropy without entropy
    assert lib.armnet_score_logprobs_bwd(*view(), 1.0, 1, P, 0, None, None, P, None, P, None) == bad
    di = lib.armnet_distill_fwd
    assert di(*view(), 1.0, 0, P, 0, 0, P, P, None, None, 0, None, None) == bad
    assert di(*view(), 1.0, 2, P, 0, 5, P, P, None, None, 0, None, None) == bad
    assert di(*view(), 1.0, 2, P, 0, 0, None, P, None, None, 0, None, None) == bad
    assert lib.armnet_distill_bwd(*view(), 1.0, 2, P, 0, 0, P, None, P, P, None) == bad


def test_row_views_need_no_copy():
    """two strides describe the leading dimensions: slices, shifted batches, expanded rows"""
    base = torch.arange(2 * 3 * 4 * 6.).view(2, 3, 4, 6)

    def rows_of(x):
        y, rows, inner, so, sr = native.rows().rows_of(x)
        d = y.shape[-1]
        st = y.untyped_storage()
        flat = torch.empty(0, dtype=y.dtype).set_(st)
        at = [(r // inner) * so + (r % inner) * sr if inner else r * sr for r in range(rows)]
        got = torch.stack([flat[y.storage_offset() + o:y.storage_offset() + o + d] for o in at]) if rows else y.reshape(0, d)
        assert torch.equal(got, x.reshape(-1, d))
        return y.data_ptr() == x.data_ptr()

    assert rows_of(base) and rows_of(base[..., 1:5]) and rows_of(base[0, :, 1:]) and rows_of(base[:, 0, 1:3])
    assert rows_of(base[0].transpose(0, 1)) and rows_of(base[:1, :, ::2]) and rows_of(base[0, 0, :1].expand(5, 6))
    assert rows_of(base[0, 0, 0]) and rows_of(base[:, :, 1:3])
    assert not rows_of(base[:, ::2, ::2]) and not rows_of(base.transpose(-1, -2)) and not rows_of(base[..., ::2])
    assert rows_of(base[..., :1])
