"""Ids past the row, in every kernel that takes a list: the report, NaN in their slots, and nothing else changes."""
import pytest
import torch

from armnet_hip import HipDistillLoss, HipScoreLogprobs, distill_loss, score_logprobs

pytestmark = pytest.mark.gpu
DEV = "cuda"
BIG = 2 ** 63 - 1


def gen(seed):
    return torch.Generator().manual_seed(seed)


# short rows, a wave a row, a block a row, rows in slices that are joined; and a wave a row of 5382 scores
SHAPES = [(6, 10), (6, 60), (6, 700), (6, 5382), (4100, 5382), (6, 150001)]


def bad_ids(c, id_type):
    past = [c, c + 1, 2 ** 31 - 1] + ([2 ** 31, 2 ** 31 + 1, 2 ** 32, 2 ** 32 + 3, BIG] if id_type == torch.int64 else [])
    return past, [-1, -c, -2 ** 31] + ([-2 ** 31 - 1, -2 ** 32, -2 ** 32 + 3, -2 ** 63] if id_type == torch.int64 else [])


@pytest.mark.parametrize("id_type", [torch.int64, torch.int32])
@pytest.mark.parametrize("n", [1, 7, 65, 300])
@pytest.mark.parametrize("rows,c", SHAPES)
def test_scores(rows, c, n, id_type):
    x = torch.randn(rows, c, generator=gen(0)).to(DEV).requires_grad_(True)
    ids = torch.randint(0, c, (rows, n), generator=gen(1)).to(id_type)
    g, gh = torch.randn(rows, n, generator=gen(2)).to(DEV), torch.randn(rows, generator=gen(3)).to(DEV)
    places = [(1, 0), (2, n - 1), (rows - 1, n // 2)]

    def with_slots(v):
        i = ids.clone()
        for p in places:
            i[p] = v
        return i.to(DEV)

    def said(i, top):
        r = score_logprobs(x, i, 1.3, min(top, c), True, check_ids=False)
        return r, torch.autograd.grad((r.logp, r.entropy), x, (g, gh))[0]

    past, empty = bad_ids(c, id_type)
    at = torch.zeros(rows, n, dtype=torch.bool)
    for p in places:
        at[p] = True
    at = at.to(DEV)
    for top in (0, 5):
        want, want_dx = said(with_slots(-1), top)
        assert want.logp[at].eq(0).all() and want.logp.isfinite().all() and want_dx.isfinite().all()
        for v in past:
            r, dx = said(with_slots(v), top)
            assert r.logp[at].isnan().all(), v
            assert torch.equal(r.logp[~at], want.logp[~at]) and torch.equal(r.entropy, want.entropy) and torch.equal(dx, want_dx), v
            assert not top or (torch.equal(r.top_ids, want.top_ids) and torch.equal(r.top_logp, want.top_logp)), v
        for v in empty:
            r, dx = said(with_slots(v), top)
            assert torch.equal(r.logp, want.logp) and torch.equal(dx, want_dx), v
    m = HipScoreLogprobs(top_k=min(5, c))
    for v in past:
        with pytest.raises(IndexError):
            score_logprobs(x, with_slots(v))
        m(x, with_slots(v))
        with pytest.raises(IndexError):
            m.poll()
    for v in empty:
        score_logprobs(x, with_slots(v))
    m(x, with_slots(c - 1))
    m.poll()


@pytest.mark.parametrize("id_type", [torch.int64, torch.int32])
@pytest.mark.parametrize("n", [1, 7, 65, 300])
@pytest.mark.parametrize("rows,c", SHAPES)
def test_distillation(rows, c, n, id_type):
    x = torch.randn(rows, c, generator=gen(0)).to(DEV).requires_grad_(True)
    ids = torch.randint(0, c, (rows, n), generator=gen(1)).to(id_type)
    ts, g = torch.randn(rows, n, generator=gen(2)).to(DEV), torch.rand(rows, generator=gen(3)).to(DEV)
    places = [(1, 0), (2, n - 1), (rows - 1, n // 2)]

    def told(v):
        i = ids.clone()
        for p in places:
            i[p] = v
        i = i.to(DEV)
        loss = distill_loss(x, i, ts, 1.3, check_ids=False)
        return i, loss, torch.autograd.grad(loss, x, g)[0]

    past, empty = bad_ids(c, id_type)
    hit = torch.zeros(rows, dtype=torch.bool)
    hit[[p[0] for p in places]] = True
    hit = hit.to(DEV)
    _, want, want_dx = told(-1)
    assert want.isfinite().all() and want_dx.isfinite().all()
    m = HipDistillLoss()
    for v in past:
        i, loss, dx = told(v)
        assert loss[hit].isnan().all(), v
        assert torch.equal(loss[~hit], want[~hit]) and torch.equal(dx[~hit], want_dx[~hit]), v
        with pytest.raises(IndexError):
            distill_loss(x, i, ts)
        m(x, i, ts)
        with pytest.raises(IndexError):
            m.poll()
    for v in empty:
        i, loss, dx = told(v)
        assert torch.equal(loss, want) and torch.equal(dx, want_dx), v
        distill_loss(x, i, ts)
