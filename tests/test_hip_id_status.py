"""The deferred id reports on the device: kernels that are queued, or replayed, when their module is gone."""
import gc

import pytest
import torch

from armnet_hip import HipDistillLoss, HipScoreLogprobs, block, embedding_forward, score_logprobs

pytestmark = pytest.mark.gpu
DEV = "cuda"


def pinned_by_others():
    return [torch.zeros(n, dtype=torch.int32).pin_memory() for n in (1, 1, 1, 8, 64, 1024, 1024, 4096) for _ in range(8)]


def test_words_are_pinned_and_reported_through():
    a, b = block.IdStatus(), block.IdStatus()
    assert a.word().is_pinned() and b.word().is_pinned() and a.word().data_ptr() != b.word().data_ptr()
    x, ids = torch.randn(3, 9, device=DEV), torch.tensor([1, 9, 2], device=DEV)
    score_logprobs(x, ids, status=a)
    score_logprobs(x, ids.clamp(max=8), status=b)
    with pytest.raises(IndexError):
        a.poll()
    a.poll(), b.poll()


def test_a_module_that_is_gone_before_its_kernels_ran():
    x = torch.randn(4000, 5000, device=DEV)
    ids = torch.full((4000, 2), 5000, device=DEV)
    ts = torch.zeros(4000, 2, device=DEV)
    torch.cuda.synchronize()
    for _ in range(30):
        HipScoreLogprobs(entropy=True)(x, ids)
        HipDistillLoss()(x, ids, ts)
    gc.collect()
    others, modules = pinned_by_others(), [HipScoreLogprobs() for _ in range(40)]
    for m in modules:
        m(x[:2], ids[:2] - 1)
    torch.cuda.synchronize()
    assert all(int(t.abs().sum()) == 0 for t in others)
    for m in modules:
        m.poll()


def test_a_graph_that_is_replayed_when_its_module_is_gone():
    x, ids = torch.randn(6, 50, device=DEV), torch.zeros(6, 2, dtype=torch.int64, device=DEV)
    m = HipScoreLogprobs(entropy=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        m(x, ids)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = m(x, ids)
    del m
    gc.collect()
    others, after = pinned_by_others(), HipScoreLogprobs()
    after(x, ids)
    ids.fill_(50)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert out.logp.isnan().all() and all(int(t.abs().sum()) == 0 for t in others)
        after.poll()
    ids.zero_()
    graph.replay()
    assert torch.equal(out.logp, score_logprobs(x, ids).logp)


def test_a_first_call_inside_a_capture():
    """its word is there already: nothing is allocated while a graph is recorded"""
    block.IdStatus().word()
    x, ids = torch.randn(6, 50, device=DEV), torch.zeros(6, 2, dtype=torch.int64, device=DEV)
    want = score_logprobs(x, ids).logp
    m = HipScoreLogprobs()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = m(x, ids).logp
    graph.replay()
    assert torch.equal(out, want)
    m.poll()


def test_stand_alone_calls_keep_their_report():
    x, table = torch.randn(5, 7, device=DEV), torch.randn(7, 4, device=DEV)
    for _ in range(3):
        with pytest.raises(IndexError):
            score_logprobs(x, torch.full((5,), 7, device=DEV))
        assert score_logprobs(x, torch.full((5,), 6, device=DEV)).logp.isfinite().all()
        with pytest.raises(IndexError):
            embedding_forward(torch.tensor([[7]], device=DEV), torch.ones(1, 1, device=DEV), table)
        embedding_forward(torch.tensor([[6]], device=DEV), torch.ones(1, 1, device=DEV), table)
