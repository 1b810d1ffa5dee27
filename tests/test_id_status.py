"""The words of the deferred id reports: memory that kernels may store into outlives whoever asked for it (no GPU: pinning is replaced)."""
import gc
import threading
import weakref

import pytest
import torch

from armnet_hip import block
from armnet_hip.block import IdStatus, _id_mode


@pytest.fixture
def pinned(monkeypatch):
    """every tensor that was pinned, by address range, and which of them were freed"""
    made, freed = [], []
    monkeypatch.setattr(block, "_words", block._Words())

    def pin(t, *args):
        t = t.clone()
        made.append((t.data_ptr(), t.numel() * t.element_size()))
        weakref.finalize(t, freed.append, t.data_ptr())
        return t

    monkeypatch.setattr(torch.Tensor, "pin_memory", pin)
    monkeypatch.setattr(torch.Tensor, "is_pinned", lambda t, *args: any(a <= t.data_ptr() < a + n for a, n in made))
    monkeypatch.setattr(torch.cuda, "synchronize", lambda device=None: None)
    return made, freed


def test_a_word_outlives_its_module_and_is_nobody_elses(pinned):
    """a queued kernel, or a captured graph that is replayed later, stores into a word whose module is gone"""
    made, freed = pinned
    seen, first = set(), []
    for i in range(3000):
        s = IdStatus()
        w = s.word()
        assert w.dtype == torch.int32 and w.numel() == 1 and int(w[0]) == 0 and s.word() is w
        assert w.data_ptr() not in seen, "a word that a queued kernel may still store into was handed out again"
        seen.add(w.data_ptr())
        if i == 0:
            first.append(s)
        del s, w
    gc.collect()
    assert not freed
    first[0].raise_if_set()                                      # nobody else's report
    assert len(made) <= 16                                       # and few allocations for many modules


def test_a_stand_alone_call_gives_its_word_back(pinned):
    """its kernels have finished when it returns"""
    seen = set()
    for i in range(3000):
        status, sync = _id_mode(True, None)
        assert sync
        w = status.word()
        assert int(w[0]) == 0
        seen.add(w.data_ptr())
        if i % 3 == 0:
            w[0] = 1                                             # what a kernel does
            with pytest.raises(IndexError):
                status.poll()
        else:
            status.poll()
        status.poll()
    assert len(seen) == 1 and not pinned[1]
    mine = IdStatus()
    held = mine.word().data_ptr()
    for deferred in (True, "sync"):
        status, sync = _id_mode(deferred, mine)
        assert status is mine and sync == (deferred == "sync")
        mine.poll()
        assert mine.word().data_ptr() == held                    # a module keeps its own


def test_two_threads_have_one_report(pinned, monkeypatch):
    """first calls of one module at once"""
    take, meet = block._words.take, threading.Barrier(2)

    def slow():
        try:
            meet.wait(0.2)                                       # both threads are here, if both may be
        except threading.BrokenBarrierError:
            pass
        return take()

    monkeypatch.setattr(block._words, "take", slow)
    s, got = IdStatus(), []
    ts = [threading.Thread(target=lambda: got.append(s.word())) for _ in range(2)]
    [t.start() for t in ts], [t.join() for t in ts]
    got[0][0] = 1
    with pytest.raises(IndexError):
        s.raise_if_set()
    got[1][0] = 1
    with pytest.raises(IndexError):
        s.raise_if_set()
