"""What the row operators' C++ calls refuse before anything else, so that it shows without a GPU: on a host tensor a call that is not
refused for its reason ends at `expected a tensor on the HIP device`."""
import pytest
import torch
import torch.autograd.forward_ad as fwd_ad

from armnet_hip import distill_loss, layer_norm, native, score_logprobs

Error = native.ArmnetNativeError


def calls(tensor):
    """every call, with each of its float inputs in turn made by `tensor(shape)`"""
    rows = native.rows()
    x, w, ids, ts = torch.randn(3, 8), torch.randn(8), torch.zeros(3, 2, dtype=torch.int64), torch.randn(3, 2)
    return {
        "layer_norm(x)": lambda: rows.layer_norm(tensor(3, 8), w, w, 1e-5),
        "layer_norm(weight)": lambda: rows.layer_norm(x, tensor(8), None, 1e-5),
        "layer_norm(bias)": lambda: rows.layer_norm(x, None, tensor(8), 1e-5),
        "score_logprobs(X)": lambda: rows.score_logprobs(tensor(3, 8), ids, 1.0, 2, True, None),
        "score_logprobs(X) without ids": lambda: rows.score_logprobs(tensor(3, 8), None, 1.0, 0, True, None),
        "distill_loss(X)": lambda: rows.distill_loss(tensor(3, 8), ids, ts, 1.0, None),
        "distill_loss(top_scores)": lambda: rows.distill_loss(x, ids, tensor(3, 2), 1.0, None),
    }


NAMES = list(calls(torch.randn))


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("reverse", [False, True])
def test_forward_mode_is_refused(name, reverse):
    """a tangent that the kernels cannot carry is no result without one"""
    with fwd_ad.dual_level():
        with pytest.raises(Error, match="forward-mode"):
            calls(lambda *s: fwd_ad.make_dual(torch.randn(s).requires_grad_(reverse), torch.ones(s)))[name]()
        with torch.no_grad(), pytest.raises(Error, match="forward-mode"):          # no_grad is about the other mode
            calls(lambda *s: fwd_ad.make_dual(torch.randn(s), torch.ones(s)))[name]()
        with pytest.raises(Error, match="HIP device"):                             # the level alone is no reason
            calls(torch.randn)[name]()


def test_forward_mode_is_refused_on_host():
    ids, ts = torch.zeros(3, 2, dtype=torch.int64), torch.randn(3, 2)
    with fwd_ad.dual_level():
        x, w = fwd_ad.make_dual(torch.randn(3, 8), torch.ones(3, 8)), fwd_ad.make_dual(torch.randn(8), torch.ones(8))
        t = fwd_ad.make_dual(ts, torch.ones(3, 2))
        for call in (lambda: layer_norm(x), lambda: layer_norm(torch.randn(3, 8), w), lambda: score_logprobs(x, ids),
                     lambda: score_logprobs(x, entropy=True), lambda: distill_loss(x, ids, ts),
                     lambda: distill_loss(torch.randn(3, 8), ids, t)):
            with pytest.raises(RuntimeError):
                call()


@pytest.mark.parametrize("name", NAMES)
def test_tracing_is_refused(name):
    """a recorder sees the outputs' allocation and not the kernels: what it replays is memory that nothing wrote"""
    from torch.fx.experimental.proxy_tensor import make_fx

    def run(a):
        return calls(lambda *s: a[0] if len(s) == 1 else a[:s[0], :s[1]])[name]()

    a = torch.randn(3, 8)
    for requires_grad in (False, True):
        with pytest.raises(Error, match="trace"):
            torch.jit.trace(run, a.requires_grad_(requires_grad), check_trace=False)
    with pytest.raises(Error, match="trace"):
        make_fx(run)(a.detach())
    with pytest.raises(Error, match="HIP device"):
        run(a)


def test_host_tensors_can_be_traced():
    x, ids = torch.randn(3, 8), torch.zeros(3, 2, dtype=torch.int64)
    f = torch.jit.trace(lambda a: layer_norm(a) * 2, torch.randn(3, 8))
    assert torch.equal(f(x), layer_norm(x) * 2)
    f = torch.jit.trace(lambda a: score_logprobs(a, ids, check_ids=False).logp, torch.randn(3, 8))
    assert torch.equal(f(x), score_logprobs(x, ids).logp)


@pytest.mark.parametrize("name", NAMES)
def test_tensors_without_memory_are_refused(name):
    """a fake view's address is an offset from nowhere"""
    from torch._subclasses import FakeTensorMode
    with FakeTensorMode() as mode:
        def fake(*s):
            t = mode.from_tensor(torch.zeros(s[:-1] + (s[-1] + 4,)))[..., 4:]
            assert t.storage_offset() == 4
            return t
        with pytest.raises(Error, match="memory"):
            calls(fake)[name]()

    def freed(*s):                                               # behind its tensors, as sharded parameters are
        t = torch.zeros(s[:-1] + (s[-1] + 4,))[..., 4:]
        t.untyped_storage().resize_(0)
        return t
    with pytest.raises(Error, match="memory"):
        calls(freed)[name]()
    with pytest.raises(Error, match="HIP device"):
        calls(torch.randn)[name]()


def test_rows_of_negated_views():
    """a view that is negated on reading (the imaginary part of a conjugate) has its values copied, whatever its strides"""
    z = torch.complex(torch.randn(4, 6), torch.randn(4, 6))
    for v in (z.conj().imag, z.conj().imag[..., :1], torch._neg_view(torch.randn(4, 6)), torch._neg_view(torch.randn(4, 6))[:, 1:]):
        assert v.is_neg()
        y, rows, inner, outer, stride = native.rows().rows_of(v)
        assert not y.is_neg() and torch.equal(y, v) and rows == 4 and inner == 0
        flat = torch.empty(0).set_(y.untyped_storage())
        for r in range(4):
            at = y.storage_offset() + r * stride
            assert torch.equal(flat[at:at + v.shape[1]], v[r])
