"""What the row operators refuse on the device through their public entries, and that nothing else changes by it."""
import pytest
import torch
import torch.autograd.forward_ad as fwd_ad

from armnet_hip import HipDistillLoss, HipLayerNorm, HipScoreLogprobs, distill_loss, layer_norm, native, score_logprobs

pytestmark = pytest.mark.gpu
DEV = "cuda"
Error = native.ArmnetNativeError


def inputs(n=5, c=40, k=3):
    g = torch.Generator().manual_seed(0)
    return (torch.randn(n, c, generator=g).to(DEV), torch.randn(c, generator=g).to(DEV),
            torch.randint(0, c, (n, k), generator=g).to(DEV), torch.randn(n, k, generator=g).to(DEV))


@pytest.mark.parametrize("c", [40, 20001])
@pytest.mark.parametrize("reverse", [False, True])
def test_forward_mode_is_refused(c, reverse):
    x, w, ids, ts = inputs(c=c)
    norm = HipLayerNorm(c).to(DEV)
    with fwd_ad.dual_level():
        dual = lambda t: fwd_ad.make_dual(t.clone().requires_grad_(reverse), torch.ones_like(t))      # noqa: E731
        for call in (lambda: layer_norm(dual(x)), lambda: layer_norm(x, dual(w)), lambda: layer_norm(x, None, dual(w)),
                     lambda: norm(dual(x)), lambda: score_logprobs(dual(x), ids), lambda: score_logprobs(dual(x), entropy=True),
                     lambda: score_logprobs(dual(x), top_k=2), lambda: HipScoreLogprobs(entropy=True)(dual(x)),
                     lambda: distill_loss(dual(x), ids, ts), lambda: HipDistillLoss()(dual(x), ids, ts)):
            with pytest.raises(Error, match="forward-mode"):
                call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode|constant"):
            distill_loss(x, ids, fwd_ad.make_dual(ts, torch.ones_like(ts)))
        assert layer_norm(x, w).isfinite().all()                 # the level alone is no reason


@pytest.mark.parametrize("c", [40, 20001])
def test_a_tangent_of_the_upstream_gradient_is_refused(c):
    x, w, ids, ts = inputs(c=c)
    x.requires_grad_(True)
    calls = (lambda: layer_norm(x, w), lambda: score_logprobs(x, ids).logp, lambda: score_logprobs(x, ids, entropy=True).entropy,
             lambda: distill_loss(x, ids, ts))
    for call in calls:
        out = call()
        want, = torch.autograd.grad(out, x, torch.ones_like(out), retain_graph=True)
        with fwd_ad.dual_level():
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(out, x, fwd_ad.make_dual(torch.ones_like(out), torch.ones_like(out)), retain_graph=True)
        assert torch.equal(torch.autograd.grad(out, x, torch.ones_like(out))[0], want)


@pytest.mark.parametrize("requires_grad", [False, True])
def test_tracing_is_refused(requires_grad):
    from torch.fx.experimental.proxy_tensor import make_fx
    x, w, ids, ts = inputs()
    norm, scores, loss = HipLayerNorm(40).to(DEV), HipScoreLogprobs(top_k=2, entropy=True), HipDistillLoss()
    a = x.clone().requires_grad_(requires_grad)
    for f in (lambda a: layer_norm(a, w), norm, lambda a: score_logprobs(a, ids, check_ids=False).logp, lambda a: scores(a, ids).top_logp,
              lambda a: distill_loss(a, ids, ts, check_ids=False), lambda a: loss(a, ids, ts)):
        with pytest.raises(RuntimeError, match="trace"):
            torch.jit.trace(f, a, check_trace=False)
        with pytest.raises(RuntimeError, match="trace"):
            make_fx(f)(x)
        f(x)                                                     # not recorded: as ever


def test_a_compiled_program_runs_around_the_kernels():
    x, w, ids, ts = inputs()
    f = lambda a: layer_norm(a * 2, w) + score_logprobs(a, ids, check_ids=False).logp.sum()      # noqa: E731
    assert torch.equal(torch.compile(f, backend="eager")(x), f(x))


def test_a_storage_that_was_freed_is_refused():
    """forward, and backward of what was saved; taken back, the same call runs"""
    base, w, ids, ts = inputs(c=44)
    x, w = base[:, 4:].detach().requires_grad_(True), w[4:].detach().requires_grad_(True)      # an offset of its own
    ids = ids % 40
    calls = (lambda a: layer_norm(a, w), lambda a: score_logprobs(a, ids, entropy=True).entropy, lambda a: distill_loss(a, ids, ts))
    for call in calls:
        want = call(x)
        up = torch.ones_like(want)
        grad, = torch.autograd.grad(want, x, up, retain_graph=True)
        keep, storage = x.detach().clone(), x.untyped_storage()
        size = storage.size()
        storage.resize_(0)
        for again in (lambda: call(x), lambda: call(x.detach()), lambda: torch.autograd.grad(want, x, up, retain_graph=True)):
            with pytest.raises(RuntimeError, match="memory"):
                again()
        storage.resize_(size)
        with torch.no_grad():
            x.copy_(keep)
        out = call(x)
        assert torch.equal(out, want) and torch.equal(torch.autograd.grad(out, x, up)[0], grad)


def test_negated_views():
    """every input, and the upstream gradients, as views that are negated on reading"""
    x, w, ids, ts = inputs()
    neg = lambda t: torch._neg_view(-t)                          # noqa: E731
    assert neg(x).is_neg() and torch.equal(neg(x), x)
    x.requires_grad_(True), w.requires_grad_(True)
    for call, args in ((layer_norm, (x, w)), (layer_norm, (x, None, w)), (lambda a: score_logprobs(a, ids).logp, (x,)),
                       (lambda a: score_logprobs(a, ids, entropy=True).entropy, (x,)), (lambda a: distill_loss(a, ids, ts), (x,))):
        want = call(*args)
        up = torch.randn(want.shape, generator=torch.Generator().manual_seed(1)).to(DEV)
        leaves = [t for t in args if t is not None]
        grads = torch.autograd.grad(want, leaves, up, retain_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(want, leaves, neg(up)), grads))
        assert torch.equal(call(*(None if t is None else neg(t.detach()) for t in args)), want)
    assert torch.equal(distill_loss(x, ids, neg(ts)), distill_loss(x, ids, ts))
    assert torch.equal(score_logprobs(x, neg(ids)).logp, score_logprobs(x, ids).logp)
    assert torch.equal(distill_loss(x, neg(ids), ts), distill_loss(x, ids, ts))
