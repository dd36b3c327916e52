"""Calls that have no forward-mode derivative refuse tensors that carry a tangent, which would be lost in them without a word."""
import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu


def dual(t):
    return forward_ad.make_dual(t, torch.ones_like(t))


def ints(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.fixture(params=["native", "python"])
def route(request, monkeypatch):
    """Both host sides of a call: in native code, and the one that words errors."""
    import qtensor.cache
    import qtensor.functional as F
    assert F._direct is not None
    if request.param == "python":
        monkeypatch.setattr(F, "_direct", None)
        monkeypatch.setattr(qtensor.cache, "_native", None)


def test_turning_refuses_tangents(route):
    from qtensor.rotary import Rotary
    rotary, q, k, at = Rotary(32), torch.ones(5, 4, 64, device="cuda"), torch.ones(5, 2, 64, device="cuda"), torch.arange(5, device="cuda")
    want = rotary.turn(q, k, at)
    with forward_ad.dual_level():
        for a, b in ((dual(q), k), (q, dual(k)), (dual(q), None), (dual(q.clone().requires_grad_()), k), (dual(q)[:, 1:], k), (q, dual(k).view(5, 2, 64))):
            with pytest.raises((NotImplementedError, RuntimeError)):
                rotary.turn(a, b, at)
        with torch.no_grad(), pytest.raises((NotImplementedError, RuntimeError)):
            rotary.turn(dual(q), k, at)
        got = rotary.turn(q, k, at)                                 # (a level alone is no reason)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        got = rotary.turn(forward_ad.unpack_dual(dual(q)).primal, k, at)
        assert torch.equal(got[0], want[0])


def test_products_refuse_tangents(route):
    from qtensor.linear import QTensorLinear
    weights = QTensorLinear(64, 16).quantize(torch.ones(16, 64, device="cuda"))
    x, bias, out = torch.ones(3, 64, device="cuda"), torch.ones(16, device="cuda"), torch.zeros(3, 16, device="cuda")
    want = weights.product(x, bias)
    with forward_ad.dual_level():
        for bad in (dict(x=dual(x)), dict(x=x, bias=dual(bias)), dict(x=x, bias=bias, out=dual(out)), dict(x=dual(x).view(1, 3, 64)), dict(x=dual(x)[1:])):
            with pytest.raises(RuntimeError):
                weights.product(**bad)
            with torch.no_grad(), pytest.raises(RuntimeError):
                weights.product(**bad)
        assert not out.any() and torch.equal(weights.product(x, bias, out), want)


def test_the_cache_refuses_tangents(route):
    from qtensor.cache import QTensorCache
    from qtensor.rotary import Rotary
    cache, rotary = QTensorCache(4, 2, 64), Rotary(64)
    q, k, table, lengths = torch.ones(3, 4, 64, device="cuda"), torch.ones(3, 2, 64, device="cuda"), ints(0, 1, 2).view(3, 1), ints(1, 1, 1)
    totals = cache.totals(table)
    with forward_ad.dual_level():
        for call in (lambda: cache.write(dual(k), k, table, lengths), lambda: cache.write(k, dual(k), table, lengths),
                     lambda: cache.write_turned(rotary, dual(q), k, k, table, lengths), lambda: cache.write_turned(rotary, q, dual(k), k, table, lengths),
                     lambda: cache.write_turned(rotary, q, k, dual(k), table, lengths), lambda: cache.write_turned(rotary, q, k, k, table, lengths, out=dual(q.clone())),
                     lambda: cache.attend(dual(q), table, lengths), lambda: cache.attend(q, table, lengths, out=dual(q.clone())),
                     lambda: cache.weigh(totals, dual(q), table, lengths)):
            with pytest.raises(RuntimeError):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError):
                call()
        assert not cache.codes.any() and not totals.any()           # (nothing was launched)
        cache.write(k, k, table, lengths)
        assert cache.codes.any() and torch.allclose(cache.attend(q, table, lengths)[:, :2], k)


def test_other_transformations_raise(route):
    """Not lost: gradients by torch.func, batched calls and batched gradients."""
    from qtensor.rotary import Rotary
    rotary, q, at = Rotary(32), torch.ones(5, 4, 64, device="cuda"), torch.arange(5, device="cuda")
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda q: rotary.turn(q, None, at)[0].sum())(q)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda q: rotary.turn(q, None, at)[0], (q,), (q,))
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda q: rotary.turn(q, None, at)[0])(q.expand(3, 5, 4, 64))
    leaf = q.clone().requires_grad_()
    out = rotary.turn(leaf, None, at)[0]
    with pytest.raises(RuntimeError):
        torch.autograd.grad(out, leaf, torch.ones(3, 5, 4, 64, device="cuda"), is_grads_batched=True)
