"""Hooks that give back something else than a turn has saved: an error, and nothing of it is read on the GPU."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("which", ["positions", "frequencies"])
@pytest.mark.parametrize("change", [lambda t: t.cpu(), lambda t: t[:3], lambda t: t.half(), lambda t: t.unsqueeze(0).unsqueeze(0), lambda t: t[:0], lambda t: t.repeat(2)])
def test_what_comes_back_is_looked_at(monkeypatch, native, which, change):
    import qtensor.functional as F
    from qtensor.rotary import Rotary
    assert F._direct is not None
    if not native:
        monkeypatch.setattr(F, "_direct", None)
    rotary, q, at = Rotary(32), torch.ones(6, 4, 64, device="cuda", requires_grad=True), torch.arange(6, device="cuda")
    mine = torch.int64 if which == "positions" else torch.float64
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: change(t) if t.dtype == mine else t):
        out = rotary.turn(q, None, at)[0]
    with pytest.raises((RuntimeError, ValueError)):
        torch.autograd.grad(out, q, torch.ones_like(out))
    out = rotary.turn(q, None, at)[0]
    got, = torch.autograd.grad(out, q, torch.ones_like(out))
    assert bool(torch.isfinite(got).all())


def test_positions_of_another_type_may_come_back():
    from qtensor.rotary import Rotary
    rotary, q, at = Rotary(32), torch.ones(2, 6, 4, 64, device="cuda", requires_grad=True), torch.arange(12, device="cuda").view(2, 6)
    want, = torch.autograd.grad(rotary.turn(q, None, at)[0].square().sum(), q)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.to(torch.int32) if t.dtype == torch.int64 else t, lambda t: t):
        out = rotary.turn(q, None, at)[0]
    assert torch.equal(torch.autograd.grad(out.square().sum(), q)[0], want)


def test_gradients_with_tangents_raise():
    from torch.autograd import forward_ad
    from qtensor.rotary import Rotary
    rotary, q, at = Rotary(32), torch.ones(6, 4, 64, device="cuda", requires_grad=True), torch.arange(6, device="cuda")
    out = rotary.turn(q, None, at)[0]
    with forward_ad.dual_level(), pytest.raises(RuntimeError):
        torch.autograd.grad(out, q, forward_ad.make_dual(torch.ones_like(out), torch.ones_like(out)))
