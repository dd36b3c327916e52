"""A gradient turns back by the angles that were turned by, whatever has become of the frequencies in between."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("native", [True, False])
def test_gradients_go_by_the_angles_of_the_call(monkeypatch, native):
    import qtensor.functional as F
    from qtensor.rotary import Rotary
    assert F._direct is not None
    if not native:
        monkeypatch.setattr(F, "_direct", None)
    g = torch.Generator().manual_seed(1)
    q, at = torch.randn(6, 4, 64, generator=g).cuda().requires_grad_(), torch.arange(6, device="cuda") + 3
    grad = torch.randn(6, 4, 64, generator=g).cuda()
    want, = torch.autograd.grad(Rotary(32).turn(q, None, at)[0], q, grad)
    for change in (lambda r: setattr(r, "frequencies", r.frequencies * 2), lambda r: setattr(r, "magnitude", 3.0), lambda r: setattr(r, "interleaved", True),
                   lambda r: (setattr(r, "dims", 16), setattr(r, "frequencies", r.frequencies[:8]))):
        rotary = Rotary(32)
        out = rotary.turn(q, None, at)[0]
        change(rotary)
        got, = torch.autograd.grad(out, q, grad)
        assert torch.equal(got, want)
    for change in (lambda r: r.frequencies.mul_(2), lambda r: at.add_(1)):          # (in place: what was saved is gone)
        rotary = Rotary(32)
        out = rotary.turn(q, None, at)[0]
        change(rotary)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(out, q, grad)
