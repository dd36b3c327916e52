"""The node in Python of a turn keeps the angles it turned by, as far as that can be seen without a GPU: with angles worked out by the oracle."""
import pytest
import torch

from oracle import rotary_ref as R


@pytest.fixture
def turn():
    from qtensor.rotary import Rotary, _Turn

    class Elsewhere(Rotary):
        def _turned(self, back, tensors, positions):
            return [R.turned(t, positions, self.frequencies, self.dims, self.magnitude, self.interleaved, back)[0].to(t.dtype) for t in tensors]
    return lambda rotary, q, k, at: _Turn.apply(rotary, False, q, k, at), Elsewhere


def test_gradients_go_by_the_angles_of_the_call(turn):
    call, Elsewhere = turn
    g = torch.Generator().manual_seed(1)
    q, k, at = torch.randn(6, 4, 64, generator=g).requires_grad_(), torch.randn(6, 2, 64, generator=g).requires_grad_(), torch.arange(6) + 3
    dq, dk = torch.randn(6, 4, 64, generator=g).requires_grad_(), torch.randn(6, 2, 64, generator=g)
    want = torch.autograd.grad(call(Elsewhere(32, device="cpu"), q, k, at), (q, k), (dq, dk))
    assert torch.equal(want[0], R.turned(dq, at, Elsewhere(32, device="cpu").frequencies, 32, back=True)[0].float())
    for change in (lambda r: setattr(r, "frequencies", r.frequencies * 2), lambda r: setattr(r, "magnitude", 3.0), lambda r: setattr(r, "interleaved", True),
                   lambda r: (setattr(r, "dims", 16), setattr(r, "frequencies", r.frequencies[:8]))):
        rotary = Elsewhere(32, device="cpu")
        out = call(rotary, q, k, at)
        change(rotary)
        first = torch.autograd.grad(out, (q, k), (dq, dk), create_graph=True)
        assert torch.equal(first[0], want[0]) and torch.equal(first[1], want[1])
        again, = torch.autograd.grad(first[0], dq, q.detach())                      # (and of the gradient's gradient)
        assert torch.equal(again, call(Elsewhere(32, device="cpu"), q.detach(), None, at)[0])
    rotary = Elsewhere(32, device="cpu")
    out = call(rotary, q, k, at)
    rotary.frequencies.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out, (q, k), (dq, dk))


def test_frequencies_made_in_inference_mode(turn):
    call, Elsewhere = turn
    with torch.inference_mode():
        rotary = Elsewhere(32, device="cpu")
    q, at = torch.ones(6, 4, 64).requires_grad_(), torch.arange(6)
    got, = torch.autograd.grad(call(rotary, q, None, at)[0].sum(), q)
    want, = torch.autograd.grad(call(Elsewhere(32, device="cpu"), q, None, at)[0].sum(), q)
    assert torch.equal(got, want)
