"""Turning by rotary positions where what it saves for its gradient goes through hooks: recomputed layers, hooks that raise, hooks that count."""
import pytest
import torch
from torch.utils.checkpoint import checkpoint

pytestmark = pytest.mark.gpu


@pytest.fixture
def inputs():
    from qtensor.rotary import Rotary
    import qtensor.functional as F
    assert F._direct is not None
    g = torch.Generator().manual_seed(1)
    return Rotary(32), torch.randn(6, 4, 64, generator=g).cuda().requires_grad_(), torch.randn(6, 2, 64, generator=g).cuda().requires_grad_(), torch.arange(6, device="cuda")


@pytest.mark.parametrize("early_stop", [True, False])
def test_a_recomputed_region_that_ends_in_a_turn(inputs, early_stop):
    from torch.utils.checkpoint import set_checkpoint_early_stop
    rotary, q, k, at = inputs

    def region(q, k):
        return rotary.turn(q * q, k.sin(), at)
    want = torch.autograd.grad([t.square().sum() for t in region(q, k)], (q, k))
    with set_checkpoint_early_stop(early_stop):
        out = checkpoint(region, q, k, use_reentrant=False)
        got = torch.autograd.grad([t.square().sum() for t in out], (q, k))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_a_recomputed_layer(inputs):
    rotary, q, k, at = inputs

    def layer(q, k):
        for _ in range(3):
            q, k = rotary.turn(q.tanh(), k.cos(), at)
        return q, k
    want = torch.autograd.grad([t.sum() for t in layer(q, k)], (q, k))
    got = torch.autograd.grad([t.sum() for t in checkpoint(layer, q, k, use_reentrant=False)], (q, k))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_hook_that_raises(inputs):
    rotary, q, k, at = inputs

    class Stop(Exception):
        pass
    calls = []

    def pack(t):
        calls.append(t.dtype)
        raise Stop("not this one")
    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t), pytest.raises(Stop, match="not this one"):
        rotary.turn(q, k, at)
    assert len(calls) == 1                                          # (not asked a second time)
    out = rotary.turn(q, k, at)
    assert out[0].requires_grad


def test_hooks_see_what_is_saved_once(inputs):
    rotary, q, k, at = inputs
    want = torch.autograd.grad([t.square().sum() for t in rotary.turn(q, k, at)], (q, k))
    packed, unpacked = [], []

    def pack(t):
        packed.append(t)
        return t.cpu()

    def unpack(t):
        unpacked.append(t)
        return t.cuda()
    with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
        out = rotary.turn(q, k, at)
    assert len(packed) <= 2 and any(t.data_ptr() == at.data_ptr() for t in packed)
    got = torch.autograd.grad([t.square().sum() for t in out], (q, k))
    assert len(unpacked) == len(packed) and torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])

    def fails(t):
        raise ValueError("lost")
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, fails):
        out = rotary.turn(q, k, at)
    with pytest.raises(ValueError, match="lost"):
        torch.autograd.grad(out[0].sum(), q)


def test_frequencies_made_in_inference_mode(inputs):
    """They cannot be saved by torch and need not be: nobody can change them in place outside that mode."""
    from qtensor.rotary import Rotary
    rotary, q, k, at = inputs
    with torch.inference_mode():
        other = Rotary(32)
    packed = []
    want = torch.autograd.grad(rotary.turn(q, k, at)[0].square().sum(), q)[0]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: packed.append(t) or t, lambda t: t):
        out = other.turn(q, k, at)
    assert len(packed) == 1
    assert torch.equal(torch.autograd.grad(out[0].square().sum(), q)[0], want)
