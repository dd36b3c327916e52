"""Tensors that carry a forward-mode tangent are refused by the checks of calls that have no derivative, and by the node of those that have a gradient only."""
import pytest
import torch
from torch.autograd import forward_ad


def test_tangents_are_refused():
    import qtensor.functional as F
    from qtensor.cache import QTensorCache
    cache, x = QTensorCache(2, 2, 64, device="cpu"), torch.ones(1, 2, 64)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, x)
        for t in (dual, dual[:], dual.view(1, 2, 64)):
            with pytest.raises(RuntimeError, match="x carries a forward-mode tangent"):
                F._check_derivatives("weights", bias=None, x=t)
            with torch.no_grad(), pytest.raises(RuntimeError, match="q carries a forward-mode tangent"):
                cache._check_vectors(t, "q", (1, 2, 64), torch.float32)
        cache._check_vectors(x, "q", (1, 2, 64), torch.float32)
        cache._check_vectors(forward_ad.unpack_dual(dual).primal, "q", (1, 2, 64), torch.float32)
    F._check_derivatives("weights", x=x, bias=None)


def test_turning_has_no_forward_mode_derivative():
    from qtensor.rotary import Rotary, _Turn

    class Elsewhere(Rotary):
        def _turned(self, back, tensors, positions):
            return [t.clone() for t in tensors]
    rotary, q, at = Elsewhere(32, device="cpu"), torch.ones(5, 2, 64), torch.arange(5)
    with forward_ad.dual_level(), pytest.raises(NotImplementedError):
        _Turn.apply(rotary, False, forward_ad.make_dual(q, q), None, at)
