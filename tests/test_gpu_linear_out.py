"""Results of a product that are given: those that carry a gradient cannot take what has none."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("native", [True, False])
def test_results_that_require_a_gradient(monkeypatch, native):
    import qtensor.functional as F
    from qtensor.linear import QTensorLinear
    if not native:
        monkeypatch.setattr(F, "_direct", None)
    weights = QTensorLinear(64, 16).quantize(torch.ones(16, 64, device="cuda"))
    x, leaf = torch.ones(3, 64, device="cuda"), torch.zeros(3, 16, device="cuda").requires_grad_()
    for out in (leaf, leaf * 2):
        with pytest.raises(RuntimeError, match="gradient"):
            weights.product(x, out=out)
        assert not out.any()
        with torch.no_grad():
            assert weights.product(x, out=out) is out
        assert bool((out == 64).all())
        with torch.no_grad():
            leaf.zero_()
