"""Tensors that have taken the place of what weights, caches and rotary positions were made of: as many numbers in another order are refused, not computed with."""
import pytest
import torch

pytestmark = pytest.mark.gpu

CHANGES = [lambda t: t.flatten(), lambda t: t.unsqueeze(0), lambda t: t.view(*t.shape[:-1], 2, -1), lambda t: t.transpose(0, 1).contiguous(), lambda t: t.transpose(-1, -2).contiguous()]


@pytest.mark.parametrize("name", ["codes", "scales"])
@pytest.mark.parametrize("change", CHANGES)
def test_weights(name, change):
    from qtensor.linear import QTensorLinear
    weights = QTensorLinear(300, 50).quantize(torch.ones(50, 300, device="cuda"))
    x = torch.ones(3, 300, device="cuda")
    weights.product(x)
    setattr(weights, name, change(getattr(weights, name)))
    with pytest.raises(ValueError):
        weights.product(x)


@pytest.mark.parametrize("name", ["codes", "scales"])
@pytest.mark.parametrize("change", CHANGES)
def test_caches(name, change):
    from qtensor.cache import QTensorCache
    from qtensor.rotary import Rotary
    cache, rotary = QTensorCache(3, 4, 130), Rotary(64)
    q, k, table, lengths = (torch.ones(1, 4, 130, device="cuda"), torch.ones(1, 4, 130, device="cuda"), torch.zeros(1, 1, dtype=torch.int32, device="cuda"),
                            torch.ones(1, dtype=torch.int32, device="cuda"))
    totals = cache.totals(table)
    cache.write(k, k, table, lengths)
    setattr(cache, name, change(getattr(cache, name)))
    for call in (lambda: cache.write(k, k, table, lengths), lambda: cache.read(table, lengths), lambda: cache.attend(q, table, lengths),
                 lambda: cache.write_turned(rotary, q, k, k, table, lengths), lambda: cache.weigh(totals, q, table, lengths), lambda: cache.evict(totals, table, lengths, 3)):
        with pytest.raises(ValueError):
            call()


def test_frequencies():
    from qtensor.rotary import Rotary
    q, at = torch.ones(5, 2, 64, device="cuda"), torch.arange(5, device="cuda")
    for change in (lambda t: t.unsqueeze(0), lambda t: t.view(2, -1), lambda t: t.float(), lambda t: t[:8]):
        rotary = Rotary(32)
        rotary.frequencies = change(rotary.frequencies)
        with pytest.raises(ValueError):
            rotary.turn(q, None, at)
