"""Projections in 4 bits, rotary positions and eviction where no GPU is involved: construction, refusals, the oracles' own pins."""
import math

import pytest
import torch

from oracle import evict_ref as E
from oracle import linear_ref as L
from oracle import rotary_ref as R


def test_projections_are_constructed_and_refused():
    from qtensor.linear import QTensorLinear
    w = QTensorLinear(130, 33, blocksize=128, device="cpu")
    assert w.codes.shape == (3, 2, 1024) and w.scales.shape == (3, 2, 16) and w._ref().inputs == 130
    for bad in (dict(blocksize=32), dict(blocksize=512), dict(inputs=0), dict(outputs=0), dict(inputs=2 ** 24 + 1), dict(outputs=-1)):
        with pytest.raises(ValueError):
            QTensorLinear(**{**dict(inputs=64, outputs=64, device="cpu"), **bad})
    for call in (lambda: w.quantize(torch.zeros(33, 130)), lambda: w.dequantize(), lambda: w.product(torch.zeros(1, 130))):
        with pytest.raises(RuntimeError):
            call()
    for name in ("codes", "scales"):
        for change in (lambda t: t[:2], lambda t: t.double(), lambda t: t[..., ::2], lambda t: t.flatten(), lambda t: t.transpose(0, 1)):
            w = QTensorLinear(130, 33, device="cpu")
            setattr(w, name, change(getattr(w, name)))
            with pytest.raises(ValueError):
                w._ref()
    w = QTensorLinear(130, 33, device="cpu")
    for key, value in (("inputs", 131), ("blocksize", 128), ("codes", w.codes[:1]), ("scales", w.scales.double())):
        with pytest.raises(ValueError):
            QTensorLinear(130, 33, device="cpu").load_state_dict({**w.state_dict(), key: value})


def test_rotary_is_constructed_and_refused():
    from qtensor.rotary import Rotary, frequencies
    r = Rotary(6, base=100.0, device="cpu")
    assert torch.equal(r.frequencies, torch.tensor([1.0, 100.0 ** (-1 / 3), 100.0 ** (-2 / 3)], dtype=torch.float64))
    assert Rotary(4, frequencies=[0.5, 0.25], device="cpu").frequencies.tolist() == [0.5, 0.25]
    for bad in (dict(dims=0), dict(dims=7), dict(dims=1026), dict(dims=4, frequencies=[1.0]), dict(dims=4, frequencies=[1.0, math.nan]),
                dict(dims=4, magnitude=math.inf)):
        with pytest.raises(ValueError):
            Rotary(**{**dict(device="cpu"), **bad})
    with pytest.raises(RuntimeError):
        r.turn(torch.zeros(1, 1, 6), None, torch.zeros(1, dtype=torch.int64))
    assert frequencies(4, 100.0, 4.0) == [0.25, 0.025]
    assert frequencies(4, 100.0, 4.0, "base") == pytest.approx([1.0, 1600.0 ** -0.5])
    # of 1000 places: the first turns 159 times and stays, the last one 0.016 times and is slowed down, the one between 1.59 times: half way from 1 to 2.18
    assert frequencies(6, 1e6, 4.0, "parts", original=1000, slow=1.0, fast=2.1830988618)[1] == pytest.approx(0.5 * (0.01 + 0.01 / 4))
    got = frequencies(6, 1e6, 4.0, "parts", original=1000)
    assert got[0] == 1.0 and got[2] == pytest.approx(1e-4 / 4)
    for bad in (dict(dims=3), dict(dims=4, stretch="x"), dict(dims=4, stretch="parts"), dict(dims=4, base=0.0), dict(dims=4, factor=math.inf),
                dict(dims=4, stretch="parts", original=10, slow=5.0, fast=2.0)):
        with pytest.raises(ValueError):
            frequencies(**bad)


def test_eviction_computes_nowhere_else():
    from qtensor.cache import QTensorCache
    from qtensor.rotary import Rotary
    c = QTensorCache(3, 2, 64, device="cpu")
    table, lengths, x = torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32), torch.zeros(1, 2, 64)
    totals = c.totals(table)
    assert totals.shape == (1, 2, 64) and not totals.any()
    for call in (lambda: c.weigh(totals, x, table, lengths), lambda: c.evict(totals, table, lengths, 3),
                 lambda: c.write_turned(Rotary(64, device="cpu"), x, x, x, table, lengths)):
        with pytest.raises(RuntimeError):
            call()


def test_the_oracles_turn_weigh_and_choose():
    x = torch.tensor([[[3.0, 4.0, 5.0, 6.0, 7.0]]])
    quarter = [math.pi / 2, 0.0]
    got, size = R.turned(x, torch.tensor([1]), quarter, 4)
    assert torch.allclose(got, torch.tensor([[[-5.0, 4.0, 3.0, 6.0, 7.0]]], dtype=torch.float64), atol=1e-6)
    got, _ = R.turned(x, torch.tensor([1]), quarter, 4, interleaved=True)
    assert torch.allclose(got, torch.tensor([[[-4.0, 3.0, 5.0, 6.0, 7.0]]], dtype=torch.float64), atol=1e-6)
    back, _ = R.turned(got, torch.tensor([1]), quarter, 4, interleaved=True, back=True)
    assert torch.allclose(back, x.double(), atol=1e-6)
    keys = torch.zeros(4, 1, 2, dtype=torch.float64)
    totals, _ = E.weigh(torch.ones(2, 3, 2), [1, 3], keys, 1.0)
    assert torch.allclose(totals, 3 * torch.tensor([[0.5 + 0.25, 0.5 + 0.25, 0.25, 0.25]], dtype=torch.float64))
    totals, _ = E.weigh(torch.ones(1, 1, 2), [3], keys, 1.0, window=2, sinks=1, there=torch.tensor([True, True, False, True]))
    assert torch.allclose(totals, torch.tensor([[0.5, 0.0, 0.0, 0.5]], dtype=torch.float64))
    assert E.evict([1.0, 5.0, 5.0, 0.0, math.nan], 5, 3) == ([1, 2, 4], [0, 1, 2])
    assert E.evict([1.0, 5.0, 5.0, 0.0, 2.0], 5, 2, recent=1, sinks=1) == ([0, 4], [0, 1])
    assert E.evict([1.0, 0.0, -0.0, 0.0], 4, 2) == ([0, 1], [0, 1])
    assert E.evict([1.0, 9.0, 9.0, 9.0], 4, 2, there=[False, True, False, True]) == ([1, 3], [1, 3])
    assert E.evict([], 0, 2) == ([], [])


def test_the_oracle_multiplies():
    w, x = torch.tensor([[6.0, 3.0, -1.0]]), torch.tensor([[1.0, 2.0, 4.0]])
    got, size = L.product(x, w, 64, torch.tensor([0.5]))
    assert float(got) == 8.5 and float(size) == 16.5
