"""What the C entry points for projections, rotary positions and eviction refuse before anything is launched: descriptions of host memory that is never read."""
import ctypes as ct

import pytest
import torch

import qtensor.functional as F
from qtensor import cache as C
from qtensor import linear as L
from qtensor import rotary as R

MEMORY = torch.zeros(4096, dtype=torch.float64)
AT = MEMORY.data_ptr()                              # (aligned to 64 bytes)


def refused(name, *arguments):
    assert getattr(F.lib, "qtensor_hip_" + name)(*arguments) in (None, 0)
    return F.lib.qtensor_hip_last_error() != 0


def linear(**change):
    return L._Linear(**{**dict(codes=AT, scales=AT, inputs=256, outputs=16, blocksize=64), **change})


@pytest.mark.parametrize("change", [dict(codes=None), dict(scales=None), dict(codes=AT + 8), dict(scales=AT + 4), dict(inputs=0), dict(inputs=2 ** 24 + 1), dict(outputs=-1),
                                    dict(blocksize=32), dict(blocksize=100)])
def test_weights(change):
    call = L._Call(AT, None, AT, 256, 16, 1, 0, 0)
    assert refused("linear_product", linear(**change), call, None)
    assert refused("linear_quantize", linear(**change), AT, 0, 256, None) and refused("linear_dequantize", linear(**change), AT, 0, 256, None)


def test_weights_to_encode():
    for address, bf16, stride in ((None, 0, 256), (AT + 2, 0, 256), (AT + 1, 1, 256), (AT, 0, -256)):
        assert refused("linear_quantize", linear(), address, bf16, stride, None)


@pytest.mark.parametrize("change", [dict(x=None), dict(out=None), dict(x=AT + 2), dict(out=AT + 2), dict(bias=AT + 2), dict(tokens=-1), dict(tokens=2 ** 31), dict(x_stride=-1),
                                    dict(out_stride=15), dict(x=AT + 1, is_bf16=1), dict(bias=AT + 1, bias_is_bf16=1)])
def test_products(change):
    call = L._Call(**{**dict(x=AT, bias=None, out=AT, x_stride=256, out_stride=16, tokens=1, is_bf16=0, bias_is_bf16=0), **change})
    assert refused("linear_product", linear(), call, None)


def angles(**change):
    return R._Rotary(**{**dict(frequencies=AT, magnitude=1.0, dims=64, interleaved=0, back=0), **change})


ANGLES = [dict(frequencies=None), dict(frequencies=AT + 4), dict(dims=0), dict(dims=7), dict(dims=66)]


@pytest.mark.parametrize("change", ANGLES)
def test_angles(change):
    call = R._Call((R._Part * 2)(R._Part(AT, AT, 0, 64, 64, 0, 64, 64, 1)), 1, 64, 0, 0, 1, 1, 0, AT)
    assert refused("rotary_turn", angles(**change), call, None)


@pytest.mark.parametrize("change", [dict(parts=0), dict(parts=3), dict(head_dim=0), dict(head_dim=1025), dict(head_dim=63), dict(batch=-1), dict(tokens=-1),
                                    dict(batch=2 ** 40, tokens=2 ** 40), dict(positions=None), dict(positions=AT + 2), dict(positions=AT + 4, long_positions=1), dict(parts=2)])
def test_vectors_to_turn(change):
    call = dict(part=(R._Part * 2)(R._Part(AT, AT, 0, 64, 64, 0, 64, 64, 1)), parts=1, head_dim=64, is_bf16=0, long_positions=0, batch=1, tokens=1, position_batch=0,
                positions=AT)
    assert refused("rotary_turn", angles(), R._Call(**{**call, **change}), None)


@pytest.mark.parametrize("change", [dict(from_=None), dict(to=None), dict(from_=AT + 2), dict(to=AT + 2), dict(heads=0), dict(heads=32768)])
def test_parts_to_turn(change):
    part = R._Part(**{**dict(from_=AT, to=AT, from_batch=0, from_token=64, from_head=64, to_batch=0, to_token=64, to_head=64, heads=1), **change})
    assert refused("rotary_turn", angles(), R._Call((R._Part * 2)(part), 1, 64, 0, 0, 1, 1, 0, AT), None)


@pytest.fixture
def held():
    cache = C.QTensorCache(4, 2, 64, page_size=16, device="cpu")
    table, lengths = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    return cache, cache._places(table, lengths, None, 1), (table, lengths)


def vectors(address=AT, bf16=0):
    return C._Vectors(address, bf16, 128, 64)


def test_what_is_turned_into_the_cache(held):
    cache, places, _ = held
    def call(rotary=angles(), q=vectors(), out=vectors(), heads=4, keys=vectors(), values=vectors(), positions=None, long_positions=0):
        return refused("cache_write_turned", cache._ref(), places, rotary, q, out, heads, keys, values, positions, long_positions, None)
    for change in ANGLES:
        assert call(rotary=angles(**change))
    for name in ("q", "out", "keys", "values"):
        for bad in (None, vectors(None), vectors(AT + 2), vectors(AT, 1)):
            assert call(**{name: bad})
    assert call(heads=0) and call(heads=32768) and call(positions=AT + 2) and call(positions=AT + 4, long_positions=1)


def test_what_is_weighed(held):
    cache, places, _ = held
    room = F.lib.qtensor_hip_cache_weigh_workspace(cache._ref(), places, 4)
    assert room > 0
    for heads in (0, 3, -2):
        assert refused("cache_weigh_workspace", cache._ref(), places, heads)
    def call(q=vectors(), heads=4, scale=0.125, window=0, sinks=0, totals=AT, of_sequence=64, of_head=32, workspace=AT, size=room):
        return refused("cache_weigh", cache._ref(), places, q, heads, scale, window, sinks, totals, of_sequence, of_head, workspace, size, None)
    for bad in (dict(q=None), dict(q=vectors(None)), dict(q=vectors(AT + 2)), dict(q=vectors(AT + 1, 1)), dict(heads=3), dict(heads=0), dict(heads=32768), dict(scale=float("inf")),
                dict(scale=float("nan")), dict(window=-1), dict(sinks=1), dict(window=4, sinks=-1), dict(totals=None), dict(totals=AT + 2), dict(of_sequence=-1), dict(of_head=-1),
                dict(workspace=None), dict(workspace=AT + 8), dict(size=room - 1)):
        assert call(**bad), bad


def test_more_rows_than_are_weighed_in_a_call(held):
    cache, _, (table, lengths) = held
    starts = torch.zeros(2, dtype=torch.int32)
    places = cache._places(table, lengths, starts, 2 ** 26)
    room = F.lib.qtensor_hip_cache_weigh_workspace(cache._ref(), places, 4)
    assert refused("cache_weigh", cache._ref(), places, vectors(), 4, 0.125, 0, 0, AT, 64, 32, AT, room, None)


def test_what_is_evicted(held):
    cache, places, (_, lengths) = held
    room = F.lib.qtensor_hip_cache_evict_workspace(cache._ref(), places, 8)
    assert room > 0 and refused("cache_evict_workspace", cache._ref(), places, 0)
    def call(totals=AT, of_sequence=64, of_head=32, keep=8, recent=0, sinks=0, new=AT, workspace=AT, size=room):
        return refused("cache_evict", cache._ref(), places, totals, of_sequence, of_head, keep, recent, sinks, new, workspace, size, None)
    for bad in (dict(totals=None), dict(totals=AT + 2), dict(of_sequence=-1), dict(of_head=-1), dict(keep=0), dict(keep=-3), dict(recent=9), dict(sinks=9), dict(recent=5, sinks=4),
                dict(recent=-1), dict(sinks=-1), dict(recent=2 ** 62, sinks=2 ** 62, keep=2 ** 63 - 1), dict(new=None), dict(new=AT + 2), dict(new=lengths.data_ptr()),
                dict(workspace=None), dict(workspace=AT + 8), dict(size=room - 1)):
        assert call(**bad), bad
