"""Rotary positions (qtensor.rotary, QTensorCache.write_turned) against their definition in 64 bits (oracle/rotary_ref.py).  On the way into the cache
they have to be turning, then writing, bit for bit."""
import math

import pytest
import torch

from oracle import rotary_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def Rotary():
    from qtensor.rotary import Rotary
    import qtensor.functional as F
    assert torch.cuda.is_available() and F.lib is not None
    return Rotary


def vectors(shape, dtype, seed):
    x = torch.randn(*shape, generator=torch.Generator().manual_seed(seed))
    x[..., ::7] *= 9.0
    return x.to(dtype)


def check(got, x, positions, rotary, back=False):
    want, size = R.turned(x, positions, rotary.frequencies.cpu(), rotary.dims, rotary.magnitude, rotary.interleaved, back)
    assert got.dtype == x.dtype and got.shape == x.shape
    off = (got.double().cpu() - want).abs()
    assert bool((off <= R.bounds(x.dtype, want, size)).all()), float((off - R.bounds(x.dtype, want, size)).max())
    assert torch.equal(got[..., rotary.dims:].cpu(), x[..., rotary.dims:])


SHAPES = [(64, 64), (128, 128), (128, 32), (80, 32), (96, 96), (7, 2), (34, 30), (33, 20), (256, 256), (2, 2), (100, 50), (1024, 1024), (1000, 998), (72, 36)]


@pytest.mark.parametrize("head_dim,dims", SHAPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_turning(Rotary, head_dim, dims, interleaved, dtype):
    for tokens, heads, kv_heads in ((1, 1, 1), (5, 4, 2), (37, 12, 3)):
        rotary = Rotary(dims, interleaved=interleaved, magnitude=1.25)
        q, k = vectors((tokens, heads, head_dim), dtype, 1), vectors((tokens, kv_heads, head_dim), dtype, 2)
        positions = 3 * torch.arange(tokens) - 4
        got = rotary.turn(q.cuda(), k.cuda(), positions.cuda())
        check(got[0], q, positions, rotary)
        check(got[1], k, positions, rotary)
        alone, nothing = rotary.turn(q.cuda(), None, positions.to(torch.int32).cuda())
        assert nothing is None and torch.equal(alone, got[0])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_far_positions_and_stretched_frequencies(Rotary, dtype):
    from qtensor.rotary import frequencies
    positions = torch.tensor([0, 1, 131071, 1048575, 2 ** 31 - 1, -(2 ** 31)])
    for kind in ("all", "base", "parts"):
        rotary = Rotary(64, frequencies=frequencies(64, 500000.0, 8.0, kind, original=4096))
        q = vectors((6, 4, 64), dtype, 3)
        check(rotary.turn(q.cuda(), None, positions.cuda())[0], q, positions, rotary)
        check(rotary.turn(q.cuda(), None, positions.to(torch.int32).cuda())[0], q, positions, rotary)
    far = torch.tensor([2 ** 40, -(2 ** 45), 5, 6, 7, 8])
    check(rotary.turn(q.cuda(), None, far.cuda())[0], q, far, rotary)


def test_sequences_strides_and_positions(Rotary):
    rotary = Rotary(48)
    for dtype in (torch.bfloat16, torch.float32):
        both = vectors((3, 11, 9, 64), dtype, 4)
        q, k = both.cuda()[:, :, :6], both.cuda()[:, :, 6:]                            # slices of one projection
        for positions in (torch.arange(11) + 5, torch.arange(33).view(3, 11) * 7, torch.arange(44).view(4, 11)[1:]):
            got = rotary.turn(q, k, positions.cuda())
            whole = positions.expand(3, 11)
            check(got[0], both[:, :, :6], whole, rotary)
            check(got[1], both[:, :, 6:], whole, rotary)
        across = both.cuda().transpose(1, 2).contiguous().transpose(1, 2)              # heads in front of tokens
        assert torch.equal(rotary.turn(across, None, positions.cuda())[0], rotary.turn(both.cuda(), None, positions.cuda())[0])
        odd = torch.full((3, 11, 9, 67), math.nan, dtype=dtype, device="cuda")
        odd[..., 1:65] = both.cuda()                                                   # not aligned
        assert torch.equal(rotary.turn(odd[..., 1:65], None, positions.cuda())[0], rotary.turn(both.cuda(), None, positions.cuda())[0])
        none = rotary.turn(q[:, :0], k[:, :0], positions[:, :0].cuda())
        assert none[0].shape == (3, 0, 6, 64) and none[1].shape == (3, 0, 3, 64)


def test_values_that_are_not_finite_stay_with_their_pairs(Rotary):
    for interleaved in (False, True):
        rotary = Rotary(32, interleaved=interleaved)
        q = vectors((4, 2, 40), torch.float32, 5)
        bad = q.clone()
        bad[1, 0, 3], bad[2, 1, 39], bad[3, 0, 20] = math.nan, math.inf, math.inf
        good, got = (rotary.turn(t.cuda(), None, torch.arange(4).cuda())[0].cpu() for t in (q, bad))
        partner = {3: 2, 20: 21} if interleaved else {3: 19, 20: 4}
        same = torch.ones(4, 2, 40, dtype=torch.bool)
        same[1, 0, 3] = same[1, 0, partner[3]] = same[2, 1, 39] = same[3, 0, 20] = same[3, 0, partner[20]] = False
        assert torch.equal(got[same], good[same]) and got[2, 1, 39] == math.inf
        assert bool(torch.isnan(got[1, 0, [3, partner[3]]]).all()) and not bool(torch.isfinite(got[3, 0, [20, partner[20]]]).any())


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gradients(Rotary, interleaved, dtype):
    rotary = Rotary(48, interleaved=interleaved, magnitude=0.75)
    shape_q, shape_k = (2, 19, 6, 64), (2, 19, 2, 64)
    q, k, dq, dk = (vectors(s, dtype, 6 + i) for i, s in enumerate((shape_q, shape_k, shape_q, shape_k)))
    positions = torch.arange(19) * 11
    a, b = q.cuda().requires_grad_(), k.cuda().requires_grad_()
    out = rotary.turn(a, b, positions.cuda())
    got = torch.autograd.grad(out, (a, b), (dq.cuda(), dk.cuda()))
    check(got[0], dq, positions, rotary, back=True)
    check(got[1], dk, positions, rotary, back=True)
    # against differences: turning is linear, so <turn(q + h e) - turn(q), dq> / h is <e, gradient> for any h
    if dtype == torch.float32:
        e = vectors(shape_q, dtype, 20)
        there = rotary.turn((q + 0.5 * e).cuda(), None, positions.cuda())[0].double() - rotary.turn((q - 0.5 * e).cuda(), None, positions.cuda())[0].double()
        left, right = (there * dq.cuda().double()).sum(), (e.cuda().double() * got[0].double()).sum()
        size = (there.abs() * dq.cuda().double().abs()).sum() + (q.abs().amax() * dq.abs().sum())
        assert abs(float(left - right)) <= float(size) * 8 * 2.0 ** -24
    # one of both, gradients of broadcast results, and a gradient of the gradient
    only = torch.autograd.grad(rotary.turn(a, k.cuda(), positions.cuda())[0], a, dq.cuda())[0]
    assert torch.equal(only, got[0])
    second = torch.autograd.grad(rotary.turn(q.cuda(), b, positions.cuda())[1], b, dk.cuda())[0]
    assert torch.equal(second, got[1])
    summed = torch.autograd.grad(rotary.turn(a, b, positions.cuda())[0].float().sum(), a)[0]
    check(summed, torch.ones(shape_q, dtype=dtype), positions, rotary, back=True)
    g = dq.cuda().requires_grad_()
    first, = torch.autograd.grad(rotary.turn(a, b, positions.cuda())[0], a, g, create_graph=True)
    again, = torch.autograd.grad(first, g, q.cuda())
    assert torch.equal(again, rotary.turn(q.cuda(), None, positions.cuda())[0])


def test_another_stream_and_a_captured_call(Rotary):
    rotary = Rotary(64)
    q, k, positions = vectors((40, 8, 64), torch.bfloat16, 8).cuda(), vectors((40, 2, 64), torch.bfloat16, 9).cuda(), torch.arange(40, device="cuda")
    want = rotary.turn(q, k, positions)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        got = rotary.turn(q, k, positions)
    stream.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph, at = torch.cuda.CUDAGraph(), positions.clone()
    with torch.cuda.graph(graph), torch.no_grad():
        out = rotary.turn(q, k, at)
    for n in range(3):
        at.copy_(positions + 100 * n)
        graph.replay()
        want = rotary.turn(q, k, positions + 100 * n)
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_refusals(Rotary):
    rotary = Rotary(32)
    q, at = torch.ones(5, 2, 64, device="cuda"), torch.arange(5, device="cuda")
    for bad in (q.double(), q.half(), q.cpu(), q[0], q[..., :30], q.transpose(0, 2), torch.ones(5, 2, 1026, device="cuda"), q[:, :0], q.view(1, 1, 5, 2, 64)):
        with pytest.raises((ValueError, RuntimeError)):
            rotary.turn(bad, None, at)
    for bad in (q.bfloat16(), q[:4], q[..., :32], q.view(1, 5, 2, 64)):
        with pytest.raises(ValueError):
            rotary.turn(q, bad, at)
    for bad in (at[:4], at.float(), at.cpu(), at.view(5, 1), torch.arange(10, device="cuda")[::2], at.to(torch.int16)):
        with pytest.raises(ValueError):
            rotary.turn(q, None, bad)
    rotary.frequencies = rotary.frequencies[:8]
    with pytest.raises(ValueError):
        rotary.turn(q, None, at)


# ------------------------------------------------------------------------------------------------ on the way into the cache
@pytest.mark.parametrize("dim,dims,blocksize,page_size", [(64, 64, 64, 16), (128, 128, 64, 64), (128, 64, 128, 32), (80, 32, 64, 16), (33, 20, 256, 16),
                                                          (2, 2, 64, 16), (192, 190, 64, 128), (256, 256, 256, 64), (200, 100, 128, 16)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_turned_into_the_cache_is_turned_then_written(Rotary, dim, dims, blocksize, page_size, interleaved, dtype):
    from qtensor.cache import QTensorCache
    rotary = Rotary(dims, interleaved=interleaved)
    lengths, news = [9, 40, 0, 17, 3], [9, 4, 0, 1, 5]                  # (the last one: longer than its sequence)
    rows, batch = sum(news), len(news)
    width = -(-max(lengths) // page_size)
    table = torch.randperm(batch * width + 2, generator=torch.Generator().manual_seed(1))[: batch * width].view(batch, width).to(torch.int32).cuda()
    table[1, -1] = -1                                                   # a page that is not there
    places = torch.tensor([n - a + i for n, a in zip(lengths, news) for i in range(a)] + [-1, -1, -1])
    counts, starts = torch.tensor(lengths, dtype=torch.int32).cuda(), torch.tensor([0, 9, 13, 13, 14, 19], dtype=torch.int32).cuda()
    for heads, kv_heads in ((4, 2), (7, 7), (1, 1), (24, 3)):
        q, k, v = (vectors((rows + 3, h, dim), dtype, 10 + i) for i, h in enumerate((heads, kv_heads, kv_heads)))
        for positions in (None, 5 * torch.arange(rows + 3) - 3):
            at = places if positions is None else positions
            caches = [QTensorCache(batch * width + 2, kv_heads, dim, page_size=page_size, blocksize=blocksize) for _ in range(2)]
            for c in caches:
                c.codes.fill_(0x11), c.scales.fill_(2.0)
            got = caches[0].write_turned(rotary, q.cuda(), k.cuda(), v.cuda(), table, counts, starts, positions=None if positions is None else positions.cuda())
            want, turned = rotary.turn(q.cuda(), k.cuda(), at.cuda())
            caches[1].write(turned, v.cuda(), table, counts, starts)
            assert torch.equal(caches[0].codes, caches[1].codes) and torch.equal(caches[0].scales, caches[1].scales)
            want[(places < 0).cuda()] = 0
            assert torch.equal(got, want)


@pytest.mark.parametrize("dim,dims,heads,kv_heads", [(128, 128, 56, 7), (80, 64, 90, 9), (256, 256, 30, 5), (33, 32, 220, 3)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_many_tokens_turned_into_the_cache(Rotary, dim, dims, heads, kv_heads, dtype):
    """As many as take the kernel's other tiles; rows behind the last sequence, a sequence that is shorter than its part."""
    from qtensor.cache import QTensorCache
    lengths, news = [403, 0, 17, 150, 4], [400, 0, 9, 150, 40]
    rows = sum(news) + 7
    width = -(-max(lengths) // 16)
    table = torch.randperm(5 * width, generator=torch.Generator().manual_seed(1)).view(5, width).to(torch.int32).cuda()
    table[3, 2] = 5 * width
    counts = torch.tensor(lengths, dtype=torch.int32).cuda()
    starts = torch.tensor([sum(news[:b]) for b in range(6)], dtype=torch.int32).cuda()
    places = torch.tensor([n - a + i for n, a in zip(lengths, news) for i in range(a)] + [-1] * 7)
    q, k, v = (vectors((rows, h, dim), dtype, 10 + i).cuda() for i, h in enumerate((heads, kv_heads, kv_heads)))
    assert q.numel() >= 2 ** 22 or dim < 128
    for interleaved in (False, True):
        rotary = Rotary(dims, interleaved=interleaved)
        caches = [QTensorCache(5 * width, kv_heads, dim, page_size=16) for _ in range(2)]
        got = caches[0].write_turned(rotary, q, k, v, table, counts, starts)
        want, turned = rotary.turn(q, k, places.cuda())
        caches[1].write(turned, v, table, counts, starts)
        want[(places < 0).cuda()] = 0
        assert torch.equal(got, want) and torch.equal(caches[0].codes, caches[1].codes) and torch.equal(caches[0].scales, caches[1].scales)


def test_a_token_of_each_sequence(Rotary):
    from qtensor.cache import QTensorCache
    rotary = Rotary(128)
    for dtype in (torch.bfloat16, torch.float32):
        lengths = torch.tensor([1, 70, 0, 500, 64], dtype=torch.int32).cuda()
        table = torch.arange(40, dtype=torch.int32).view(5, 8).cuda()
        q, k, v = (vectors((5, h, 128), dtype, 13 + i).cuda() for i, h in enumerate((32, 8, 8)))
        caches = [QTensorCache(40, 8, 128) for _ in range(2)]
        out = torch.full((7, 32, 128), 3.0, dtype=dtype, device="cuda")
        got = caches[0].write_turned(rotary, q, k, v, table, lengths, out=out[1:6])
        want, turned = rotary.turn(q, k, (lengths - 1).long())
        caches[1].write(turned, v, table, lengths)
        want[2] = 0
        assert torch.equal(got, want) and bool((out[0] == 3).all()) and bool((out[6] == 3).all())
        assert torch.equal(caches[0].codes, caches[1].codes) and torch.equal(caches[0].scales, caches[1].scales)
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            captured = caches[0].write_turned(rotary, q, k, v, table, lengths)
        for n in range(3):
            lengths += 1
            graph.replay()
            want, turned = rotary.turn(q, k, (lengths - 1).long())
            caches[1].write(turned, v, table, lengths)
            assert torch.equal(captured, want) and torch.equal(caches[0].codes, caches[1].codes) and torch.equal(caches[0].scales, caches[1].scales)


def test_refusals_of_the_cache(Rotary):
    from qtensor.cache import QTensorCache
    cache, rotary = QTensorCache(4, 2, 64), Rotary(64)
    q, k = torch.ones(3, 4, 64, device="cuda"), torch.ones(3, 2, 64, device="cuda")
    table, lengths = torch.zeros(3, 1, dtype=torch.int32, device="cuda"), torch.ones(3, dtype=torch.int32, device="cuda")
    good = dict(rotary=rotary, q=q, keys=k, values=k, table=table, lengths=lengths)
    cache.write_turned(**good)
    for bad in (dict(q=q.bfloat16()), dict(q=q[:2]), dict(keys=q), dict(values=k.double()), dict(rotary=Rotary(66)), dict(out=q), dict(out=q[:2]),
                dict(positions=torch.arange(2, device="cuda")), dict(positions=torch.arange(3.0, device="cuda")), dict(positions=torch.arange(6, device="cuda")[::2]),
                dict(table=table[:2]), dict(lengths=lengths.long()), dict(q=q.clone().requires_grad_()), dict(q=q[..., :32])):
        with pytest.raises((ValueError, RuntimeError)):
            cache.write_turned(**{**good, **bad})
