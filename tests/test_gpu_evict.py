"""What of a 4-bit attention cache is kept (QTensorCache.weigh, evict) against the definitions in 64 bits (oracle/evict_ref.py)."""
import math

import pytest
import torch

from oracle import cache_ref as C
from oracle import evict_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def Cache():
    from qtensor.cache import QTensorCache
    import qtensor.functional as F
    assert torch.cuda.is_available() and F.lib is not None
    return QTensorCache


def vectors(shape, dtype, seed):
    x = torch.randn(*shape, generator=torch.Generator().manual_seed(seed))
    x[..., ::13] *= 3.0
    return x.to(dtype)


def filled(Cache, lengths, kv_heads, dim, dtype, page_size=16, blocksize=64, spare=3, seed=0, wide=0):
    """(cache, table, lengths, keys, values) with the pages of all sequences in random order."""
    g = torch.Generator().manual_seed(seed)
    width = max(1, max(-(-n // page_size) for n in lengths)) + wide
    pages = len(lengths) * width + spare
    table = torch.randperm(pages, generator=g)[: len(lengths) * width].view(len(lengths), width).to(torch.int32).cuda()
    cache = Cache(pages, kv_heads, dim, page_size=page_size, blocksize=blocksize)
    counts = torch.tensor(lengths, dtype=torch.int32).cuda()
    k, v = (vectors((sum(lengths), kv_heads, dim), dtype, seed + i) for i in (1, 2))
    starts = torch.tensor([sum(lengths[:b]) for b in range(len(lengths) + 1)], dtype=torch.int32).cuda()
    cache.write(k.cuda(), v.cuda(), table, counts, starts)
    return cache, table, counts, k.split(lengths), v.split(lengths)


def check_weights(cache, got, before, q, lengths, news, keys, blocksize, scale=None, window=None, sinks=0, there=None):
    dim, at = q.shape[2], 0
    scale = 1 / math.sqrt(dim) if scale is None else scale
    for b, (n, new) in enumerate(zip(lengths, news)):
        want, spread = R.weigh(q[at:at + new], range(n - new, n), C.held(keys[b], blocksize), scale, window, sinks, None if there is None else there[b])
        rows = new * q.shape[1] // cache.kv_heads
        off = (got[b, :, :n].double().cpu() - before[b, :, :n].double() - want).abs()
        limit = R.bound(dim, rows, want, spread) + 2.0 ** -23 * (before[b, :, :n].double().abs() + want)
        assert bool((off <= limit).all()), f"sequence {b}: off by {float((off / limit).max()):.3g} of the bound"
        assert torch.equal(got[b, :, n:].cpu(), before[b, :, n:])
        at += new


@pytest.mark.parametrize("dim,blocksize,page_size", [(64, 64, 16), (128, 64, 64), (128, 128, 32), (80, 64, 16), (33, 256, 16), (1, 64, 16), (192, 64, 128),
                                                     (256, 64, 16), (256, 256, 64), (200, 128, 16), (96, 64, 4096)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_weights_of_a_token_of_each_sequence(Cache, dim, blocksize, page_size, dtype):
    lengths = [1, 70, 15, 300, 64, 17]
    for kv_heads, heads in ((2, 8), (3, 3), (1, 24)):
        cache, table, counts, keys, _ = filled(Cache, lengths, kv_heads, dim, dtype, page_size, blocksize)
        q = vectors((6, heads, dim), dtype, 9)
        totals = torch.rand(6, kv_heads, table.shape[1] * page_size + 5, generator=torch.Generator().manual_seed(3))
        got = totals.cuda()
        assert cache.weigh(got, q.cuda(), table, counts) is got
        check_weights(cache, got, totals, q, lengths, [1] * 6, keys, blocksize)


@pytest.mark.parametrize("dim", [64, 80, 128, 256])
@pytest.mark.parametrize("window,sinks", [(None, 0), (1, 0), (20, 0), (33, 4), (7, 50), (2 ** 31 - 1, 0)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_weights_of_pieces_of_prompts(Cache, dim, window, sinks, dtype):
    lengths, news = [90, 33, 1, 140, 0, 64], [90, 5, 1, 17, 0, 33]
    for kv_heads, heads in ((2, 6), (1, 1)):
        cache, table, counts, keys, _ = filled(Cache, lengths, kv_heads, dim, dtype)
        q = vectors((sum(news) + 2, heads, dim), dtype, 9)          # (the last two are of no sequence)
        starts = torch.tensor([sum(news[:b]) for b in range(7)], dtype=torch.int32).cuda()
        totals = cache.totals(table)
        cache.weigh(totals, q.cuda(), table, counts, starts, scale=0.2, window=window, sinks=sinks)
        check_weights(cache, totals, torch.zeros(totals.shape), q, lengths, news, keys, 64, 0.2, window, sinks)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_weights_over_long_sequences(Cache, dtype):
    """Rows that are cut into parts, of one query and of several; what is there already is added to."""
    lengths = [5000, 9, 2111]
    cache, table, counts, keys, _ = filled(Cache, lengths, 2, 128, dtype, 64)
    for news in ([1, 1, 1], [40, 9, 3]):
        q = vectors((sum(news), 4, 128), dtype, 9)
        starts = None if max(news) == 1 else torch.tensor([sum(news[:b]) for b in range(4)], dtype=torch.int32).cuda()
        totals = cache.totals(table)
        cache.weigh(totals, q.cuda(), table, counts, starts)
        check_weights(cache, totals, torch.zeros(totals.shape), q, lengths, news, keys, 64)
        once = totals.clone()
        cache.weigh(totals, q.cuda(), table, counts, starts)
        assert torch.equal(totals, once + once)                     # (the same sum again, every time)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_weights_with_room_for_many_more_tokens(Cache, dim, dtype):
    """A table that has room for so many tokens that scores are worked out twice, or that every wave has tokens of its own."""
    lengths = [300]
    cache, table, counts, keys, _ = filled(Cache, lengths, 1, dim, dtype, 4096)
    table = torch.cat([table, torch.full((1, 2099), -1, dtype=torch.int32, device="cuda")], 1)
    q = vectors((1, 16, dim), dtype, 9)
    totals = torch.rand(1, 1, table.shape[1] * 4096, generator=torch.Generator().manual_seed(3))
    for window, sinks in ((None, 0), (100, 7)):
        got = cache.weigh(totals.cuda(), q.cuda(), table, counts, window=window, sinks=sinks)
        check_weights(cache, got, totals, q, lengths, [1], keys, 64, window=window, sinks=sinks)
    lengths, news = [200, 33, 0, 64, 1, 100, 90, 300], [40, 5, 0, 64, 1, 100, 2, 3]
    cache, table, counts, keys, _ = filled(Cache, lengths, 8, dim, dtype, 16, wide=500)
    q = vectors((sum(news), 16, dim), dtype, 9)
    starts = torch.tensor([sum(news[:b]) for b in range(9)], dtype=torch.int32).cuda()
    for window, sinks in ((None, 0), (30, 20)):
        totals = cache.weigh(cache.totals(table), q.cuda(), table, counts, starts, window=window, sinks=sinks)
        check_weights(cache, totals, torch.zeros(totals.shape), q, lengths, news, keys, 64, window=window, sinks=sinks)


@pytest.mark.parametrize("heads,kv_heads", [(17, 1), (40, 2), (130, 1), (16, 16), (15, 5)])
def test_weights_of_groups_of_all_sizes(Cache, heads, kv_heads):
    lengths = [1, 70, 300]
    cache, table, counts, keys, _ = filled(Cache, lengths, kv_heads, 64, torch.bfloat16)
    q = vectors((3, heads, 64), torch.bfloat16, 9)
    totals = cache.weigh(cache.totals(table), q.cuda(), table, counts)
    check_weights(cache, totals, torch.zeros(totals.shape), q, lengths, [1] * 3, keys, 64)
    news = [1, 5, 40]
    q = vectors((46, heads, 64), torch.bfloat16, 9)
    totals = cache.weigh(cache.totals(table), q.cuda(), table, counts, torch.tensor([0, 1, 6, 46], dtype=torch.int32).cuda())
    check_weights(cache, totals, torch.zeros(totals.shape), q, lengths, news, keys, 64)


def test_weights_are_those_of_attention(Cache):
    """Values that are 1 for one token at a time: attention gives its weight."""
    cache, table, counts, keys, _ = filled(Cache, [37], 1, 64, torch.float32)
    q, starts = vectors((5, 3, 64), torch.float32, 4).cuda(), torch.tensor([0, 5], dtype=torch.int32).cuda()
    totals = cache.weigh(cache.totals(table), q, table, counts, starts)
    for t in (0, 20, 33, 36):
        v = torch.zeros(37, 1, 64)
        v[t] = 6.0
        cache.write(keys[0].cuda(), v.cuda(), table, counts, torch.tensor([0, 37], dtype=torch.int32).cuda())
        out = cache.attend(q, table, counts, starts)
        assert abs(float(out[..., 0].double().sum()) / 6 - float(totals[0, 0, t])) <= 15 * 2.0 ** -16


def test_tokens_that_are_not_there(Cache):
    lengths, news = [100, 40, 64], [3, 1, 64]
    cache, table, counts, keys, _ = filled(Cache, lengths, 2, 64, torch.bfloat16)
    table[0, 1], table[0, 6], table[1, :], table[2, 0] = -1, cache.pages, -7, 2 ** 31 - 1
    there = [torch.ones(n, dtype=torch.bool) for n in lengths]
    there[0][16:32], there[0][96:], there[1][:], there[2][:16] = False, False, False, False
    q = vectors((sum(news), 4, 64), torch.bfloat16, 9)
    starts = torch.tensor([0, 3, 4, 68], dtype=torch.int32).cuda()
    totals = cache.totals(table)
    cache.weigh(totals, q.cuda(), table, counts, starts)
    check_weights(cache, totals, torch.zeros(totals.shape), q, lengths, news, keys, 64, there=there)
    longer = counts + 40                                            # places behind the table
    totals = cache.totals(table[:, :2])
    cache.weigh(totals, q[:3].cuda(), table[:, :2], longer)
    assert bool(torch.isfinite(totals).all()) and not totals[1].any() and not totals[2, :, :16].any()
    assert torch.allclose(totals[0].sum(-1).cpu(), torch.full((2,), 2.0))
    short = torch.tensor([1, 0, -5], dtype=torch.int32).cuda()      # sequences shorter than their part of the call
    totals = cache.totals(table)
    cache.weigh(totals, q.cuda(), table, short, starts)
    assert totals[0, :, 0].tolist() == [2.0, 2.0] and float(totals.sum()) == 4.0


def test_values_that_are_not_finite(Cache):
    """A key that is not finite makes the weights of those that see it NaN, and of nobody else; so does a query of its tokens."""
    for dtype in (torch.bfloat16, torch.float32):
        cache, table, counts, keys, values = filled(Cache, [50, 30], 2, 64, dtype)
        k = keys[0].clone()
        k[40, 1, 5] = math.nan
        cache.write(k.cuda(), values[0].cuda(), table[:1], counts[:1], torch.tensor([0, 50], dtype=torch.int32).cuda())
        q = vectors((50 + 30, 4, 64), dtype, 9)
        q[60, 3, 7] = math.inf
        starts = torch.tensor([0, 50, 80], dtype=torch.int32).cuda()
        totals = cache.weigh(cache.totals(table), q.cuda(), table, counts, starts).cpu()
        assert bool(torch.isnan(totals[0, 1, :50]).all()) and bool(torch.isfinite(totals[0, 0]).all())
        assert bool(torch.isnan(totals[1, 1, :11]).all()) and bool(torch.isfinite(totals[1, 1, 11:]).all()) and bool(torch.isfinite(totals[1, 0]).all())
        few = cache.weigh(cache.totals(table), q[30:40].cuda(), table, counts - torch.tensor([10, 0], dtype=torch.int32).cuda(),
                          torch.tensor([0, 10, 10], dtype=torch.int32).cuda())
        assert bool(torch.isfinite(few).all()) and float(few.sum()) > 39.9        # (token 40 is seen by none of these)


# ------------------------------------------------------------------------------------------------ eviction
def everything(cache, table, lengths):
    rows = int(lengths.clamp(min=0).sum())
    starts = torch.cat([torch.zeros(1, dtype=torch.int32, device="cuda"), lengths.clamp(min=0).cumsum(0).to(torch.int32)])
    k, v = cache.read(table, lengths, starts, tokens=rows)
    return k.cpu().split(lengths.clamp(min=0).tolist()), v.cpu().split(lengths.clamp(min=0).tolist())


def check_evicted(cache, table, counts, totals, keep, recent, sinks, there=None):
    lengths = counts.tolist()
    room = table.shape[1] * cache.page_size
    keys, values = everything(cache, table, counts.clamp(max=room))
    before, whole = totals.cpu(), [cache.codes.clone(), cache.scales.clone()]
    got = cache.evict(totals, table, counts, keep, recent=recent, sinks=sinks)
    assert got.dtype == torch.int32 and counts.tolist() == lengths
    after_k, after_v = everything(cache, table, counts.clamp(max=room))
    expected = before.clone()
    for b, n in enumerate(lengths):
        n_here = min(max(n, 0), room)
        want = keys[b].clone(), values[b].clone()
        to = []
        for h in range(cache.kv_heads):
            is_there = [t < n_here and (there is None or bool(there[b][t])) for t in range(max(n, 0))]
            come, to = R.evict(before[b, h].tolist() + [0.0] * max(0, n), max(n, 0), keep, recent, sinks, is_there)
            for old, new in zip((keys[b], values[b]), want):
                new[to, h] = old[come, h]
            expected[b, h, to] = before[b, h, come]
        assert int(got[b]) == (to[-1] + 1 if to else 0)
        assert torch.equal(torch.nan_to_num(after_k[b], nan=77.0), torch.nan_to_num(want[0], nan=77.0))
        assert torch.equal(torch.nan_to_num(after_v[b], nan=77.0), torch.nan_to_num(want[1], nan=77.0))
    assert torch.equal(torch.nan_to_num(totals.cpu(), nan=77.0), torch.nan_to_num(expected, nan=77.0))
    used = torch.zeros(cache.pages, dtype=torch.bool)
    used[[int(p) for p in table.flatten().tolist() if 0 <= p < cache.pages]] = True
    assert torch.equal(cache.codes[:, ~used.cuda()], whole[0][:, ~used.cuda()]) and torch.equal(cache.scales[:, ~used.cuda()], whole[1][:, ~used.cuda()])
    return got


@pytest.mark.parametrize("dim,blocksize,page_size", [(64, 64, 16), (128, 64, 64), (33, 256, 16), (1, 64, 16), (192, 64, 128), (256, 256, 64), (200, 128, 32)])
@pytest.mark.parametrize("keep,recent,sinks", [(1, 0, 0), (40, 0, 0), (40, 16, 4), (40, 40, 0), (40, 0, 40), (1000, 10, 10), (2 ** 40, 2 ** 39, 2 ** 39)])
def test_tokens_with_the_largest_totals_stay(Cache, dim, blocksize, page_size, keep, recent, sinks):
    lengths = [1, 70, 40, 300, 0, 41, 39]
    cache, table, counts, _, _ = filled(Cache, lengths, 2, dim, torch.bfloat16, page_size, blocksize, wide=1)
    totals = torch.rand(7, 2, table.shape[1] * page_size + 3, generator=torch.Generator().manual_seed(5))
    check_evicted(cache, table, counts, totals.cuda(), keep, recent, sinks)


def test_ties_zeroes_and_totals_that_are_not_finite(Cache):
    lengths = [200, 200, 200, 200, 200]
    cache, table, counts, _, _ = filled(Cache, lengths, 2, 64, torch.bfloat16)
    totals = torch.zeros(5, 2, table.shape[1] * 16)
    totals[0, 0, 50:60] = 1.0
    totals[1] = (torch.arange(208) % 7).float()
    totals[2] = torch.randn(2, 208, generator=torch.Generator().manual_seed(6))
    totals[2, :, 3], totals[2, :, 9], totals[2, 0, 100:140], totals[2, 1, 11] = math.inf, -math.inf, math.nan, -math.nan
    totals[3, :, ::2] = -0.0
    totals[4] = -math.inf
    for keep, recent, sinks in ((30, 0, 0), (64, 10, 3), (199, 0, 1)):
        check_evicted(cache, table, counts, totals.cuda(), keep, recent, sinks)


def test_places_that_are_empty(Cache):
    lengths = [100, 90, 64, 400, -3]
    cache, table, counts, _, _ = filled(Cache, [100, 90, 64, 112, 0], 3, 64, torch.float32)
    counts = torch.tensor(lengths, dtype=torch.int32).cuda()        # (the fourth is longer than the table)
    table[0, 0], table[0, 3], table[1, 4], table[2, :] = -1, cache.pages + 5, -2, -1
    there = [torch.ones(max(n, 0), dtype=torch.bool) for n in lengths]
    there[0][:16], there[0][48:64], there[1][64:80], there[2][:] = False, False, False, False
    totals = torch.rand(5, 3, table.shape[1] * 16, generator=torch.Generator().manual_seed(7))
    for keep, recent, sinks in ((200, 0, 0), (50, 20, 20), (10, 0, 5), (3, 1, 1)):
        check_evicted(cache, table, counts, totals.cuda(), keep, recent, sinks, there)


def test_a_long_sequence(Cache):
    lengths = [20000, 3]
    cache, table, counts, _, _ = filled(Cache, lengths, 2, 32, torch.bfloat16, 128)
    totals = (torch.rand(2, 2, table.shape[1] * 128, generator=torch.Generator().manual_seed(8)) * 300).round() / 64
    check_evicted(cache, table, counts, totals.cuda(), 7001, 500, 4)


def test_generation_goes_on_after_an_eviction(Cache):
    """As it would be used: prompts are written and weighed, tokens evicted, and steps attend to what is left."""
    lengths = [60, 33]
    cache, table, counts, keys, values = filled(Cache, lengths, 2, 64, torch.bfloat16, wide=1)
    q = vectors((93, 4, 64), torch.bfloat16, 9)
    starts = torch.tensor([0, 60, 93], dtype=torch.int32).cuda()
    totals = cache.weigh(cache.totals(table), q.cuda(), table, counts, starts)
    kept = [[R.evict(totals[b, h].tolist(), n, 24, 8, 2)[0] for h in range(2)] for b, n in enumerate(lengths)]
    counts.copy_(cache.evict(totals, table, counts, 24, recent=8, sinks=2))
    assert counts.tolist() == [24, 24]
    held_k = [torch.stack([C.held(keys[b][kept[b][h], h], 64) for h in range(2)], 1) for b in range(2)]
    held_v = [torch.stack([C.held(values[b][kept[b][h], h], 64) for h in range(2)], 1) for b in range(2)]
    for step in range(3):
        counts += 1
        k, v, x = (vectors((2, h, 64), torch.bfloat16, 30 + 3 * step + i) for i, h in enumerate((2, 2, 4)))
        cache.write(k.cuda(), v.cuda(), table, counts)
        got = cache.attend(x.cuda(), table, counts)
        for b in range(2):
            held_k[b], held_v[b] = torch.cat([held_k[b], C.held(k[b:b + 1], 64)]), torch.cat([held_v[b], C.held(v[b:b + 1], 64)])
            want, size, spread = C.attend(x[b:b + 1], [24 + step], held_k[b], held_v[b], 0.125)
            assert bool(((got[b:b + 1].double().cpu() - want).abs() <= C.bounds(torch.bfloat16, want, size, spread, 64)).all())


def test_captured_and_on_another_stream(Cache):
    lengths = [500, 70, 33]
    made = [filled(Cache, lengths, 2, 64, torch.bfloat16) for _ in range(2)]
    q = vectors((3, 8, 64), torch.bfloat16, 9).cuda()
    totals = [m[0].totals(m[1]) for m in made]
    graph, out = torch.cuda.CUDAGraph(), None
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        made[0][0].weigh(totals[0], q, made[0][1], made[0][2])
        out = made[0][0].evict(totals[0], made[0][1], made[0][2], 200, recent=20)
    stream = torch.cuda.Stream()
    for n in range(3):
        graph.replay()
        with torch.cuda.stream(stream):
            made[1][0].weigh(totals[1], q, made[1][1], made[1][2])
            want = made[1][0].evict(totals[1], made[1][1], made[1][2], 200, recent=20)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(totals[0], totals[1])
        assert torch.equal(made[0][0].codes, made[1][0].codes) and torch.equal(made[0][0].scales, made[1][0].scales)
        for m in made:
            m[2].copy_(want + 40)
        q.mul_(0.5)
        torch.cuda.synchronize()


def test_refusals(Cache):
    cache, table, counts, _, _ = filled(Cache, [20, 30], 2, 64, torch.bfloat16)
    totals, q = cache.totals(table), torch.ones(2, 4, 64, dtype=torch.bfloat16, device="cuda")
    for bad in (totals[:1], totals[:, :1], totals[..., :31], totals.double(), totals.cpu(), totals.transpose(1, 2), totals[0]):
        with pytest.raises((ValueError, RuntimeError)):
            cache.weigh(bad, q, table, counts)
        with pytest.raises((ValueError, RuntimeError)):
            cache.evict(bad, table, counts, 5)
    for bad in (q[:, :3], q[:1], q.half(), q[..., :32], q.cpu(), q.float().requires_grad_()):
        with pytest.raises((ValueError, RuntimeError)):
            cache.weigh(totals, bad, table, counts)
    for bad in (dict(window=0), dict(sinks=3), dict(window=5, sinks=-1), dict(scale=math.inf), dict(scale=math.nan)):
        with pytest.raises(ValueError):
            cache.weigh(totals, q, table, counts, **bad)
    for bad in (dict(keep=0), dict(keep=-1), dict(keep=5, recent=6), dict(keep=5, recent=3, sinks=3), dict(keep=5, recent=-1), dict(keep=5, sinks=-1)):
        with pytest.raises(ValueError):
            cache.evict(totals, table, counts, **bad)
    for bad in (table[:1], table.long(), table.cpu()):
        with pytest.raises((ValueError, RuntimeError)):
            cache.evict(totals, bad, counts, 5)
    assert not totals.any()
