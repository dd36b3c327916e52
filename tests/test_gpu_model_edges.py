"""Projections, rotary positions and eviction in calls at the edge of what is allowed: the most tokens, graphs that share memory, captured gradients, results in places that
are read."""
import math

import pytest
import torch

from oracle import evict_ref as E

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def library():
    import qtensor.functional as F
    assert torch.cuda.is_available() and F.lib is not None


def random(shape, seed, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def made(lengths, kv_heads, dim, seed=0, page_size=16):
    """(cache, table, lengths) of sequences that are in the cache already."""
    from qtensor.cache import QTensorCache
    width = -(-max(lengths) // page_size) + 1
    cache = QTensorCache(len(lengths) * width, kv_heads, dim, page_size=page_size)
    table = torch.randperm(len(lengths) * width, generator=torch.Generator().manual_seed(seed)).view(len(lengths), width).to(torch.int32).cuda()
    starts = torch.tensor([sum(lengths[:b]) for b in range(len(lengths) + 1)], dtype=torch.int32).cuda()
    counts = torch.tensor(lengths, dtype=torch.int32).cuda()
    cache.write(random((sum(lengths), kv_heads, dim), seed + 1), random((sum(lengths), kv_heads, dim), seed + 2), table, counts, starts)
    return cache, table, counts


def test_more_tokens_than_a_launch_takes():
    from qtensor.rotary import Rotary
    rotary, tokens = Rotary(2, frequencies=[0.37]), 2 ** 26 + 9
    positions = torch.arange(tokens, dtype=torch.int32, device="cuda")
    q = (positions.remainder(29) - 14).to(torch.bfloat16).view(tokens, 1, 1).repeat(1, 1, 2)
    got = rotary.turn(q, None, positions)[0]
    for some in (slice(0, 100), slice(2 ** 26 - 50, 2 ** 26), slice(2 ** 26 - 10, tokens)):
        assert torch.equal(got[some], rotary.turn(q[some], None, positions[some])[0])


def test_results_where_something_is_read():
    from qtensor.cache import QTensorCache
    from qtensor.linear import QTensorLinear
    from qtensor.rotary import Rotary
    weights = QTensorLinear(64, 64).quantize(random((64, 64), 1))
    both = torch.zeros(2, 64, device="cuda")
    for tokens in (1, 2):
        with pytest.raises(ValueError):
            weights.product(torch.ones(tokens, 64, device="cuda"), both[0], out=both[:tokens])
    cache, rotary = QTensorCache(4, 2, 64), Rotary(64)
    q, k = random((3, 4, 64), 2), random((3, 2, 64), 3)
    table, lengths = torch.tensor([[0], [1], [2]], dtype=torch.int32, device="cuda"), torch.ones(3, dtype=torch.int32, device="cuda")
    memory = torch.zeros(3 * 4 * 64, dtype=torch.bfloat16, device="cuda")
    for shape, strides in (((3, 4, 64), (0, 64, 1)), ((3, 4, 64), (64, 0, 1)), ((3, 4, 64), (64, 64, 1)), ((3, 4, 64), (32, 192, 1)), ((3, 4, 64), (128, 64, 1))):
        with pytest.raises(ValueError):
            cache.write_turned(rotary, q, k, k, table, lengths, out=memory.as_strided(shape, strides))
    want = cache.write_turned(rotary, q, k, k, table, lengths)
    for strides in ((64, 192, 1), (256, 64, 1)):
        out = memory.as_strided((3, 4, 64), strides)
        assert cache.write_turned(rotary, q, k, k, table, lengths, out=out) is out and torch.equal(out, want)
    one = memory.as_strided((1, 4, 64), (0, 64, 1))
    assert torch.equal(cache.write_turned(rotary, q[:1], k[:1], k[:1], table[:1], lengths[:1], out=one), want[:1])
    totals = torch.zeros(3, 2, 64, device="cuda")
    with pytest.raises(ValueError):
        cache.weigh(totals, totals.view(3, 2, 64), table, lengths)
    assert not totals.any()


@pytest.mark.parametrize("tokens", [1, 300])
def test_graphs_that_share_their_memory(tokens):
    """Scratch of a captured call is the graph's: two graphs of one pool, replayed in turn, with eager calls between them."""
    from qtensor.linear import QTensorLinear
    lengths, heads = [700, 90], 8
    cache, table, counts = made(lengths, 2, 64)
    weights = QTensorLinear(512, 320).quantize(random((320, 512), 5))
    q, x = random((2 * tokens if tokens > 1 else 2, heads, 64), 6), random((tokens, 512), 7)
    starts = torch.tensor([0, tokens, tokens + min(tokens, 90)], dtype=torch.int32, device="cuda") if tokens > 1 else None
    totals = [cache.totals(table) for _ in range(3)]
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], [None, None]
    want = cache.weigh(torch.zeros_like(totals[0]), q, table, counts, starts)
    product = weights.product(x)
    torch.cuda.synchronize()
    pool = torch.cuda.graph_pool_handle()
    for n, graph in enumerate(graphs):
        with torch.cuda.graph(graph, pool=pool):
            cache.weigh(totals[n], q, table, counts, starts)
            outs[n] = weights.product(x)
    for turn in range(3):
        for n in (0, 1):
            totals[n].zero_()
            graphs[n].replay()
            cache.weigh(totals[2].zero_(), q, table, counts, starts)
            assert torch.equal(totals[n], want) and torch.equal(totals[2], want) and torch.equal(outs[n], product)
        torch.cuda.synchronize()


def test_gradients_in_a_graph():
    from qtensor.rotary import Rotary
    rotary = Rotary(64)
    q, k = random((2, 50, 4, 64), 8).requires_grad_(), random((2, 50, 2, 64), 9).requires_grad_()
    at = torch.arange(50, device="cuda")

    def gradients():
        a, b = rotary.turn(q, k, at)
        return torch.autograd.grad((a.float() * a.float()).sum(-1).cos().sum() + (b.float() ** 3).sum(), (q, k))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        gradients()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = gradients()
    for n in range(3):
        with torch.no_grad():
            q.mul_(0.5), at.add_(100)
        graph.replay()
        want = gradients()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        torch.cuda.synchronize()


def test_many_prompts_weighed_in_parts():
    """Few rows over long sequences are cut into parts: what is added is the same however wide the table is, and in whichever sequence of the call."""
    lengths = [4000, 33, 2500]
    cache, table, counts = made(lengths, 2, 128, seed=20)
    news = [48, 20, 7]
    q = random((sum(news), 8, 128), 24)
    starts = torch.tensor([0, 48, 68, 75], dtype=torch.int32, device="cuda")
    all_of_them = cache.weigh(cache.totals(table), q, table, counts, starts)
    for b in range(3):
        alone = cache.weigh(cache.totals(table[b:b + 1]), q[starts[b]:starts[b + 1]], table[b:b + 1], counts[b:b + 1], torch.tensor([0, news[b]], dtype=torch.int32, device="cuda"))
        # of a weight: a lane adds fewer than 100 terms, each off by the exponent's rounding (|s - m| below 32, by 2^-20) and the exponential's own, and the parts' sums are
        # joined in another order: below 128 2^-24 + 2^-19 < 2^-16, of 4 news weights of at most 1; the total adds as many in fp32
        assert float((alone[0] - all_of_them[b]).abs().max()) <= 2.0 ** -16 * news[b] * 4
    total = all_of_them.double().sum(-1).cpu()
    for b in range(3):
        assert float((total[b] - news[b] * 4).abs().max()) <= 2.0 ** -15 * news[b] * 4


@pytest.mark.parametrize("batch,heads,kv_heads,dim,window,sinks,single", [(150, 4, 2, 64, None, 0, False), (150, 8, 2, 128, 40, 5, False), (200, 20, 1, 64, None, 0, True),
                                                                          (130, 4, 4, 96, None, 0, True), (65, 3, 1, 256, 30, 0, False)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_batches_of_more_sequences_than_a_wave_has_lanes(batch, heads, kv_heads, dim, window, sinks, single, dtype):
    """Work is found by lanes that have a sequence each, sixty-four at a time: batches of several times that, with empty ones among them."""
    lengths = [(37 * b) % 130 + (b % 7 == 0) * 300 if b % 11 else 0 for b in range(batch)]
    news = [1] * batch if single else [min(n, (5 * b) % 23) for b, n in enumerate(lengths)]
    cache, table, counts = made(lengths, kv_heads, dim, seed=30)
    q = random((sum(news), heads, dim), 33, dtype)
    starts = None if single else torch.tensor([sum(news[:b]) for b in range(batch + 1)], dtype=torch.int32, device="cuda")
    totals = cache.weigh(cache.totals(table), q, table, counts, starts, window=window, sinks=sinks)
    keys, _ = cache.read(table, counts, torch.tensor([sum(lengths[:b]) for b in range(batch + 1)], dtype=torch.int32, device="cuda"), tokens=sum(lengths))
    at = first = 0
    for b, (n, new) in enumerate(zip(lengths, news)):
        if n:
            want, spread = E.weigh(q[at:at + new].cpu(), range(n - new, n), keys[first:first + n].double().cpu(), 1 / math.sqrt(dim), window, sinks)
            off = (totals[b, :, :n].double().cpu() - want).abs()
            limit = E.bound(dim, new * heads // kv_heads, want, spread) + 2.0 ** -23 * want
            assert bool((off <= limit).all()), f"sequence {b}: off by {float((off / limit).max()):.3g} of the bound"
        assert not totals[b, :, n:].any()
        at, first = at + new, first + n


def test_more_tiles_of_rows_than_a_dimension_of_a_grid():
    """A prompt whose rows are more than 2^15 tiles, with a window: weights of a query add up to 1, and the last tokens' are those of a call with the last queries."""
    from qtensor.cache import QTensorCache
    tokens, heads, window = 270000, 4, 32
    cache = QTensorCache(-(-tokens // 4096), 1, 64, page_size=4096)
    table = torch.arange(cache.pages, dtype=torch.int32, device="cuda").view(1, -1)
    counts = torch.tensor([tokens], dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(40)
    q, k = (torch.randn(tokens, n, 64, generator=g, device="cuda").bfloat16() for n in (heads, 1))
    starts = torch.tensor([0, tokens], dtype=torch.int32, device="cuda")
    cache.write(k, k, table, counts, starts)
    totals = cache.weigh(cache.totals(table), q, table, counts, starts, window=window)
    last = cache.weigh(cache.totals(table), q[-1000:], table, counts, torch.tensor([0, 1000], dtype=torch.int32, device="cuda"), window=window)
    # (as above: a weight is good to 2^-16, and a token has 32 x 4 of them; all of them in 64 bits)
    some = slice(tokens - 900, tokens)
    assert float((totals[0, 0, some] - last[0, 0, some]).abs().max()) <= 2.0 ** -16 * window * heads
    per = totals[0, 0, :tokens].double()
    assert abs(float(per.sum()) - tokens * heads) <= 2.0 ** -16 * tokens * heads
    # any stretch of tokens has what its queries give it, less or more what a window reaches over both ends
    for first in (0, 100000, 200000):
        assert abs(float(per[first:first + 5000].sum()) - 5000 * heads) <= window * heads * 2


@pytest.mark.parametrize("lengths,news,heads,kv_heads,dim,window,sinks", [([700, 33, 0, 1100], [700, 33, 0, 1100], 8, 2, 64, None, 0), ([1300], [1300], 8, 1, 128, 200, 7),
                                                                          ([900, 500], [640, 500], 4, 2, 256, None, 0), ([2000, 1, 64], [700, 1, 64], 16, 1, 80, 64, 0)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_of_prompts_cut_into_parts(lengths, news, heads, kv_heads, dim, window, sinks, dtype):
    """Few tokens that many rows see: the rows are cut too, and their sums added in order; a page that is not there, totals that were not zero."""
    cache, table, counts = made(lengths, kv_heads, dim, seed=50)
    keys, _ = cache.read(table, counts, torch.tensor([sum(lengths[:b]) for b in range(len(lengths) + 1)], dtype=torch.int32, device="cuda"), tokens=sum(lengths))
    table[0, 2] = -1
    q = random((sum(news), heads, dim), 53, dtype)
    starts = torch.tensor([sum(news[:b]) for b in range(len(news) + 1)], dtype=torch.int32, device="cuda")
    before = torch.rand(cache.totals(table).shape, generator=torch.Generator().manual_seed(54)).cuda()
    totals = cache.weigh(before.clone(), q, table, counts, starts, window=window, sinks=sinks)
    assert torch.equal(cache.weigh(before.clone(), q, table, counts, starts, window=window, sinks=sinks), totals)
    at = first = 0
    for b, (n, new) in enumerate(zip(lengths, news)):
        there = torch.ones(n, dtype=torch.bool)
        if b == 0:
            there[32:48] = False
        want, spread = E.weigh(q[at:at + new].cpu(), range(n - new, n), keys[first:first + n].double().cpu(), 1 / math.sqrt(dim), window, sinks, there)
        start = before[b, :, :n].double().cpu()
        off = (totals[b, :, :n].double().cpu() - start - want).abs()
        limit = E.bound(dim, new * heads // kv_heads, want, spread) + 2.0 ** -23 * (start + want)
        assert bool((off <= limit).all()), f"sequence {b}: off by {float((off / limit).max()):.3g} of the bound"
        assert torch.equal(totals[b, :, n:], before[b, :, n:])
        at, first = at + new, first + n


@pytest.mark.parametrize("lengths,kv_heads,dim,blocksize,keep", [([9000, 40, 2500], 2, 128, 64, 2000), ([20000], 1, 80, 128, 9000), ([5000], 4, 256, 64, 1536), ([1700, 0], 1, 33, 256, 4000)])
def test_few_sequences_cut_down_through_room_of_their_own(lengths, kv_heads, dim, blocksize, keep):
    from qtensor.cache import QTensorCache
    width = -(-max(lengths) // 64) + 1
    cache = QTensorCache(len(lengths) * width + 2, kv_heads, dim, page_size=64, blocksize=blocksize)
    table = torch.randperm(cache.pages, generator=torch.Generator().manual_seed(60))[:len(lengths) * width].view(len(lengths), width).to(torch.int32).cuda()
    starts = torch.tensor([sum(lengths[:b]) for b in range(len(lengths) + 1)], dtype=torch.int32, device="cuda")
    counts = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    k, v = random((sum(lengths), kv_heads, dim), 61), random((sum(lengths), kv_heads, dim), 62)
    cache.write(k, v, table, counts, starts)
    table[0, 3] = -1
    before = cache.read(table, counts, starts, tokens=sum(lengths))
    totals = torch.rand(cache.totals(table).shape, generator=torch.Generator().manual_seed(63)).cuda()
    was = totals.clone()
    new = cache.evict(totals, table, counts, keep, recent=30, sinks=5)
    after = cache.read(table, counts, starts, tokens=sum(lengths))
    for b, n in enumerate(lengths):
        there = [not (b == 0 and 192 <= t < 256) for t in range(n)]
        at = int(starts[b])
        for h in range(kv_heads):
            source, target = E.evict(was[b, h, :n].tolist(), n, keep, 30, 5, there)
            assert int(new[b]) == (target[-1] + 1 if target else 0)
            i, j = torch.tensor(source, dtype=torch.long, device="cuda"), torch.tensor(target, dtype=torch.long, device="cuda")
            for x, y in zip(before, after):
                assert torch.equal(y[at + j, h], x[at + i, h])
            assert torch.equal(totals[b, h, j], was[b, h, i])
            stay = torch.ones(totals.shape[2], dtype=torch.bool, device="cuda")
            stay[j] = False
            assert torch.equal(totals[b, h][stay], was[b, h][stay])
