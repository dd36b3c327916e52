"""The attention cache held in 4 bits (qtensor.cache) against its definition in 64 bits (oracle/cache_ref.py).

Written and read values have to be equal bit for bit: the format's roundings are all defined.  Attention is held to the error
bounds of oracle.cache_ref.bounds, which follow from the operands' and the weights' roundings."""
import math

import pytest
import torch

from oracle import cache_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def Cache():
    from qtensor.cache import QTensorCache
    import qtensor.functional as F
    assert torch.cuda.is_available() and F.lib is not None
    return QTensorCache


def made(cache_type, lengths, news, kv_heads=2, dim=64, page_size=16, blocksize=64, spare=3, seed=0):
    """A cache with the pages of all sequences in random order, and the three arrays of a call."""
    g = torch.Generator().manual_seed(seed)
    width = max(1, max(-(-n // page_size) for n in lengths))
    pages = len(lengths) * width + spare
    table = torch.randperm(pages, generator=g)[: len(lengths) * width].view(len(lengths), width).to(torch.int32).cuda()
    starts = None if news is None else torch.tensor([sum(news[:b]) for b in range(len(news) + 1)], dtype=torch.int32).cuda()
    return (cache_type(pages, kv_heads, dim, page_size=page_size, blocksize=blocksize), table,
            torch.tensor(lengths, dtype=torch.int32).cuda(), starts)


def tokens(count, kv_heads, dim, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(count, kv_heads, dim, generator=g)
    x[..., ::13] *= 7.0
    x[::5] *= 0.01
    return x.to(dtype)


def fill(cache, table, lengths, dtype, seed, step=None):
    """Writes whole sequences; returns their keys and values per sequence (CPU, as written)."""
    counts = lengths.tolist()
    kept = [(tokens(n, cache.kv_heads, cache.head_dim, dtype, seed + 2 * b), tokens(n, cache.kv_heads, cache.head_dim, dtype, seed + 2 * b + 1))
            for b, n in enumerate(counts)]
    starts = torch.tensor([sum(counts[:b]) for b in range(len(counts) + 1)], dtype=torch.int32).cuda()
    cache.write(torch.cat([k for k, _ in kept]).cuda(), torch.cat([v for _, v in kept]).cuda(), table, lengths, starts)
    return kept


def equal(a, b):
    return torch.equal(torch.nan_to_num(a, nan=12345.0), torch.nan_to_num(b, nan=12345.0))


# ------------------------------------------------------------------------------------------------ writing and reading
@pytest.mark.parametrize("dim,blocksize,page_size", [(64, 64, 16), (128, 64, 64), (128, 128, 32), (80, 64, 16), (33, 256, 16), (1, 64, 16),
                                                     (192, 64, 128), (256, 64, 16), (256, 256, 64), (200, 128, 16), (96, 64, 4096)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_what_is_written_reads_as_its_definition(Cache, dim, blocksize, page_size, dtype):
    lengths = [37, 0, 1, 16, 17, 250]
    cache, table, lens, _ = made(Cache, lengths, None, 3, dim, page_size, blocksize)
    kept = fill(cache, table, lens, dtype, 11)
    starts = torch.tensor([sum(lengths[:b]) for b in range(7)], dtype=torch.int32).cuda()
    for out in (torch.float32, torch.bfloat16):
        keys, values = cache.read(table, lens, starts, tokens=sum(lengths), dtype=out)
        assert equal(keys.cpu(), R.held(torch.cat([k for k, _ in kept]), blocksize).float().to(out))
        assert equal(values.cpu(), R.held(torch.cat([v for _, v in kept]), blocksize).float().to(out))


def test_ties_and_ends_of_the_number_format(Cache):
    cache, table, lens, starts = made(Cache, [16], [16], 1, 64)
    x = torch.zeros(16, 1, 64)
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0])
    for t in range(16):
        near = ties if t % 3 == 0 else torch.nextafter(ties, torch.full_like(ties, math.inf if t % 3 == 1 else -math.inf))
        x[t, 0, :8], x[t, 0, 8:16] = near, -near
        x[t, 0, 16] = 6.0
        x[t] *= 2.0 ** (7 * t - 50)                      # powers of two: quotients stay what they are
    cache.write(x.cuda(), x.cuda(), table, lens, starts)
    keys, _ = cache.read(table, lens, starts, tokens=16)
    assert equal(keys.cpu(), R.held(x, 64).float())
    want = torch.tensor([0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 6.0]) * 2.0 ** -50
    assert torch.equal(keys[0, 0, :8].cpu(), want)


def test_zero_tiny_infinite_and_nan_segments(Cache):
    cache, table, lens, starts = made(Cache, [6], [6], 1, 128)
    x = torch.randn(6, 1, 128, generator=torch.Generator().manual_seed(3))
    x[0] = 0.0
    x[1, 0, :64] *= 1e-44
    x[2, 0, 64:] *= 3e38 / 4
    x[3, 0, 5] = math.inf
    x[4, 0, 70] = math.nan
    x[5, 0, ::2] = -0.0
    x = x.clamp(-3.4e38, 3.4e38).where(torch.isfinite(x), x)
    cache.write(x.cuda(), x.cuda(), table, lens, starts)
    keys, _ = cache.read(table, lens, starts, tokens=6)
    keys, want = keys.cpu(), R.held(x, 64).float()
    assert torch.isnan(keys[3, 0, :64]).all() and torch.isnan(keys[4, 0, 64:]).all()
    for t, part in ((0, slice(0, 128)), (1, slice(0, 128)), (2, slice(0, 128)), (3, slice(64, 128)), (4, slice(0, 64)), (5, slice(0, 128))):
        assert torch.equal(keys[t, 0, part], want[t, 0, part])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_new_tokens_land_behind_the_old_ones_and_nothing_else_moves(Cache, dtype):
    lengths, news = [40, 5, 17, 0, 33], [7, 5, 0, 0, 1]
    cache, table, lens, starts = made(Cache, lengths, news, 2, 80, 16, 64, seed=4)
    kept = fill(cache, table, lens, dtype, 21)
    before = (cache.codes.clone(), cache.scales.clone())
    k, v = tokens(13, 2, 80, dtype, 1), tokens(13, 2, 80, dtype, 2)
    cache.write(k.cuda(), v.cuda(), table, lens, starts)
    at = 0
    expect = []
    for (old_k, old_v), new, n in zip(kept, news, lengths):
        expect.append((torch.cat([old_k[: n - new], k[at:at + new]]), torch.cat([old_v[: n - new], v[at:at + new]])))
        at += new
    whole = torch.tensor([sum(lengths[:b]) for b in range(6)], dtype=torch.int32).cuda()
    keys, values = cache.read(table, lens, whole, tokens=sum(lengths))
    assert equal(keys.cpu(), R.held(torch.cat([a for a, _ in expect]), 64).float())
    assert equal(values.cpu(), R.held(torch.cat([b for _, b in expect]), 64).float())
    untouched = torch.ones(cache.pages, dtype=torch.bool)
    untouched[table.cpu().flatten().long()] = False
    assert torch.equal(cache.codes[:, untouched.cuda()], before[0][:, untouched.cuda()])
    # one token of each sequence, without starts
    one_k, one_v = tokens(5, 2, 80, dtype, 5), tokens(5, 2, 80, dtype, 6)
    cache.write(one_k.cuda(), one_v.cuda(), table, lens)
    keys, values = cache.read(table, lens)
    have = torch.tensor([n > 0 for n in lengths])
    assert equal(keys.cpu()[have], R.held(one_k, 64).float()[have]) and equal(values.cpu()[have], R.held(one_v, 64).float()[have])
    assert not keys[3].any() and not values[3].any()


def test_strided_and_unaligned_vectors(Cache):
    """Keys and values as parts of one projection's result, at addresses of one element."""
    cache, table, lens, starts = made(Cache, [30], [30], 3, 72, 16, 64)
    for dtype in (torch.bfloat16, torch.float32):
        whole = tokens(30, 9, 72, dtype, 8).reshape(30, -1).cuda()
        flat = torch.cat([whole.new_zeros(30, 1), whole], 1)                  # rows of an odd length, one element in
        k, v = (flat[:, 1 + 216 * i: 1 + 216 * (i + 1)].unflatten(1, (3, 72)) for i in (1, 2))
        assert k.data_ptr() % 16 and not k.is_contiguous()
        cache.write(k, v, table, lens, starts)
        keys, values = cache.read(table, lens, starts, tokens=30)
        assert equal(keys.cpu(), R.held(k.cpu(), 64).float()) and equal(values.cpu(), R.held(v.cpu(), 64).float())


# ------------------------------------------------------------------------------------------------ attention
def check(cache, table, lengths, news, dtype, group, seed, window=None, sinks=0, scale=None, there=None, kept=None):
    kept = fill(cache, table, lengths, dtype, seed) if kept is None else kept
    counts = lengths.tolist()
    rows = len(counts) if news is None else sum(news)
    starts = None if news is None else torch.tensor([sum(news[:b]) for b in range(len(news) + 1)], dtype=torch.int32).cuda()
    q = tokens(rows, cache.kv_heads * group, cache.head_dim, dtype, seed + 1000)
    out = cache.attend(q.cuda(), table, lengths, starts, scale=scale, window=window, sinks=sinks).cpu()
    assert out.shape == q.shape and out.dtype == dtype
    factor = 1.0 / math.sqrt(cache.head_dim) if scale is None else scale
    at = 0
    for b, n in enumerate(counts):
        new = 1 if news is None else news[b]
        keys, values = (R.held(x, cache.blocksize) for x in kept[b])
        result, size, spread = R.attend(q[at:at + new], range(n - new, n), keys, values, factor, window, sinks,
                                        None if there is None else there[b])
        off = (out[at:at + new].double() - result).abs()
        limit = R.bounds(dtype, result, size, spread, cache.head_dim)
        assert (off <= limit).all(), (b, n, new, float((off - limit).max()), float(off.max()), float(size.max()), float(spread.max()))
        at += new
    return q, out


@pytest.mark.parametrize("dim,blocksize,group", [(64, 64, 1), (64, 128, 5), (128, 64, 4), (128, 128, 8), (80, 64, 3), (96, 256, 2), (33, 64, 1),
                                                 (1, 64, 2), (192, 64, 6), (256, 64, 7), (256, 128, 4), (256, 256, 16), (112, 64, 17), (64, 64, 40)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_one_token_of_each_sequence(Cache, dim, blocksize, group, dtype):
    lengths = [1, 0, 2, 15, 16, 17, 129, 300, 64]
    cache, table, lens, _ = made(Cache, lengths, None, 2, dim, 16, blocksize, seed=dim)
    check(cache, table, lens, None, dtype, group, 31)


@pytest.mark.parametrize("length", [127, 128, 129, 511, 512, 513, 1025, 3000])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_longer_sequences_in_few_heads(Cache, length, dtype):
    cache, table, lens, _ = made(Cache, [length, 40], None, 1, 128, 64, 64, seed=length)
    check(cache, table, lens, None, dtype, 4, 41)


@pytest.mark.parametrize("dim,blocksize", [(64, 64), (128, 64), (128, 128), (80, 64), (256, 64), (192, 256)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_new_tokens_of_every_number(Cache, dim, blocksize, dtype):
    lengths, news = [150, 9, 33, 0, 70, 64, 200], [150, 1, 0, 0, 19, 2, 37]
    cache, table, lens, _ = made(Cache, lengths, None, 2, dim, 32, blocksize, seed=dim + 1)
    check(cache, table, lens, news, dtype, 3, 51)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (64, 0), (100, 130), (127, 5), (1000, 16), (5000, 4)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_windows_and_sinks(Cache, window, sinks, dtype):
    lengths = [1, 0, 17, 128, 700, 1300]
    cache, table, lens, _ = made(Cache, lengths, None, 2, 64, 16, 64, seed=window)
    check(cache, table, lens, None, dtype, 4, 61, window, sinks)
    check(cache, table, lens, [1, 0, 17, 5, 90, 40], dtype, 4, 61, window, sinks)


def test_scale_is_the_callers(Cache):
    cache, table, lens, _ = made(Cache, [90, 5], None, 2, 64)
    for scale in (0.0, -0.3, 0.9):
        check(cache, table, lens, None, torch.float32, 2, 71, scale=scale)


def test_weights_that_are_all_in_one_token_and_all_alike(Cache):
    """Scores hundreds apart, and long runs of equal ones with a large value at the end."""
    cache, table, lens, _ = made(Cache, [2000], None, 1, 64, 64)
    for sharp in (60.0, 0.0):
        for dtype in (torch.bfloat16, torch.float32):
            k, v = tokens(2000, 1, 64, dtype, 3), tokens(2000, 1, 64, dtype, 4)
            v[-3] *= 1000.0
            starts = torch.tensor([0, 2000], dtype=torch.int32).cuda()
            cache.write(k.cuda(), v.cuda(), table, lens, starts)
            check(cache, table, lens, None, dtype, 2, 81, scale=sharp, kept=[(k, v)])


def test_tails_of_tiny_weights_are_not_lost(Cache):
    """One token ahead of a hundred thousand that weigh 2^-17 of it each and make half of the sum."""
    n = 1 << 17
    cache, table, lens, starts = made(Cache, [n], [n], 1, 64, 256)
    k, v = torch.zeros(n, 1, 64), torch.ones(n, 1, 64)
    k[5, 0, 0], v[5] = 6.0, -1.0
    cache.write(k.cuda(), v.cuda(), table, lens, starts)
    q = torch.zeros(1, 1, 64)
    q[0, 0, 0] = 17 * math.log(2) / 6.0
    for dtype, limit in ((torch.float32, 2.0 ** -15), (torch.bfloat16, 2.0 ** -6)):
        query = q.to(dtype)
        lead = math.exp(6.0 * float(query[0, 0, 0]))
        want = ((n - 1) - lead) / ((n - 1) + lead)
        out = cache.attend(query.cuda(), table, lens, scale=1.0)
        assert (out.cpu().float() - want).abs().max() <= limit


def test_nothing_that_is_not_seen_is_looked_at(Cache):
    """NaN and infinities after the last token, behind the window and in the pages of other sequences change no bit."""
    for dtype in (torch.bfloat16, torch.float32):
        lengths = [100, 75, 0]
        cache, table, lens, _ = made(Cache, [200, 200, 200], None, 2, 64, 16, 64)
        clean = fill(cache, table, lens, dtype, 91)
        short = torch.tensor(lengths, dtype=torch.int32).cuda()
        q = tokens(3, 4, 64, dtype, 92).cuda()
        news = torch.tensor([0, 30, 60, 60], dtype=torch.int32).cuda()
        many = tokens(60, 4, 64, dtype, 93).cuda()
        calls = [lambda: cache.attend(q, table, short), lambda: cache.attend(q, table, short, window=20, sinks=3),
                 lambda: cache.attend(many, table, short, news, window=20, sinks=3)]
        before = [c() for c in calls]
        for bad in (math.nan, math.inf):
            spoiled = [(k.clone(), v.clone()) for k, v in clean]
            for b, n in enumerate(lengths):
                for x in spoiled[b]:
                    x[n:] = bad
            where = torch.tensor([0, 200, 400, 600], dtype=torch.int32).cuda()
            cache.write(torch.cat([k for k, _ in spoiled]).cuda(), torch.cat([v for _, v in spoiled]).cuda(), table, lens, where)
            assert torch.equal(calls[0](), before[0])
            for b, n in enumerate(lengths):
                for x in spoiled[b]:
                    x[3:max(3, n - 30 - 20)] = bad
            cache.write(torch.cat([k for k, _ in spoiled]).cuda(), torch.cat([v for _, v in spoiled]).cuda(), table, lens, where)
            assert torch.equal(calls[1](), before[1]) and torch.equal(calls[2](), before[2])


def test_nan_in_a_token_that_is_seen_reaches_only_its_head(Cache):
    cache, table, lens, _ = made(Cache, [50, 50], None, 2, 64)
    kept = fill(cache, table, lens, torch.float32, 95)
    q = tokens(2, 4, 64, torch.float32, 96).cuda()
    before = cache.attend(q, table, lens)
    k = kept[0][0].clone()
    k[20, 1, 3] = math.nan
    starts = torch.tensor([0, 50, 50], dtype=torch.int32).cuda()
    cache.write(k.cuda(), kept[0][1].cuda(), table, lens, starts)
    after = cache.attend(q, table, lens)
    assert torch.isnan(after[0, 2:]).all()
    assert torch.equal(after[0, :2], before[0, :2]) and torch.equal(after[1], before[1])


@pytest.mark.parametrize("dim,blocksize", [(64, 64), (33, 64), (128, 64), (128, 128), (256, 64), (256, 256)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_infinite_keys_are_nan_to_every_query_that_sees_them(Cache, dim, blocksize, dtype):
    """A key's segment with an infinity stands for NaN, whatever the tokens beside it hold."""
    cache, table, lens, _ = made(Cache, [50], None, 1, dim, 16, blocksize)
    (k, v), = fill(cache, table, lens, dtype, 98)
    k[::7, 0, 0], starts = math.inf, torch.tensor([0, 50], dtype=torch.int32).cuda()
    cache.write(k.cuda(), v.cuda(), table, lens, starts)
    for new in (1, 8):
        for seed in range(5):
            q = tokens(new, 2, dim, dtype, 200 + seed).cuda()
            at = torch.tensor([0, new], dtype=torch.int32).cuda()
            assert torch.isnan(cache.attend(q, table, lens, at)).all()
            see = cache.attend(q[-1:], table, lens, window=1)
            assert torch.isnan(see).all() if 49 % 7 == 0 else torch.isfinite(see).all()
    lens -= 1
    assert torch.isfinite(cache.attend(q[-1:], table, lens, window=6)).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_pages_that_are_not_there(Cache, dtype):
    """Pages marked -1 or beyond the cache, and lengths beyond the table: not written, zeros, not seen."""
    lengths = [160, 90]
    cache, table, lens, _ = made(Cache, lengths, None, 2, 64, 16, 64)
    kept = fill(cache, table, lens, dtype, 97)
    holed = table.clone()
    holed[0, 2], holed[0, 9], holed[1, 0] = -1, cache.pages, 2 ** 31 - 1
    there = [torch.ones(160, dtype=torch.bool), torch.ones(90, dtype=torch.bool)]
    there[0][32:48], there[0][144:], there[1][:16] = False, False, False
    check(cache, holed, lens, None, dtype, 3, 97, there=there, kept=kept)
    check(cache, holed, lens, [40, 90], dtype, 3, 97, there=there, kept=kept)
    keys, _ = cache.read(holed, lens, torch.tensor([0, 160, 250], dtype=torch.int32).cuda(), tokens=250)
    gone = ~torch.cat(there)
    assert not keys[gone.cuda()].any() and keys[~gone.cuda()].any()
    before = cache.codes.clone()
    cache.write(*(tokens(2, 2, 64, dtype, 1).cuda() for _ in range(2)), torch.full_like(table, -1), lens)
    assert torch.equal(cache.codes, before)
    # two pages of the first sequence only: the rest of its tokens is nowhere
    there = [torch.arange(160) < 32, torch.arange(90) < 32]
    check(cache, table[:, :2], lens, None, dtype, 3, 97, there=there, kept=kept)
    huge = torch.tensor([2 ** 31 - 1, 90], dtype=torch.int32).cuda()
    assert torch.isfinite(cache.attend(tokens(2, 2, 64, dtype, 5).cuda(), table, huge).float()).all()


def test_queries_and_results_of_any_stride(Cache):
    cache, table, lens, _ = made(Cache, [70, 30, 110], None, 2, 72, 16, 64)
    for dtype in (torch.bfloat16, torch.float32):
        fill(cache, table, lens, dtype, 99)
        for starts in (None, torch.tensor([0, 20, 21, 60], dtype=torch.int32).cuda()):
            rows = 3 if starts is None else 60
            plain = tokens(rows, 6, 72, dtype, 100).cuda()
            wide = torch.zeros(rows, 11 * 72 + 1, dtype=dtype, device="cuda")
            view = wide[:, 73:73 + 6 * 72].unflatten(1, (6, 72))
            view.copy_(plain)
            out = torch.full((6, rows, 75), 3.0, dtype=dtype, device="cuda")
            got = cache.attend(view, table, lens, starts, out=out[:, :, 2:74].transpose(0, 1))
            assert torch.equal(got, cache.attend(plain, table, lens, starts))
            assert (out[:, :, :2] == 3).all() and (out[:, :, 74:] == 3).all()


def test_a_cache_beyond_four_gigabytes(Cache):
    """Offsets into codes and scales that 32 bits do not hold."""
    pages = 40000                                            # 40000 pages x 8 heads x 256 tokens x 64 bytes: 5.2 GB of keys
    cache = Cache(pages, 8, 128, page_size=256, blocksize=64)
    assert cache.codes[0].numel() > 2 ** 32
    table = torch.tensor([[39999, 3], [0, 33000]], dtype=torch.int32).cuda()
    lens = torch.tensor([300, 512], dtype=torch.int32).cuda()
    check(cache, table, lens, None, torch.bfloat16, 2, 101)
    check(cache, table, lens, [20, 3], torch.float32, 2, 103)
    del cache
    torch.cuda.empty_cache()


def test_another_stream_and_replayed_graphs(Cache):
    """Calls follow the current stream; a captured step of generation takes other lengths, pages and tokens at every replay."""
    lengths = [40, 3, 250]
    cache, table, lens, _ = made(Cache, [260, 260, 260], None, 2, 128, 16, 64)
    fill(cache, table, lens, torch.bfloat16, 105)
    k, v, q = (tokens(3, h, 128, torch.bfloat16, 106 + h).cuda() for h in (2, 2, 8))
    now = torch.tensor(lengths, dtype=torch.int32).cuda()
    out = torch.empty_like(q)

    def step():
        cache.write(k, v, table, now)
        cache.attend(q, table, now, window=200, sinks=2, out=out)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    first = out.clone()
    step()
    assert torch.equal(out, first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for turn in range(4):
        now.copy_(torch.tensor([41 + turn, 4 + 30 * turn, 251 + turn], dtype=torch.int32))
        q.copy_(tokens(3, 8, 128, torch.bfloat16, 200 + turn))
        k.copy_(tokens(3, 2, 128, torch.bfloat16, 300 + turn))
        graph.replay()
        torch.cuda.synchronize()
        replayed = out.clone()
        out.zero_()
        step()
        assert torch.equal(out, replayed)


def test_the_same_bits_every_time(Cache):
    cache, table, lens, _ = made(Cache, [900, 2500, 3], None, 2, 128, 64, 64)
    fill(cache, table, lens, torch.bfloat16, 107)
    q = tokens(3, 8, 128, torch.bfloat16, 108).cuda()
    many, starts = tokens(300, 8, 128, torch.bfloat16, 109).cuda(), torch.tensor([0, 250, 298, 300], dtype=torch.int32).cuda()
    one, more = cache.attend(q, table, lens), cache.attend(many, table, lens, starts)
    for _ in range(5):
        assert torch.equal(cache.attend(q, table, lens), one) and torch.equal(cache.attend(many, table, lens, starts), more)


def test_state_dict_round_trip(Cache):
    cache, table, lens, _ = made(Cache, [50, 20], None, 2, 80)
    fill(cache, table, lens, torch.float32, 110)
    other = Cache(cache.pages, 2, 80, page_size=16, blocksize=64)
    other.load_state_dict(cache.state_dict())
    q = tokens(2, 4, 80, torch.float32, 111).cuda()
    assert torch.equal(other.attend(q, table, lens), cache.attend(q, table, lens))
    with pytest.raises(ValueError):
        Cache(cache.pages, 2, 80, page_size=32, blocksize=64).load_state_dict(cache.state_dict())
    with pytest.raises(ValueError):
        Cache(cache.pages + 1, 2, 80, page_size=16, blocksize=64).load_state_dict(cache.state_dict())


def test_no_tokens_at_all(Cache):
    cache, table, lens, _ = made(Cache, [50, 20], None, 2, 64)
    starts = torch.zeros(3, dtype=torch.int32).cuda()
    none = torch.empty(0, 2, 64, device="cuda")
    cache.write(none, none, table, lens, starts)
    assert cache.attend(none, table, lens, starts).shape == (0, 2, 64)
    assert cache.read(table, lens, starts, tokens=0)[0].shape == (0, 2, 64)


def test_refusals(Cache):
    cache, table, lens, starts = made(Cache, [50, 20], [3, 2], 2, 64)
    k = torch.zeros(5, 2, 64, device="cuda")
    q = torch.zeros(5, 4, 64, device="cuda")
    before = cache.codes.clone()
    good = (table, lens, starts)
    for bad in (lambda: cache.write(k.half(), k.half(), *good), lambda: cache.write(k, k.bfloat16(), *good), lambda: cache.write(k[:4], k, *good),
                lambda: cache.write(k, k[..., :32], *good), lambda: cache.write(k.transpose(0, 2), k, *good), lambda: cache.write(k.cpu(), k, *good),
                lambda: cache.write(k[..., ::2], k[..., ::2], *good), lambda: cache.write(k, k, table.long(), lens, starts),
                lambda: cache.write(k, k, table[:1], lens, starts), lambda: cache.write(k, k, table, lens.long(), starts),
                lambda: cache.write(k, k, table, lens, starts[:2]), lambda: cache.write(k, k, table, lens), lambda: cache.write(k[0], k[0], *good),
                lambda: cache.read(*good), lambda: cache.read(*good, tokens=5, dtype=torch.float16), lambda: cache.read(table, lens, tokens=5),
                lambda: cache.read(*good, tokens=-1),
                lambda: cache.attend(q.half(), *good), lambda: cache.attend(q[:, :3], *good), lambda: cache.attend(q, *good, window=0),
                lambda: cache.attend(q, *good, sinks=2), lambda: cache.attend(q, *good, window=4, sinks=-1),
                lambda: cache.attend(q, *good, scale=math.nan), lambda: cache.attend(q, *good, scale=math.inf),
                lambda: cache.attend(q, *good, out=q.bfloat16()), lambda: cache.attend(q, *good, out=torch.zeros(5, 2, 64, device="cuda")),
                lambda: cache.attend(q, table.cpu(), lens, starts)):
        with pytest.raises((ValueError, RuntimeError)):
            bad()
    with pytest.raises(RuntimeError):
        cache.write(k.clone().requires_grad_(), k, *good)
    with torch.no_grad():
        cache.attend(q.clone().requires_grad_(), *good)
    torch.cuda.synchronize()
    assert torch.equal(cache.codes, before)


def test_the_host_side_in_python_does_the_same(Cache, monkeypatch):
    """Calls that native code does not take (or all of them, without it) have the same bits."""
    import qtensor.cache as C
    assert C._native is not None
    cache, table, lens, _ = made(Cache, [70, 0, 300], None, 2, 96, 16, 64)
    starts = torch.tensor([0, 30, 30, 41], dtype=torch.int32).cuda()
    k, v, q = (tokens(41, h, 96, torch.bfloat16, 120 + h).cuda() for h in (2, 3, 6))
    v = v[:, :2]

    def everything():
        cache.codes.zero_(), cache.scales.zero_()
        cache.write(k, v, table, lens, starts)
        cache.write(k[:3], v[:3], table, lens)
        out = torch.zeros(41, 6, 96, dtype=torch.bfloat16, device="cuda")
        given = cache.attend(q, table, lens, starts, scale=0.3, window=50, sinks=3, out=out)
        assert given is out
        return [*cache.read(table, lens, starts, tokens=41, dtype=torch.bfloat16), *cache.read(table, lens), out, cache.attend(q[:3], table, lens),
                cache.attend(q, table, lens, starts, window=7)]

    native = everything()
    calls = []

    class Spy:
        def __getattr__(self, name):
            return lambda *a: calls.append((name, getattr(real, name)(*a))) or calls[-1][1]

    real = C._native
    monkeypatch.setattr(C, "_native", Spy())
    everything()
    assert len(calls) == 7 and all(done is not None for _, done in calls)
    monkeypatch.setattr(C, "_native", None)
    for a, b in zip(native, everything()):
        assert a.dtype == b.dtype and torch.equal(a, b)
