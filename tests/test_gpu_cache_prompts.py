"""Attention of many queries over the 4-bit cache where its fp16 operands have to follow what they are given: scales that grow,
zeros, values that are not finite; and the cuts, strides and head sizes of its own.  Against oracle/cache_ref.py in 64 bits.

A score is a sum of products of three fp16 roundings (query, scale and key: 2^-12 each), so it is off by at most 3 * 2^-12 of
`spread`; a weight by the factor exp of twice that.  Weights, scales and values round to 2^-12 each and what is dropped of small
weights is less, so 2^-8 of `size` holds them and the 2^-9 of the rounding of a result of that size."""
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


@pytest.fixture(params=["little", "much"], autouse=True)
def room(request):
    """How calls are taken depends on the tokens that the table has room for: with much of it, many queries go their own way."""
    prepared.room = 0 if request.param == "little" else 1 << 23


def widened(table, page_size):
    """Pages that are not there behind a sequence's, which change nothing."""
    more = max(0, prepared.room // page_size - table.shape[1])
    return torch.cat([table, torch.full((table.shape[0], more), -1, dtype=torch.int32, device=table.device)], 1)


def prepared(cache_type, keys, values, page_size=16, blocksize=64):
    """A cache of one sequence in pages of random order: (cache, table, lengths)."""
    n, kv_heads, dim = keys.shape
    width = -(-n // page_size)
    table = torch.randperm(width + 2, generator=torch.Generator().manual_seed(n))[:width].view(1, width).to(torch.int32).cuda()
    cache = cache_type(width + 2, kv_heads, dim, page_size=page_size, blocksize=blocksize)
    lengths, starts = torch.tensor([n], dtype=torch.int32).cuda(), torch.tensor([0, n], dtype=torch.int32).cuda()
    cache.write(keys.cuda(), values.cuda(), table, lengths, starts)
    return cache, widened(table, page_size), lengths


def normal(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def compare(out, q, new, keys, values, blocksize, scale=None, window=None, sinks=0, there=None):
    """Finite elements within the bound, the others NaN where the formula has NaN."""
    n = keys.shape[0]
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else scale
    k, v = R.held(keys, blocksize), R.held(values, blocksize)
    positions = range(n - new, n)
    want, _, _ = R.attend(q, positions, k, v, scale, window, sinks, there)
    _, size, spread = R.attend(q, positions, torch.nan_to_num(k), torch.nan_to_num(v), scale, window, sinks, there)
    out = out.cpu().double()
    assert torch.equal(torch.isnan(out), torch.isnan(want))
    off = torch.nan_to_num((out - want).abs())
    limit = size * (6 * 2.0 ** -12 * spread + 2.0 ** -8) + 2.0 ** -8 * torch.nan_to_num(want).abs()
    assert (off <= limit).all(), (float((off - limit).max()), float(off.max()), float(size.max()), float(spread.max()))


def attend(cache, table, lengths, q, **how):
    return cache.attend(q.cuda(), table, lengths, torch.tensor([0, q.shape[0]], dtype=torch.int32).cuda(), **how)


@pytest.mark.parametrize("dim,blocksize", [(64, 64), (128, 64), (128, 128), (256, 64), (256, 256)])
@pytest.mark.parametrize("which", ["keys", "values", "both"])
def test_scales_that_grow_from_tile_to_tile(Cache, dim, blocksize, which):
    """2^13 times larger from token 100 on, 2^11 times more from token 205 on; the last tokens are of ordinary size."""
    n, new = 300, 210
    size = torch.full((n, 1, 1), 2.0 ** -24)
    size[100:] = 2.0 ** -11
    size[205:] = 1.0
    k, v = normal(1, n, 2, dim), normal(2, n, 2, dim)
    k, v = (k * size if which != "values" else k).bfloat16(), (v * size if which != "keys" else v).bfloat16()
    q = normal(3, new, 4, dim).bfloat16()
    cache, table, lengths = prepared(Cache, k, v, 16, blocksize)
    compare(attend(cache, table, lengths, q), q, new, k, v, blocksize)
    # and in the other order: the largest come first
    k, v = k.flip(0), v.flip(0)
    cache, table, lengths = prepared(Cache, k, v, 16, blocksize)
    compare(attend(cache, table, lengths, q, window=80), q, new, k, v, blocksize, window=80)


@pytest.mark.parametrize("dim", [64, 128, 192])
def test_zeros_first_and_zeros_only(Cache, dim):
    n = 200
    k, v, q = normal(4, n, 1, dim).bfloat16(), normal(5, n, 1, dim).bfloat16(), normal(6, n, 3, dim).bfloat16()
    k[:90], v[:90] = 0.0, 0.0
    cache, table, lengths = prepared(Cache, k, v)
    compare(attend(cache, table, lengths, q), q, n, k, v, 64)
    cache, table, lengths = prepared(Cache, torch.zeros_like(k), torch.zeros_like(v))
    assert not attend(cache, table, lengths, q).any()
    compare(attend(cache, table, lengths, torch.zeros_like(q)), torch.zeros_like(q), n, torch.zeros_like(k), torch.zeros_like(v), 64)


@pytest.mark.parametrize("dim,blocksize", [(64, 64), (128, 64), (128, 128), (256, 64)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_values_and_keys_that_are_not_finite_reach_those_that_see_them(Cache, dim, blocksize, bad):
    n = 260
    k, v, q = normal(7, n, 2, dim).bfloat16(), normal(8, n, 2, dim).bfloat16(), normal(9, n, 4, dim).bfloat16()
    v[150, 1, dim - 3] = bad                # one segment of one head
    cache, table, lengths = prepared(Cache, k, v, 16, blocksize)
    out = attend(cache, table, lengths, q)
    compare(out, q, n, k, v, blocksize)
    assert torch.isnan(out[150:, 2:, dim - 3]).all() and torch.isfinite(out[:150]).all() and torch.isfinite(out[:, :2]).all()
    out = attend(cache, table, lengths, q, window=30, sinks=2)
    compare(out, q, n, k, v, blocksize, window=30, sinks=2)
    assert torch.isfinite(out[180:]).all()
    k[40, 0, 1] = bad
    cache, table, lengths = prepared(Cache, k, v, 16, blocksize)
    out = attend(cache, table, lengths, q, window=90)
    compare(out, q, n, k, v, blocksize, window=90)
    assert torch.isnan(out[40:130, :2]).all() and torch.isfinite(out[:40]).all() and torch.isfinite(out[130:, :2]).all()


@pytest.mark.parametrize("dim,blocksize,group", [(33, 64, 2), (1, 64, 3), (72, 64, 1), (100, 64, 5), (129, 128, 2), (255, 64, 1), (250, 256, 3)])
def test_heads_of_odd_sizes_and_queries_at_odd_places(Cache, dim, blocksize, group):
    n, new = 170, 150
    k, v, q = normal(10, n, 2, dim).bfloat16(), normal(11, n, 2, dim).bfloat16(), normal(12, new, 2 * group, dim).bfloat16()
    cache, table, lengths = prepared(Cache, k, v, 32, blocksize)
    straight = attend(cache, table, lengths, q)
    compare(straight, q, new, k, v, blocksize)
    wide = torch.zeros(new, 2 * group * dim + 3, dtype=torch.bfloat16)
    view = wide[:, 1:1 + 2 * group * dim].unflatten(1, (2 * group, dim))
    view.copy_(q)
    wide = wide.cuda()
    starts = torch.tensor([0, new], dtype=torch.int32).cuda()
    assert torch.equal(cache.attend(wide[:, 1:1 + 2 * group * dim].unflatten(1, (2 * group, dim)), table, lengths, starts), straight)


@pytest.mark.parametrize("dim,blocksize", [(64, 64), (128, 64), (256, 128)])
@pytest.mark.parametrize("new,group,window,sinks", [(40, 2, None, 0), (33, 1, None, 0), (100, 3, 1500, 70), (40, 2, 1, 0)])
def test_some_queries_at_the_end_of_long_sequences(Cache, dim, blocksize, new, group, window, sinks):
    """So few rows of tiles that each is cut into pieces."""
    n = 5000
    k, v, q = normal(13, n, 1, dim).bfloat16(), normal(14, n, 1, dim).bfloat16(), normal(15, new, group, dim).bfloat16()
    cache, table, lengths = prepared(Cache, k, v, 64, blocksize)
    compare(attend(cache, table, lengths, q, window=window, sinks=sinks), q, new, k, v, blocksize, window=window, sinks=sinks)


@pytest.mark.parametrize("bad", [False, True])
def test_pieces_of_different_sizes_are_joined(Cache, bad):
    """Scales that grow inside a later piece, and a value that is not finite in one of them."""
    n, new = 4000, 48
    k, v, q = normal(16, n, 1, 128), normal(17, n, 1, 128), normal(18, new, 2, 128).bfloat16()
    k[:2500] *= 2.0 ** -14
    v[:3100] *= 2.0 ** -12
    if bad:
        v[700, 0, 5] = math.inf
    k, v = k.bfloat16(), v.bfloat16()
    cache, table, lengths = prepared(Cache, k, v, 64, 64)
    compare(attend(cache, table, lengths, q), q, new, k, v, 64)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("window,sinks", [(None, 0), (50, 0), (50, 20), (1, 1)])
def test_pages_that_are_not_there_and_tokens_that_are_not_seen(Cache, dim, window, sinks):
    """Missing pages are not seen; NaN behind the window of every query and behind the last token change no bit."""
    n, new = 330, 90
    k, v, q = normal(27, n, 2, dim).bfloat16(), normal(28, n, 2, dim).bfloat16(), normal(29, new, 4, dim).bfloat16()
    cache, table, lengths = prepared(Cache, k, v, 16, 64)
    lengths -= 10
    clean = attend(cache, table, lengths, q, window=window, sinks=sinks)
    compare(clean, q, new, k[:-10], v[:-10], 64, window=window, sinks=sinks)
    bad = [t.clone() for t in (k, v)]
    for t in bad:
        t[-10:] = math.nan
        if window is not None:
            t[sinks:n - 10 - new - window + 1] = math.nan
    lengths += 10
    cache.write(*(t.cuda() for t in bad), table, lengths, torch.tensor([0, n], dtype=torch.int32).cuda())
    lengths -= 10
    assert torch.equal(attend(cache, table, lengths, q, window=window, sinks=sinks), clean)
    cache, table, lengths = prepared(Cache, k, v, 16, 64)
    table[0, 1], table[0, 17], table[0, 19] = -1, cache.pages, -7
    there = torch.ones(n, dtype=torch.bool)
    there[16:32], there[272:288], there[304:320] = False, False, False
    compare(attend(cache, table, lengths, q, window=window, sinks=sinks), q, new, k, v, 64, window=window, sinks=sinks, there=there)


@pytest.mark.parametrize("n", [1, 5, 700, 3000])
@pytest.mark.parametrize("group", [33, 64, 150])
def test_one_token_of_many_heads_that_share_one(Cache, n, group):
    k, v, q = normal(19, n, 2, 64).bfloat16(), normal(20, n, 2, 64).bfloat16(), normal(21, 1, 2 * group, 64).bfloat16()
    cache, table, lengths = prepared(Cache, k, v)
    compare(cache.attend(q.cuda(), table, lengths), q, 1, k, v, 64)


def test_sequences_of_few_and_many_new_tokens_in_one_call_and_more_than_a_wave_has_lanes(Cache):
    """150 sequences: each is found by a wave that looks at 64 at a time."""
    lens = [(37 * b) % 90 for b in range(150)]
    news = [min(n, (0, 1, 3, 60, 90)[b % 5]) for b, n in enumerate(lens)]
    total = sum(lens)
    k, v = normal(22, total, 1, 64).bfloat16(), normal(23, total, 1, 64).bfloat16()
    q = normal(24, sum(news), 2, 64).bfloat16()
    width = 6
    table = torch.randperm(150 * width, generator=torch.Generator().manual_seed(1)).view(150, width).to(torch.int32).cuda()
    cache = Cache(150 * width, 1, 64, page_size=16)
    lengths = torch.tensor(lens, dtype=torch.int32).cuda()
    table = widened(table, 16)
    at = [[sum(x[:b]) for b in range(151)] for x in (lens, news)]
    cache.write(k.cuda(), v.cuda(), table, lengths, torch.tensor(at[0], dtype=torch.int32).cuda())
    keys, values = cache.read(table, lengths, torch.tensor(at[0], dtype=torch.int32).cuda(), tokens=total)
    assert torch.equal(keys.cpu(), R.held(k, 64).float()) and torch.equal(values.cpu(), R.held(v, 64).float())
    out = cache.attend(q.cuda(), table, lengths, torch.tensor(at[1], dtype=torch.int32).cuda())
    for b in range(150):
        if news[b]:
            rows, kept = slice(at[1][b], at[1][b + 1]), slice(at[0][b], at[0][b + 1])
            compare(out[rows], q[rows], news[b], k[kept], v[kept], 64)


def test_a_workspace_too_small_is_refused(Cache):
    import ctypes as ct
    import qtensor.functional as F
    import qtensor.cache as C
    k, q = normal(25, 20, 1, 64).bfloat16(), normal(26, 1, 2, 64).bfloat16().cuda()
    cache, table, lengths = prepared(Cache, k, k)
    out = torch.full_like(q, 7.0)
    need = F.lib.qtensor_hip_cache_attend_workspace(cache._ref(), 2, 1, 0)
    assert need > 0
    room = torch.empty(need, dtype=torch.uint8, device="cuda")
    places = cache._places(table, lengths, None, 1)
    for have, at in ((need - 1, room.data_ptr()), (need, 0)):
        F.lib.qtensor_hip_cache_attend(cache._ref(), places, C._vectors(q), C._vectors(out), 2, 0.1, 0, 0, at, have, 0)
        assert F.lib.qtensor_hip_last_error() != 0
    torch.cuda.synchronize()
    assert (out == 7.0).all()
    F.lib.qtensor_hip_cache_attend(cache._ref(), places, C._vectors(q), C._vectors(out), 2, 0.1, 0, 0, room.data_ptr(), need, 0)
    assert F.lib.qtensor_hip_last_error() == 0
    torch.cuda.synchronize()
    assert not (out == 7.0).all()
