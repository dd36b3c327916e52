"""The 4-bit attention cache where calls end and where their numbers are far apart.  Against the definition in 64 bits.

The bound on the route of many queries, in units of `size` = sum_j p_j max |v_j| over the tokens that a query sees itself: keys are rounded
twice to 2^-12 (scale and product), so a score is off by 2 * 2^-12 of `sharp` = max_j scale sum_d |q_d k_jd|; elements of a query below fp16's
normal numbers by 2^-25 against keys of at most 768 there, dim * 768 * 2^-25 in exponents of 2; a weight by the factor exp of twice that.  Weights
and values round to 2^-11 each, the result to 2^-9: 2^-8 of `size` holds these."""
import math

import pytest
import torch

from oracle import cache_ref as R

pytestmark = pytest.mark.gpu

MUCH = 1 << 23                          # with so much room in the table, sequences of many queries go their own way


@pytest.fixture(scope="module")
def Cache():
    from qtensor.cache import QTensorCache
    import qtensor.functional as F
    assert torch.cuda.is_available() and F.lib is not None
    return QTensorCache


def normal(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def ints(*x):
    return torch.tensor(x, dtype=torch.int32).cuda()


def one_sequence(cache_type, k, v, blocksize=64, page_size=16, pages=None, room=0):
    """(cache, table, lengths): one sequence in pages of random order, of which the table has `pages`, and -1 up to `room` tokens."""
    n, kv_heads, dim = k.shape
    width = -(-n // page_size) if pages is None else pages
    table = torch.randperm(width + 2, generator=torch.Generator().manual_seed(n))[:width].view(1, width).to(torch.int32)
    table = torch.cat([table, torch.full((1, max(0, room // page_size - width)), -1, dtype=torch.int32)], 1).cuda()
    cache = cache_type(width + 2, kv_heads, dim, page_size=page_size, blocksize=blocksize)
    cache.write(k.cuda(), v.cuda(), table, ints(n), ints(0, n))
    return cache, table, ints(n)


def expected(q, first, k, v, blocksize, scale=None, window=None, sinks=0, there=None):
    """(result, size, sharp) of queries at `first` and on, all fp64."""
    new, heads, dim = q.shape
    count, kv_heads, _ = k.shape
    scale = dim ** -0.5 if scale is None else scale
    K, V = R.held(k, blocksize), R.held(v, blocksize)
    i, j = torch.arange(first, first + new)[:, None], torch.arange(count)[None, :]
    see = j <= i
    if window is not None:
        see = see & ((i - j < window) | (j < sinks))
    if there is not None:
        see = see & there[None, :]
    out, size, sharp = torch.zeros(new, heads, dim).double(), torch.zeros(new, heads, 1).double(), torch.zeros(new, heads, 1).double()
    any_seen = see.any(1)
    for h in range(heads):
        kh, vh, qh = K[:, h // (heads // kv_heads)], V[:, h // (heads // kv_heads)], q[:, h].double()
        # (what a query does not see is left out of its sums, so that what it holds does not matter)
        s = (scale * (qh @ torch.nan_to_num(kh).T)).masked_fill(~see, -math.inf)
        nan = (see & ~torch.isfinite(kh).all(1)[None, :]).any(1) | ~torch.isfinite(qh).all(1)
        p = torch.nan_to_num(torch.softmax(torch.nan_to_num(s, nan=0.0, neginf=-math.inf), 1))
        out[:, h] = p @ vh
        out[nan & any_seen, h] = math.nan
        size[:, h, 0] = p @ vh.abs().amax(1)
        sharp[:, h, 0] = (abs(scale) * (torch.nan_to_num(qh, 0.0, 0.0, 0.0).abs() @ torch.nan_to_num(kh).abs().T)).masked_fill(~see, 0.0).amax(1)
    out[~any_seen] = 0.0
    return out, size, sharp


def compare_many(out, q, first, k, v, blocksize, **how):
    want, size, sharp = expected(q, first, k, v, blocksize, **how)
    dim = q.shape[-1]
    out = out.cpu().double()
    assert torch.equal(torch.isnan(out), torch.isnan(want))
    off = torch.nan_to_num((out - want).abs())
    limit = size * (2 * (2 * 2.0 ** -12 * sharp + math.log(2) * dim * 768 * 2.0 ** -25) + 2.0 ** -8) + 2.0 ** -8 * torch.nan_to_num(want).abs()
    assert (off <= limit).all(), (int((off > limit).sum()), float((off / size.clamp(min=1e-300)).max()), float(sharp.max()))


# ------------------------------------------------------------------------------------------------ tables that end inside a tile
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page_size", [16, 32])
@pytest.mark.parametrize("cut", [False, True])
@pytest.mark.parametrize("window,sinks", [(None, 0), (200, 5)])
def test_tokens_behind_the_table_are_not_seen(Cache, dim, page_size, cut, window, sinks):
    """Queries on both sides of the last token that the table has a page for, which is inside a tile of 64."""
    kv_heads, covered = (2, 3600 if page_size == 16 else 3616) if cut else (8, 1008 if page_size == 16 else 992)
    assert covered % 64 and 1200 * kv_heads * covered > MUCH
    n, new, group = covered + 40, 300, 4
    k, v, q = normal(1, n, kv_heads, dim).bfloat16(), normal(2, n, kv_heads, dim).bfloat16(), normal(3, new, kv_heads * group, dim).bfloat16()
    cache, table, lengths = one_sequence(Cache, k, v, page_size=page_size, pages=covered // page_size)
    out = cache.attend(q.cuda(), table, lengths, ints(0, new), window=window, sinks=sinks)
    compare_many(out, q, n - new, k, v, 64, window=window, sinks=sinks, there=torch.arange(n) < covered)


# ------------------------------------------------------------------------------------------------ numbers that are far apart
@pytest.mark.parametrize("dim,blocksize", [(64, 64), (128, 64), (128, 128), (256, 64)])
@pytest.mark.parametrize("large", [8000.0, 1.0e6])
def test_large_queries_and_keys_in_different_channels(Cache, dim, blocksize, large):
    """Products of their largest elements are beyond fp16, the scores are not; the large keys are later than some of the queries."""
    n, new = 300, 260
    k, v, q = normal(4, n, 2, dim), normal(5, n, 2, dim).bfloat16(), normal(6, new, 4, dim)
    k[200:, :, 5], q[:, :, 5] = large, 0.0
    q[::3, :, dim - 2], k[:, :, dim - 2] = large, 0.0
    k, q = k.bfloat16(), q.bfloat16()
    cache, table, lengths = one_sequence(Cache, k, v, blocksize, room=MUCH)
    out = cache.attend(q.cuda(), table, lengths, ints(0, new))
    assert torch.isfinite(out).all()
    compare_many(out, q, n - new, k, v, blocksize)


@pytest.mark.parametrize("dim", [64, 128, 192])
@pytest.mark.parametrize("n,new", [(300, 260), (4000, 48)])
def test_queries_that_are_not_finite(Cache, dim, n, new):
    """An infinite element makes every product infinite or NaN, whatever its sign and that of the keys: the formula has NaN."""
    k, v, q = normal(7, n, 2, dim), normal(8, n, 2, dim).bfloat16(), normal(9, new, 4, dim).bfloat16()
    k[:, :, 7] = k[:, :, 7].abs() + 0.5
    k = k.bfloat16()
    q[3, 0, 7], q[20, 1, 7], q[21, 3, 1], q[30, 2, 7] = -math.inf, math.inf, math.nan, -math.inf
    cache, table, lengths = one_sequence(Cache, k, v, 64, 64, room=MUCH)
    out = cache.attend(q.cuda(), table, lengths, ints(0, new))
    assert torch.isnan(out[3, 0]).all() and torch.isnan(out[30, 2]).all() and int(torch.isnan(out).sum()) == 4 * dim
    compare_many(out, q, n - new, k, v, 64)


@pytest.mark.parametrize("dim,blocksize", [(64, 64), (128, 64), (128, 128), (256, 256), (1, 64), (33, 64), (100, 64), (200, 128), (224, 64), (255, 64)])
@pytest.mark.parametrize("exponent", [-10, -18, -30, -90])
def test_values_much_smaller_than_those_of_later_tokens(Cache, dim, blocksize, exponent):
    """The first queries see only the small ones: what comes later must not take their bits."""
    n = 330
    k, v, q = normal(10, n, 2, dim).bfloat16(), normal(11, n, 2, dim), normal(12, n, 4, dim).bfloat16()
    v[:100] *= 2.0 ** exponent
    v = v.bfloat16()
    cache, table, lengths = one_sequence(Cache, k, v, blocksize, room=MUCH)
    compare_many(cache.attend(q.cuda(), table, lengths, ints(0, n)), q, 0, k, v, blocksize)
    # and larger ones that the window has left behind, in the first tiles of the same workgroup
    k, v = k.flip(0), v.flip(0)
    cache, table, lengths = one_sequence(Cache, k, v, blocksize, room=MUCH)
    compare_many(cache.attend(q.cuda(), table, lengths, ints(0, n), window=20), q, 0, k, v, blocksize, window=20)


@pytest.mark.parametrize("dim,blocksize", [(64, 64), (128, 128)])
def test_values_far_apart_in_pieces(Cache, dim, blocksize):
    n, new = 4000, 48
    k, v, q = normal(13, n, 1, dim).bfloat16(), normal(14, n, 1, dim), normal(15, new, 2, dim).bfloat16()
    v[:3970] = v[:3970].abs() * 2.0 ** -40
    v = v.bfloat16()
    cache, table, lengths = one_sequence(Cache, k, v, blocksize, 64, room=MUCH)
    compare_many(cache.attend(q.cuda(), table, lengths, ints(0, new)), q, n - new, k, v, blocksize)


@pytest.mark.parametrize("dim,blocksize", [(64, 64), (128, 64), (256, 64)])
@pytest.mark.parametrize("grown,query", [(2.0 ** 8, 2.0 ** -6), (2.0 ** 30, 2.0 ** -18), (2.0 ** 20, 2.0 ** 12), (1.0, 2.0 ** -40), (1.0, 2.0 ** 14)])
def test_keys_that_grow_and_queries_of_any_size(Cache, dim, blocksize, grown, query):
    """Scores of a few: of large keys and small queries, or the reverse; the first tokens' keys are smaller yet."""
    n, new = 300, 230
    k, v, q = normal(16, n, 2, dim), normal(17, n, 2, dim).bfloat16(), (query * normal(18, new, 4, dim)).bfloat16()
    k[64:] *= grown
    k = (k * 4.0 / (query * grown)).bfloat16()
    cache, table, lengths = one_sequence(Cache, k, v, blocksize, room=MUCH)
    compare_many(cache.attend(q.cuda(), table, lengths, ints(0, new)), q, n - new, k, v, blocksize)


@pytest.mark.parametrize("dim,blocksize", [(64, 64), (128, 64), (128, 128), (256, 64)])
def test_queries_below_what_fp16_holds_with_keys_that_grow(Cache, dim, blocksize):
    """All elements alike, so that what they lose adds up: keys of 6 and then of +-6 * 2^9, queries that make 2^-25 more or less of one another."""
    n, new = 200, 130
    k, v = torch.full((n, 1, dim), 6.0), torch.ones(n, 1, dim)
    k[64:] *= 2.0 ** 9
    k[65::2] *= -1.0
    v[65::2] *= -1.0
    q = torch.full((new, 2, dim), 1.5 * 2.0 ** -21)
    q[1::2] *= 5.0 / 3.0
    k, v, q = k.bfloat16(), v.bfloat16(), q.bfloat16()
    cache, table, lengths = one_sequence(Cache, k, v, blocksize, room=MUCH)
    scale = math.log(2.0)
    compare_many(cache.attend(q.cuda(), table, lengths, ints(0, new), scale=scale), q, n - new, k, v, blocksize, scale=scale)


@pytest.mark.parametrize("dim,blocksize", [(64, 64), (128, 64), (128, 128), (256, 64)])
def test_keys_below_what_fp16_holds_with_large_queries(Cache, dim, blocksize):
    """All elements alike again: small keys that differ by less than a step of fp16 beside large ones, in a channel where queries are zero."""
    n, new = 260, 150
    k, v = torch.full((n, 1, dim), 6.0 * 2.0 ** -26), torch.ones(n, 1, dim)
    k[1::2] *= 1.125
    v[1::2] *= -1.0
    k[130:, :, 3] = 6.0
    q = torch.full((new, 2, dim), 2.0 ** 27 / (6.75 * dim))
    q[:, :, 3] = 0.0
    k, v, q = k.bfloat16(), v.bfloat16(), q.bfloat16()
    cache, table, lengths = one_sequence(Cache, k, v, blocksize, room=MUCH)
    scale = math.log(2.0)
    compare_many(cache.attend(q.cuda(), table, lengths, ints(0, new), scale=scale), q, n - new, k, v, blocksize, scale=scale)


@pytest.mark.parametrize("scale", [0.0, -0.3, 1.0e-30, 3.0])
def test_scales_of_scores_of_any_sign_and_size(Cache, scale):
    n, new = 300, 230
    k, v, q = normal(19, n, 2, 64).bfloat16(), normal(20, n, 2, 64).bfloat16(), normal(21, new, 4, 64).bfloat16()
    cache, table, lengths = one_sequence(Cache, k, v, room=MUCH)
    compare_many(cache.attend(q.cuda(), table, lengths, ints(0, new), scale=scale), q, n - new, k, v, 64, scale=scale)


# ------------------------------------------------------------------------------------------------ windows beyond every length
@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("window,sinks", [(2 ** 31 - 1, 0), (2 ** 31, 0), (2 ** 32, 7), (2 ** 32 + 5, 0), (10, 2 ** 31), (10, 2 ** 32 + 1)])
def test_windows_and_sinks_beyond_32_bits_are_all_tokens(Cache, monkeypatch, native, window, sinks):
    import qtensor.cache as C
    if not native:
        monkeypatch.setattr(C, "_native", None)
    k, v, q = normal(22, 200, 2, 64), normal(23, 200, 2, 64), normal(24, 9, 4, 64)
    cache, table, lengths = one_sequence(Cache, k, v)
    out = cache.attend(q.cuda(), table, lengths, ints(0, 9), window=window, sinks=sinks).cpu().double()
    want, size, spread = R.attend(q, range(191, 200), R.held(k, 64), R.held(v, 64), 0.125)
    assert ((out - want).abs() <= R.bounds(torch.float32, want, size, spread, 64)).all()


def test_more_tokens_than_the_library_counts_are_refused(Cache):
    k = normal(34, 20, 1, 64)
    cache, table, lengths = one_sequence(Cache, k, k)
    for tokens in (2 ** 31, 2 ** 32 + 20):
        with pytest.raises(ValueError):
            cache.read(table, lengths, ints(0, 20), tokens=tokens)


@pytest.mark.parametrize("room", [0, MUCH])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 200])
def test_the_largest_windows_of_a_sequence_shorter_than_its_part(Cache, room, dtype, window):
    """Its first rows have negative positions and see nothing; the others see all up to themselves."""
    n, new = 100, 300
    k, v, q = normal(25, n, 2, 64).to(dtype), normal(26, n, 2, 64).to(dtype), normal(27, new, 4, 64).to(dtype)
    cache, table, lengths = one_sequence(Cache, k, v, room=room)
    out = cache.attend(q.cuda(), table, lengths, ints(0, new), window=window)
    assert not out[:200].any()
    compare_many(out[200:], q[200:], 0, k, v, 64)


# ------------------------------------------------------------------------------------------------ rows of no sequence
@pytest.mark.parametrize("room", [0, MUCH])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim", [64, 80, 256])
@pytest.mark.parametrize("tokens", [41, 42, 48, 300])
def test_rows_behind_the_last_start_are_zeros(Cache, room, dtype, dim, tokens):
    """A step captured with room for more tokens than there are."""
    k, v = normal(28, 90, 2, dim).to(dtype), normal(29, 90, 2, dim).to(dtype)
    cache, table, _ = one_sequence(Cache, k, v, room=room)
    table, lengths, starts = table.repeat(3, 1), ints(90, 0, 50), ints(0, 40, 40, 41)
    q = normal(30, tokens, 6, dim).to(dtype).cuda()
    for stride in (1, 2):
        whole = torch.full((tokens, 6 * stride, dim), math.nan, dtype=dtype, device="cuda")
        out = cache.attend(q, table, lengths, starts, out=whole[:, ::stride])
        assert torch.equal(out[:41], cache.attend(q[:41].contiguous(), table, lengths, starts)) and not out[41:].any()
        assert stride == 1 or torch.isnan(whole[:, 1::2]).all()
    # no tokens at all, and starts that promise more than there are
    nothing = torch.full_like(q, math.nan)
    assert not cache.attend(q, table, lengths, ints(0, 0, 0, 0), out=nothing).any()
    out = cache.attend(q, table, lengths, ints(0, 40, 40, tokens + 1), out=torch.full_like(q, math.nan))
    assert torch.equal(out[:40], cache.attend(q[:40].contiguous(), table[:1], lengths[:1], ints(0, 40))) and not out[40:].any()


def test_a_captured_step_with_fewer_tokens_at_a_replay(Cache):
    k, v = normal(31, 90, 2, 64).bfloat16(), normal(32, 90, 2, 64).bfloat16()
    cache, table, _ = one_sequence(Cache, k, v)
    table, lengths, starts = table.repeat(2, 1), ints(90, 60), ints(0, 20, 24)
    q, out = normal(33, 24, 4, 64).bfloat16().cuda(), torch.empty(24, 4, 64, dtype=torch.bfloat16, device="cuda")
    cache.attend(q, table, lengths, starts, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.attend(q, table, lengths, starts, out=out)
    for counts in ((0, 20, 24), (0, 3, 5), (0, 0, 0), (0, 24, 24), (0, 0, 1)):
        starts.copy_(torch.tensor(counts, dtype=torch.int32))
        out.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        replayed = out.clone()
        assert torch.equal(replayed, cache.attend(q, table, lengths, starts)) and not replayed[counts[2]:].any()
        assert torch.isfinite(replayed).all()


# ------------------------------------------------------------------------------------------------ few queries beside outliers
@pytest.mark.parametrize("dim,blocksize", [(64, 64), (64, 128), (128, 64), (128, 128), (96, 64), (256, 64), (256, 256)])
@pytest.mark.parametrize("outlier", [1.0, 30.0, 300.0, 1000.0])
@pytest.mark.parametrize("n,new,group", [(700, 1, 4), (60, 12, 2), (5000, 3, 1)])
def test_bf16_queries_beside_outliers(Cache, dim, blocksize, outlier, n, new, group):
    """Large elements of queries and keys in different channels of the same 32: the scores are ordinary, and no bits of the small elements may be
    lost to the large ones.  What a score may be off by: 2^-7 of an exponent of 2, four times the 2^-9 that the kernel leaves on average; weights and
    values 2^-8 of `size`, the result's rounding 2^-9."""
    k, v, q = normal(35, n, 2, dim), normal(36, n, 2, dim).bfloat16(), normal(37, new, 2 * group, dim)
    k[:, :, 9], k[:, :, 20] = 0.0, outlier * k[:, :, 20].sign()
    q[:, :, 9], q[:, :, 20] = outlier, q[:, :, 20] / outlier
    k, q = k.bfloat16(), q.bfloat16()
    cache, table, lengths = one_sequence(Cache, k, v, blocksize)
    out = cache.attend(q.cuda(), table, lengths, ints(0, new))
    want, size, _ = expected(q, n - new, k, v, blocksize)
    off = (out.cpu().double() - want).abs()
    limit = size * (2 * math.log(2) * 2.0 ** -7 + 2.0 ** -8) + 2.0 ** -8 * want.abs()
    assert (off <= limit).all(), (int((off > limit).sum()), float((off / size).max()))
