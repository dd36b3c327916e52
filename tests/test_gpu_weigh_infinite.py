"""Weights that queries with an infinite element give: the formula has NaN for every token that such a query sees, and for no other."""
import math

import pytest
import torch

from oracle import cache_ref as C
from oracle import evict_ref as R

pytestmark = pytest.mark.gpu


def vectors(shape, dtype, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def filled(lengths, kv_heads, dim, dtype, wide=0):
    """Keys whose element 7 is positive: an infinite product has the sign of the query's element there."""
    from qtensor.cache import QTensorCache
    width = -(-max(lengths) // 16)
    table = torch.arange(len(lengths) * width, dtype=torch.int32).view(len(lengths), width)
    table = torch.cat([table, torch.full((len(lengths), wide), -1, dtype=torch.int32)], 1).cuda()
    cache = QTensorCache(len(lengths) * width, kv_heads, dim, page_size=16)
    k = vectors((sum(lengths), kv_heads, dim), torch.float32, 1)
    k[..., 7] = k[..., 7].abs() + 0.5
    k = k.to(dtype)
    starts = torch.tensor([sum(lengths[:b]) for b in range(len(lengths) + 1)], dtype=torch.int32).cuda()
    counts = torch.tensor(lengths, dtype=torch.int32).cuda()
    cache.write(k.cuda(), k.cuda(), table, counts, starts)
    return cache, table, counts, k.split(lengths)


def check(cache, got, q, lengths, news, keys, there=None, **seen):
    at = 0
    for b, (n, new) in enumerate(zip(lengths, news)):
        want, _ = R.weigh(q[at:at + new], range(n - new, n), C.held(keys[b], 64), 1 / math.sqrt(q.shape[2]), **seen)
        here = got[b, :, :n].double().cpu()
        assert torch.equal(torch.isnan(here), torch.isnan(want)), f"sequence {b}"
        good = ~torch.isnan(want)
        assert torch.allclose(here[good], want[good], rtol=2.0 ** -10, atol=0)      # (how near is looked at elsewhere)
        assert not got[b, :, n:].any()
        at += new


@pytest.mark.parametrize("bad", [-math.inf, math.inf])
@pytest.mark.parametrize("dim", [64, 128, 200])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("wide", [0, 2 ** 19 + 3])
def test_a_token_of_each_sequence(dtype, dim, bad, wide):
    """With room for the scores, and with a table so wide that there is none."""
    lengths = [1, 70, 300]
    cache, table, counts, keys = filled(lengths, 2, dim, dtype, wide)
    q = vectors((3, 8 if not wide else 32, dim), dtype, 2)
    q[0, 1, 7] = q[2, -1, 7] = bad
    got = cache.weigh(cache.totals(table), q.cuda(), table, counts)
    check(cache, got, q, lengths, [1, 1, 1], keys)


@pytest.mark.parametrize("bad", [-math.inf, math.inf])
@pytest.mark.parametrize("dim", [64, 128, 200])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("seen", [{}, dict(window=9, sinks=2)])
def test_pieces_of_prompts(dtype, dim, bad, seen):
    lengths, news = [90, 3000, 33], [90, 40, 5]
    cache, table, counts, keys = filled(lengths, 2, dim, dtype)
    q = vectors((sum(news), 4, dim), dtype, 2)
    q[0, 0, 7] = q[60, 3, 7] = q[100, 1, 7] = q[134, 2, 7] = bad
    starts = torch.tensor([0, 90, 130, 135], dtype=torch.int32).cuda()
    got = cache.weigh(cache.totals(table), q.cuda(), table, counts, starts, **seen)
    check(cache, got, q, lengths, news, keys, **seen)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_of_few_tokens_agrees(dtype):
    cache, table, counts, keys = filled([1, 70, 300], 2, 64, dtype)
    for bad in (-math.inf, math.inf):
        q = vectors((3, 4, 64), dtype, 2)
        q[0, 1, 7] = q[2, 3, 7] = bad
        out = cache.attend(q.cuda(), table, counts).cpu()
        assert bool(torch.isnan(out[0, 1]).all()) and bool(torch.isnan(out[2, 3]).all()) and int(torch.isnan(out).sum()) == 128


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_queries_that_see_nothing(dtype):
    """In front of their sequence, or where none of its pages is there: no weights, whatever they hold."""
    cache, table, counts, _ = filled([20, 40], 2, 64, dtype, 3)
    table[1] = -1
    q = vectors((66, 4, 64), dtype, 2)
    q[:6, :, 7] = -math.inf
    q[26:, :, 7] = math.inf
    got = cache.weigh(cache.totals(table), q.cuda(), table, counts, torch.tensor([0, 26, 66], dtype=torch.int32).cuda()).cpu()
    assert bool(torch.isfinite(got).all()) and not got[1].any() and torch.allclose(got[0].sum(-1), torch.full((2,), 40.0))
    got = cache.weigh(cache.totals(table), q[-2:].cuda(), table, counts * torch.tensor([0, 1], dtype=torch.int32).cuda())
    assert not got.any()
