"""All 24 bits of fp32 operands reach the sums of products with weights, and of weighed tokens.  Bounds that add up the roundings of long sums do not show it: inputs with one
element that is not zero do, as their result is one product, and has a handful of roundings (oracle/all_bits_ref.py)."""
import pytest
import torch

from oracle import all_bits_ref as A
from oracle import cache_ref as C

pytestmark = pytest.mark.gpu


# (outputs that take all routes of a product: few tokens with one, two, four and eight tiles of outputs to a workgroup, eight and sixteen waves, many with inputs shared by
# halves of a workgroup, by one, and in large tiles)
@pytest.mark.parametrize("tokens,inputs,outputs", [(1, 130, 33), (5, 300, 64), (8, 2100, 40), (9, 128, 16), (16, 300, 4096), (16, 2200, 8100), (16, 130, 16300), (13, 300, 20000),
                                                   (40, 257, 4000), (47, 300, 28700), (48, 300, 28700), (48, 2177, 500), (256, 300, 7168), (300, 129, 5800), (512, 385, 4400), (1024, 260, 10900)])
@pytest.mark.parametrize("blocksize", [64, 128, 256])
@pytest.mark.parametrize("aligned", [True, False])
def test_products(tokens, inputs, outputs, blocksize, aligned):
    from qtensor.linear import QTensorLinear
    w = torch.randn(outputs, inputs, generator=torch.Generator().manual_seed(1))
    held = C.held(w, blocksize)
    weights = QTensorLinear(inputs, outputs, blocksize=blocksize).quantize(w.cuda())
    # few tokens are sent several times, so that every element of a block is met
    for first in range(0, min(inputs, 128) if tokens < 64 else 1, tokens):
        x, where = A.one_each(tokens, inputs, first, seed=first)
        given = x.cuda()
        if not aligned:
            given = torch.full((tokens, inputs + 3), float("nan"), device="cuda")
            given[:, 1:inputs + 1] = x.cuda()
            given = given[:, 1:inputs + 1]
        want, limit = A.product(x, where, held)
        off = (weights.product(given).double().cpu() - want).abs()
        assert bool((off <= limit).all()), f"elements from {first} on: off by {float((off / limit.clamp(min=1e-300)).max()):.3g} of the bound"


@pytest.mark.parametrize("power", [-100, -118, -126, -140])
@pytest.mark.parametrize("tokens,outputs", [(16, 64), (512, 4400)])
def test_products_of_tokens_so_small_that_pieces_end(power, tokens, outputs):
    """bf16 ends at 2^-133: an element loses what it has behind that, times a number and its scale."""
    from qtensor.linear import QTensorLinear
    w = torch.randn(outputs, 128, generator=torch.Generator().manual_seed(1)) * 2.0 ** 100
    held = C.held(w, 64)
    x, where = A.one_each(tokens, 128, 3, seed=4)
    x *= 2.0 ** power
    want, limit = A.product(x, where, held)
    off = (QTensorLinear(128, outputs).quantize(w.cuda()).product(x.cuda()).double().cpu() - want).abs()
    assert bool((off <= limit + 2.0 ** -133 * held[:, where].T.abs()).all())


def placed(lengths, kv_heads, dim, blocksize, wide=0):
    from qtensor.cache import QTensorCache
    width = -(-max(lengths) // 16)
    table = torch.arange(len(lengths) * width, dtype=torch.int32).view(len(lengths), width)
    table = torch.cat([table, torch.full((len(lengths), wide), -1, dtype=torch.int32)], 1).cuda()
    cache = QTensorCache(len(lengths) * width, kv_heads, dim, page_size=16, blocksize=blocksize)
    k = torch.randn(sum(lengths), kv_heads, dim, generator=torch.Generator().manual_seed(3))
    counts, starts = torch.tensor(lengths, dtype=torch.int32).cuda(), torch.tensor([sum(lengths[:b]) for b in range(len(lengths) + 1)], dtype=torch.int32).cuda()
    cache.write(k.cuda(), k.cuda(), table, counts, starts)
    return cache, table, counts, k.split(lengths)


def compare(got, q, lengths, news, keys, blocksize):
    at = 0
    for b, (n, new) in enumerate(zip(lengths, news)):
        want, limit = A.weigh(q[at:at + new], range(n - new, n), C.held(keys[b], blocksize))
        off = (got[b, :, :n].double().cpu() - want).abs()
        assert bool((off <= limit).all()), f"sequence {b}: off by {float((off / limit).max()):.3g} of the bound"
        at += new


@pytest.mark.parametrize("dim,blocksize", A.HEADS)
@pytest.mark.parametrize("wide", [0, 2 ** 19])
def test_weights_of_a_token_of_each_sequence(dim, blocksize, wide):
    """With their scores kept, and with a table that leaves no room for them."""
    lengths = A.LENGTHS[:2] if wide else A.LENGTHS
    cache, table, counts, keys = placed(lengths, 2, dim, blocksize, wide)
    for first in range(0, dim, A.HEADS_OF_A_CALL * len(lengths)):
        q = A.queries(len(lengths), A.HEADS_OF_A_CALL, dim, first)
        compare(cache.weigh(cache.totals(table), q.cuda(), table, counts, scale=1.0), q, lengths, [1] * len(lengths), keys, blocksize)


@pytest.mark.parametrize("dim,blocksize", A.HEADS)
@pytest.mark.parametrize("wide", [0, 2000])
def test_weights_of_pieces_of_prompts(dim, blocksize, wide):
    """By workgroups that share tokens, and by waves with tokens of their own."""
    cache, table, counts, keys = placed(A.LENGTHS, 2, dim, blocksize, wide)
    q = A.queries(sum(A.NEWS), 4, dim, 0)
    starts = torch.tensor([sum(A.NEWS[:b]) for b in range(len(A.NEWS) + 1)], dtype=torch.int32).cuda()
    compare(cache.weigh(cache.totals(table), q.cuda(), table, counts, starts, scale=1.0), q, A.LENGTHS, A.NEWS, keys, blocksize)
