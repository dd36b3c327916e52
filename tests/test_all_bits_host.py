"""What the tests of all bits (test_gpu_all_bits.py) can see: results of operands that have lost their last eight bits are beyond the bounds, for every place of an element."""
import pytest
import torch

from oracle import all_bits_ref as A
from oracle import cache_ref as C


def test_numbers_of_all_bits():
    x = A.all_bits((4000,), torch.Generator().manual_seed(1))
    assert bool(((x.abs() >= 1) & (x.abs() < 8)).all())
    lost = ((x.double() - A.cut(x).double()) / x.double()).abs()
    assert float(lost.min()) >= 2.0 ** -17 and float(lost.max()) < 2.0 ** -15
    pieces = [A.cut(x), x - A.cut(x)]
    assert torch.equal(pieces[0].double() + pieces[1].double(), x.double())


@pytest.mark.parametrize("inputs,blocksize", [(64, 64), (300, 64), (2200, 256)])
def test_products_of_cut_tokens_are_seen(inputs, blocksize):
    held = C.held(torch.randn(50, inputs, generator=torch.Generator().manual_seed(1)), blocksize)
    x, where = A.one_each(inputs, inputs, 5, seed=2)
    want, limit = A.product(x, where, held)
    assert torch.allclose(x.double() @ held.T, want, rtol=1e-15, atol=0)
    less, _ = A.product(A.cut(x), where, held)
    assert bool(((less - want).abs() > 8 * limit)[want != 0].all()) and float((want != 0).double().mean()) > 0.5
    assert not ((want.float().double() - want).abs() > limit).any()


@pytest.mark.parametrize("dim,blocksize", A.HEADS)
def test_weights_of_cut_queries_are_seen(dim, blocksize):
    g = torch.Generator().manual_seed(3)
    for n, new, heads in [(n, new, 4) for n, new in zip(A.LENGTHS, A.NEWS)] + [(n, 1, A.HEADS_OF_A_CALL) for n in A.LENGTHS]:
        keys = C.held(torch.randn(n, 2, dim, generator=g), blocksize)
        q = A.queries(new, heads, dim, 11)
        want, limit = A.weigh(q, range(n - new, n), keys)
        assert abs(float(want.sum()) - new * heads) < 1e-9
        less, _ = A.weigh(A.cut(q), range(n - new, n), keys)
        assert float(((less - want).abs() / limit).max()) > 4
