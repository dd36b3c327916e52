"""Weights held in 4 bits (qtensor.linear) against their definition in 64 bits (oracle/linear_ref.py): what is held bit for bit, products
to the bounds of oracle.linear_ref.bounds, which follow from the number of roundings."""
import math

import pytest
import torch

from oracle import cache_ref as C
from oracle import linear_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def Linear():
    from qtensor.linear import QTensorLinear
    import qtensor.functional as F
    assert torch.cuda.is_available() and F.lib is not None
    return QTensorLinear


def matrix(rows, columns, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, columns, generator=g)
    x[:, ::13] *= 7.0
    x[::5] *= 0.01
    return x.to(dtype)


def equal(a, b):
    return torch.equal(torch.nan_to_num(a, nan=12345.0), torch.nan_to_num(b, nan=12345.0))


def check(got, x, w, blocksize, bias=None):
    want, size = R.product(x, w, blocksize, bias)
    off = (got.double().cpu() - want).abs()
    limit = R.bounds(x.dtype, want, size, w.shape[1], blocksize)
    assert got.dtype == x.dtype and tuple(got.shape) == tuple(want.shape)
    assert bool((off <= limit).all()), f"off by {float((off / limit.clamp(min=1e-300)).max()):.3g} of the bound"


@pytest.mark.parametrize("inputs,outputs", [(64, 16), (1, 1), (128, 5), (130, 33), (257, 17), (63, 100), (1000, 50), (768, 48)])
@pytest.mark.parametrize("blocksize", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_what_is_held_is_its_definition(Linear, inputs, outputs, blocksize, dtype):
    w = matrix(outputs, inputs, dtype, inputs + outputs)
    if outputs > 3:
        w[1] = 0
        w[2] *= 1e-30
        w[3, inputs // 2] = math.inf
    wide = torch.full((outputs, inputs + 3), 5.0, dtype=dtype).cuda()
    wide[:, :inputs] = w.cuda()
    held = Linear(inputs, outputs, blocksize=blocksize).quantize(wide[:, :inputs])
    want = C.held(w, blocksize)
    assert equal(held.dequantize(), want.float().cuda())
    assert equal(held.dequantize(torch.bfloat16), want.float().to(torch.bfloat16).cuda())


@pytest.mark.parametrize("tokens", [1, 2, 3, 15, 16, 17, 31, 33, 64, 65, 100, 129, 200, 300, 513])
@pytest.mark.parametrize("inputs,outputs", [(64, 16), (1, 3), (129, 33), (768, 257), (1000, 128)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_products(Linear, tokens, inputs, outputs, dtype):
    for blocksize in (64, 128, 256):
        w, x = matrix(outputs, inputs, dtype, 1), matrix(tokens, inputs, dtype, 2)
        bias = torch.randn(outputs, generator=torch.Generator().manual_seed(3))
        held = Linear(inputs, outputs, blocksize=blocksize).quantize(w.cuda())
        check(held.product(x.cuda()), x, w, blocksize)
        check(held.product(x.cuda(), bias.cuda()), x, w, blocksize, bias)
        if dtype == torch.bfloat16:
            check(held.product(x.cuda(), bias.to(dtype).cuda()), x, w, blocksize, bias.to(dtype))


@pytest.mark.parametrize("tokens,inputs,outputs", [(1, 8192, 2304), (4, 5000, 4001), (20, 4096, 1024), (700, 2048, 640), (1, 30000, 16)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_larger_products(Linear, tokens, inputs, outputs, dtype):
    w, x = matrix(outputs, inputs, dtype, 4), matrix(tokens, inputs, dtype, 5)
    check(Linear(inputs, outputs).quantize(w.cuda()).product(x.cuda()), x, w, 64)


@pytest.mark.parametrize("tokens,inputs,outputs", [(3, 70, 17000), (20, 129, 17000), (40, 70, 17001), (30, 200, 9000), (60, 70, 8300), (64, 257, 8321),
                                                   (15, 300, 9000), (9, 140, 5000), (250, 131, 4090)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_tiles_of_all_sizes(Linear, tokens, inputs, outputs, dtype):
    w, x = matrix(outputs, inputs, dtype, 14), matrix(tokens, inputs, dtype, 15)
    for blocksize in (64, 128, 256):
        held, bias = Linear(inputs, outputs, blocksize=blocksize).quantize(w.cuda()), torch.randn(outputs, generator=torch.Generator().manual_seed(16))
        check(held.product(x.cuda(), bias.cuda()), x, w, blocksize, bias)


@pytest.mark.parametrize("tokens,inputs,outputs", [(1030, 130, 2100), (1100, 64, 2050), (4200, 70, 8200), (70, 385, 33000)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_many_tokens_and_outputs(Linear, tokens, inputs, outputs, dtype):
    """Enough of both for the kernels of many tokens, with edges in every direction; tokens that are not finite, rows that are not aligned."""
    w, x = matrix(outputs, inputs, dtype, 4), matrix(tokens, inputs, dtype, 5)
    held, bias = Linear(inputs, outputs, blocksize=128).quantize(w.cuda()), torch.randn(outputs, generator=torch.Generator().manual_seed(6))
    got = held.product(x.cuda(), bias.cuda())
    check(got, x, w, 128, bias)
    wide = torch.full((tokens, inputs + 3), math.nan, dtype=dtype, device="cuda")
    wide[:, 1:inputs + 1] = x.cuda()
    assert torch.equal(held.product(wide[:, 1:inputs + 1], bias.cuda()), got)
    wide = torch.full((tokens, inputs + 8 - inputs % 8), math.nan, dtype=dtype, device="cuda")
    wide[:, :inputs] = x.cuda()
    wide[tokens // 2, 3] = math.inf
    other = held.product(wide[:, :inputs], bias.cuda())
    assert not bool(torch.isfinite(other[tokens // 2]).any())
    other[tokens // 2] = got[tokens // 2]
    assert torch.equal(other, got)


@pytest.mark.parametrize("tokens", [1, 20, 300])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides_shapes_and_given_results(Linear, tokens, dtype):
    w, x = matrix(50, 200, dtype, 6), matrix(tokens, 200, dtype, 7)
    held = Linear(200, 50).quantize(w.cuda())
    want = held.product(x.cuda())
    check(want, x, w, 64)
    for offset in (1, 3):                                        # rows and first elements that are not aligned
        wide = torch.full((tokens, 207), math.nan, dtype=dtype, device="cuda")
        wide[:, offset:offset + 200] = x.cuda()
        assert torch.equal(held.product(wide[:, offset:offset + 200]), want)
    assert torch.equal(held.product(x.cuda().view(1, tokens, 1, 200)), want.view(1, tokens, 1, 50))
    assert torch.equal(held.product(x.cuda()[0]), held.product(x[:1].cuda())[0])
    assert torch.equal(held.product(x[:1].cuda().expand(tokens, 200)), held.product(x[:1].repeat(tokens, 1).cuda()))
    guarded = torch.full((tokens + 2, 50), 7.0, dtype=dtype, device="cuda")
    out = guarded[1:-1]
    assert held.product(x.cuda(), out=out) is out and torch.equal(out, want)
    assert bool((guarded[0] == 7).all()) and bool((guarded[-1] == 7).all())
    assert held.product(x.cuda()[:0]).shape == (0, 50)


@pytest.mark.parametrize("tokens", [3, 40, 300])
def test_numbers_that_are_not_finite(Linear, tokens):
    """An infinite or NaN element reaches its token alone, an infinite weight its output alone."""
    w, x = matrix(40, 300, torch.float32, 8), matrix(tokens, 300, torch.float32, 9)
    w[w == 0] = 1.0
    for dtype in (torch.float32, torch.bfloat16):
        good = Linear(300, 40).quantize(w.cuda()).product(x.to(dtype).cuda())
        bad = x.clone()
        bad[1, 7], bad[2, 299] = math.inf, math.nan
        got = Linear(300, 40).quantize(w.cuda()).product(bad.to(dtype).cuda())
        assert torch.equal(got[0], good[0]) and torch.equal(got[3:], good[3:])
        want = bad[1:3].to(dtype).double() @ C.held(w, 64).T
        assert equal(torch.isfinite(got[1:3]).float().cpu(), torch.isfinite(want).float())
        assert equal(torch.isnan(got[1:3]).float().cpu(), torch.isnan(want).float())
        broken = w.clone()
        broken[5, 299] = math.inf
        got = Linear(300, 40).quantize(broken.cuda()).product(x.to(dtype).cuda())
        assert bool(torch.isnan(got[:, 5]).all())
        rest = [i for i in range(40) if i != 5]
        assert torch.equal(got[:, rest], good[:, rest])
    tiny = torch.tensor([[0x7f800001]], dtype=torch.int32).view(torch.float32).expand(1, 300).contiguous()     # a NaN of low bits alone
    assert bool(torch.isnan(Linear(300, 40).quantize(w.cuda()).product(tiny.cuda())).all())
    large = torch.full((1, 300), 3.4e38)
    large[0, 1:] = 0
    small = w * 1e-30
    check(Linear(300, 40).quantize(small.cuda()).product((large / 1024).cuda()), large / 1024, small, 64)


@pytest.mark.parametrize("tokens", [1, 40, 300])
def test_another_stream_and_a_captured_call(Linear, tokens):
    w, x = matrix(64, 256, torch.bfloat16, 10).cuda(), matrix(tokens, 256, torch.bfloat16, 11).cuda()
    held = Linear(256, 64).quantize(w)
    want = held.product(x)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        got = held.product(x)
    stream.synchronize()
    assert torch.equal(got, want)
    graph, given = torch.cuda.CUDAGraph(), x.clone()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = held.product(given)
    for n in range(3):
        given.copy_(x * (n + 1))
        graph.replay()
        assert torch.equal(out, held.product(x * (n + 1)))


def test_results_do_not_change_from_call_to_call(Linear):
    for tokens in (1, 30, 500):
        w, x = matrix(300, 2000, torch.float32, 12).cuda(), matrix(tokens, 2000, torch.float32, 13).cuda()
        held = Linear(2000, 300).quantize(w)
        want = held.product(x)
        for _ in range(5):
            assert torch.equal(held.product(x), want)


def test_refusals(Linear):
    held = Linear(128, 20).quantize(torch.ones(20, 128, device="cuda"))
    x = torch.ones(4, 128, device="cuda")
    for bad in (x[:, :64], x.double(), x.half(), x.cpu(), x.T, torch.ones((), device="cuda"), torch.ones(4, 256, device="cuda")[:, ::2]):
        with pytest.raises((ValueError, RuntimeError)):
            held.product(bad)
    for bad in (torch.ones(19, device="cuda"), torch.ones(20, dtype=torch.bfloat16, device="cuda"), torch.ones(20), torch.ones(40, device="cuda")[::2]):
        with pytest.raises(ValueError):
            held.product(x, bad)
    square = Linear(128, 128).quantize(torch.ones(128, 128, device="cuda"))
    for bad in (x, x[:2], torch.ones(4, 128, dtype=torch.bfloat16, device="cuda"), torch.ones(128, 4, device="cuda").T):
        with pytest.raises(ValueError):
            square.product(x, out=bad)
    with pytest.raises(RuntimeError):
        held.product(x.clone().requires_grad_())
    with torch.no_grad():
        held.product(x.clone().requires_grad_())
    for bad in (torch.ones(20, 127, device="cuda"), torch.ones(20, 128), torch.ones(128, 20, device="cuda").T, torch.ones(20, 128, device="cuda").half()):
        with pytest.raises((ValueError, RuntimeError)):
            held.quantize(bad)
    held.scales = held.scales[:1]
    with pytest.raises(ValueError):
        held.product(x)


def test_a_checkpoint(Linear, tmp_path):
    held = Linear(200, 30, blocksize=128).quantize(matrix(30, 200, torch.float32, 14).cuda())
    torch.save(held.state_dict(), tmp_path / "w.pt")
    other = Linear(200, 30, blocksize=128)
    other.load_state_dict(torch.load(tmp_path / "w.pt", weights_only=True))
    assert torch.equal(other.dequantize(), held.dequantize())
    with pytest.raises(ValueError):
        Linear(200, 30).load_state_dict(held.state_dict())


@pytest.mark.parametrize("inputs", [50, 128, 130, 384, 520, 1000])
@pytest.mark.parametrize("tokens,outputs", [(900, 2048), (1000, 1950), (130, 10001)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_inputs_shared_by_the_halves_of_a_workgroup(Linear, tokens, outputs, inputs, dtype):
    """As many tiles as units or a little less: one block of inputs, which leaves a half without any, odd and even numbers of them."""
    w, x = matrix(outputs, inputs, dtype, 24), matrix(tokens, inputs, dtype, 25)
    held, bias = Linear(inputs, outputs).quantize(w.cuda()), torch.randn(outputs, generator=torch.Generator().manual_seed(26))
    got = held.product(x.cuda(), bias.cuda())
    check(got, x, w, 64, bias)
    assert torch.equal(held.product(x.cuda(), bias.cuda()), got)
    wide = torch.full((tokens, inputs + 3), math.nan, dtype=dtype, device="cuda")
    wide[:, 1:inputs + 1] = x.cuda()
    assert torch.equal(held.product(wide[:, 1:inputs + 1], bias.cuda()), got)


@pytest.mark.parametrize("tokens", [1, 7, 16, 32, 33, 48, 49])
@pytest.mark.parametrize("inputs,outputs", [(130, 40001), (257, 30000)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_few_tokens_and_as_many_outputs_as_a_vocabulary(Linear, tokens, inputs, outputs, dtype):
    w, x = matrix(outputs, inputs, dtype, 34), matrix(tokens, inputs, dtype, 35)
    for blocksize in (64, 256):
        check(Linear(inputs, outputs, blocksize=blocksize).quantize(w.cuda()).product(x.cuda()), x, w, blocksize)


@pytest.mark.parametrize("tokens", [1, 3, 16, 40])
@pytest.mark.parametrize("inputs", [2048, 2049, 2200, 9813])
@pytest.mark.parametrize("outputs", [20, 2100, 5001, 9000])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_long_inputs(Linear, tokens, inputs, outputs, dtype):
    """More blocks of inputs than waves, fewer of the last ones, and as few as make eight waves enough."""
    if inputs == 9813 and outputs > 2100:
        outputs //= 4
    w, x = matrix(outputs, inputs, dtype, 44), matrix(tokens, inputs, dtype, 45)
    check(Linear(inputs, outputs).quantize(w.cuda()).product(x.cuda()), x, w, 64)
