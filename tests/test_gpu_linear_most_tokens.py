"""Products of as many tokens as a call may have, which are more than a launch takes."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens,inputs,outputs,dtype", [(2 ** 30 + 77, 1, 1, torch.bfloat16), (2 ** 31 - 256, 8, 1, torch.bfloat16), (2 ** 31 - 300, 3, 2, torch.float32)])
def test_more_tokens_than_a_launch_takes(tokens, inputs, outputs, dtype):
    """Tokens that repeat every 4099th: their results do too, and the first ones are looked at."""
    from qtensor.linear import QTensorLinear
    g = torch.Generator().manual_seed(1)
    w, few = torch.randn(outputs, inputs, generator=g), torch.randn(4099, inputs, generator=g).to(dtype)
    bias = torch.randn(outputs, generator=g)
    weights = QTensorLinear(inputs, outputs).quantize(w.cuda())
    whole = few.cuda().repeat(-(-tokens // 4099), 1)[:tokens]
    want = weights.product(few.cuda(), bias.cuda())
    held = weights.dequantize().double()
    assert torch.allclose(want.double(), few.cuda().double() @ held.T + bias.cuda().double(), rtol=2.0 ** -7, atol=2.0 ** -7)
    got = weights.product(whole, bias.cuda())
    del whole
    assert got.shape == (tokens, outputs)
    step = 4099 * 2 ** 14
    again = want.repeat(2 ** 14, 1)
    for first in range(0, tokens, step):
        part = got[first:first + step]
        assert torch.equal(part, again[:part.shape[0]]), first


def test_more_tokens_than_a_call_takes():
    from qtensor.linear import QTensorLinear
    weights = QTensorLinear(1, 1).quantize(torch.ones(1, 1, device="cuda"))
    with pytest.raises(RuntimeError):
        weights.product(torch.ones(1, device="cuda").expand(2 ** 31 - 255, 1))
