"""Products with weights held in 4 bits, from the definition, in 64 bits on the CPU."""
import torch

from oracle.cache_ref import held


def product(x, weight, blocksize, bias=None):
    """(result, size) in fp64 of x [tokens, inputs] with weight [outputs, inputs] as it is held; size: the sum of the products' magnitudes, with which
    the errors of sums scale."""
    w = held(weight, blocksize)
    out, size = x.double() @ w.T, x.double().abs() @ w.abs().T
    return (out, size) if bias is None else (out + bias.double(), size + bias.double().abs())


def bounds(dtype, result, size, inputs, blocksize):
    """Largest error that a correct product may have.  Products are exact; every sum of fp32 numbers in it is off by at most half a step, 2^-24 of a number
    that is no larger than `size`, and in whatever order: inputs additions, one multiplication by a scale and one addition for every segment, the bias.
    (fp32 operands go through in three pieces: three times the additions.)  The result is rounded once to its type."""
    steps = (3 if dtype == torch.float32 else 1) * inputs + 2 * (-(-inputs // blocksize)) + 16
    half = torch.finfo(dtype).eps / 2
    return size * steps * 2.0 ** -24 + half * result.abs()
