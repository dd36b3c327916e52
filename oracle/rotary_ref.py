"""Rotary positions from their definition, in 64 bits on the CPU."""
import torch


def turned(x, positions, frequencies, dims, magnitude=1.0, interleaved=False, back=False):
    """(result, size) in fp64 of x [.., tokens, heads, head_dim] at positions [.., tokens]; size: the sum of the magnitudes of a result's two products."""
    angle = positions.double().unsqueeze(-1).unsqueeze(-1) * torch.as_tensor(frequencies, dtype=torch.float64)
    c, s = (magnitude * angle.cos()).float().double(), (magnitude * angle.sin()).float().double()
    if back:
        s = -s
    x = x.double()
    first, second = (torch.arange(0, dims, 2), torch.arange(1, dims, 2)) if interleaved else (torch.arange(dims // 2), torch.arange(dims // 2, dims))
    out, size = x.clone(), torch.zeros_like(x)
    a, b = x[..., first], x[..., second]
    out[..., first], out[..., second] = a * c - b * s, b * c + a * s
    size[..., first], size[..., second] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    return out, size


def bounds(dtype, result, size):
    """Largest error of a correct result: cosines and sines next to the border of two fp32 numbers may be the other one (2^-23 of them), a rounding of each
    product and of their sum (2^-24), and the result's."""
    return size * (2.0 ** -23 + 2 * 2.0 ** -24) + torch.finfo(dtype).eps / 2 * result.abs()
