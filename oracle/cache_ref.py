"""The 4-bit attention cache from its definition, in 64 bits on the CPU: what a written vector stands for, and attention over
tokens that are given as such values.  Scales and quotients are numbers of 32 bits by definition; everything else is exact or
in 64 bits."""
import math

import torch


def held(x, blocksize):
    """fp64: what the cache stands for after x [.., head_dim] (fp32 or bf16) has been written."""
    out = torch.zeros(x.shape, dtype=torch.float64)
    for first in range(0, x.shape[-1], blocksize):
        piece = x[..., first:first + blocksize].double()
        top = piece.abs().amax(-1, keepdim=True)
        scale = (top / 6.0).float().double()
        safe = torch.where(scale == 0, torch.ones_like(scale), scale)
        part = (piece / safe).float().double()
        size = part.abs().clamp(max=6.0)
        step = torch.where(size < 2, 0.5, torch.where(size < 4, 1.0, 2.0)).double()
        number = torch.round(size / step) * step * torch.where(part < 0, -1.0, 1.0).double()
        out[..., first:first + blocksize] = torch.where(scale == 0, torch.zeros_like(number), number * scale)
    return out


def seen(position, count, window=None, sinks=0):
    """bool [count]: which tokens a query at `position` sees."""
    j = torch.arange(count)
    see = j <= position
    if window is not None:
        see &= (position - j < window) | (j < sinks)
    return see


def attend(q, positions, keys, values, scale, window=None, sinks=0, there=None):
    """(result, size, spread) for one sequence, all fp64: q [n, heads, dim] at `positions`, keys and values [count, kv_heads, dim];
    there: bool [count], tokens that are in the cache.  size: sum_j p_j max|v_j|, the size that errors of the weights scale
    with; spread: scale sum_d |q_d k_d| with q's largest element per 32 in place of q, the most over the tokens seen: errors of
    q relative to its largest elements scale with that."""
    n, heads, dim = q.shape
    count, kv_heads, _ = keys.shape
    out = torch.zeros(n, heads, dim, dtype=torch.float64)
    size, spread = torch.zeros(n, heads, 1, dtype=torch.float64), torch.zeros(n, heads, 1, dtype=torch.float64)
    for i, position in enumerate(positions):
        see = seen(position, count, window, sinks) if position >= 0 else torch.zeros(count, dtype=torch.bool)
        if there is not None:
            see = see & there
        if not see.any():
            continue
        for h in range(heads):
            k, v = keys[see, h // (heads // kv_heads)], values[see, h // (heads // kv_heads)]
            p = torch.softmax(scale * (k @ q[i, h].double()), 0)
            out[i, h] = p @ v
            size[i, h] = (p * v.abs().amax(-1)).sum()
            coarse = torch.cat([c.abs().amax().expand(c.numel()) for c in q[i, h].double().split(32)])
            spread[i, h] = abs(scale) * (k.abs() @ coarse).max()
    return out, size, spread


def bounds(dtype, result, size, spread, dim):
    """Largest error that a correct kernel may have, element by element.  A weight is off by the factor exp(2 d), d the error
    of a score; its roundings scale with `size`.
      float32: scores are sums of dim + 8 roundings of 2^-24; the weights, 24 bits of the largest of 32 tokens, with exponentials
               good to 2^-20: 2^-18 in all
      bfloat16: queries to 2^-14 of the largest of 32 elements, so scores to 2^-13 with the rest; weights of 8 bits: 2^-9 each, and as
               much again for the split; the result is rounded to 8 bits"""
    if dtype == torch.float32:
        return size * (2 * (dim + 8) * 2.0 ** -24 * spread + 2.0 ** -18) + 2.0 ** -23 * result.abs()
    return size * (2 * 2.0 ** -13 * spread + 2.0 ** -8) + 2.0 ** -8 * result.abs()
