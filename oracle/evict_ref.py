"""What of an attention cache is kept, from the definition, in 64 bits on the CPU."""
import math

import torch

from oracle.cache_ref import seen


def weigh(q, positions, keys, scale, window=None, sinks=0, there=None):
    """(totals, spread) of one sequence in fp64: totals [kv_heads, count] for queries q [n, heads, dim] at `positions` and keys [count, kv_heads, dim];
    there: bool [count], tokens that are in the cache.  spread: the largest scale * sum |q_d k_d| of a query and a token that it sees, with which errors of
    scores scale."""
    n, heads, _ = q.shape
    count, kv_heads, _ = keys.shape
    totals, spread = torch.zeros(kv_heads, count, dtype=torch.float64), 0.0
    for i, position in enumerate(positions):
        see = seen(position, count, window, sinks) if position >= 0 else torch.zeros(count, dtype=torch.bool)
        if there is not None:
            see = see & there
        if not see.any():
            continue
        for h in range(heads):
            k, x = keys[see, h // (heads // kv_heads)], q[i, h].double()
            totals[h // (heads // kv_heads), see] += torch.softmax(scale * (k @ x), 0)
            spread = max(spread, float(abs(scale) * (k.abs() @ x.abs()).max()))
    return totals, spread


def bound(dim, rows, total, spread):
    """Largest error of totals.  A score is a sum of dim products and scales in fp32 (three times as many for fp32 queries), 2^-24 of `spread` each, and so is the
    largest one that it is taken from; an exponential and its argument are good to 2^-21 of the weight, its sums and the division to 2^-20; rows are added
    in fp32."""
    return total * (2 * (3 * dim + 16) * 2.0 ** -24 * max(1.0, spread) + 2.0 ** -19 + rows * 2.0 ** -24) + 2.0 ** -100


def evict(totals, length, keep, recent=0, sinks=0, there=None):
    """(from, to) of one sequence and head: places of the tokens that stay, and where they go."""
    places = [t for t in range(length) if there is None or there[t]]

    def order(t):
        x = float(totals[t])
        return (t < sinks or t >= length - recent, math.isnan(x), 0.0 if math.isnan(x) else x, -t)
    stay = sorted(sorted(places, key=order, reverse=True)[:keep])
    return stay, places[:len(stay)]
