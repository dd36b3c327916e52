"""Inputs whose results show every bit of an fp32 operand, and how far a correct result may be off, in 64 bits on the CPU.

A vector with one element x that is not zero has the product x w with another one.  Its bits are multiplied in three pieces of eight, each times a number of two bits: the sums of the
two lower ones are numbers of 18 bits, exact, and that with the first one, of 26 bits, is rounded once, by a step of 2^-23 at most whichever way the matrix
instructions round.  Everything that is added to it is zero."""
import torch

HEADS = [(64, 64), (64, 256), (80, 64), (128, 64), (128, 128), (200, 64), (256, 64), (256, 256)]      # elements of a head, and of a segment
HEADS_OF_A_CALL = 16
LENGTHS, NEWS = [60, 128, 17, 100, 90], [20, 16, 5, 7, 16]


def all_bits(shape, g):
    """fp32 numbers of 24 bits, of any sign and size 1 to 8, whose last eight are 128 or more: what is left of one without them is off by 2^-17 or more."""
    bits = 2 ** 23 + (torch.randint(2 ** 15, shape, generator=g) << 8) + 128 + 2 * torch.randint(64, shape, generator=g) + 1
    return (bits.double() * 2.0 ** -23 * 2.0 ** torch.randint(3, shape, generator=g) * (1.0 - 2.0 * torch.randint(2, shape, generator=g))).float()


def cut(x):
    """What two pieces of eight bits hold of an fp32 number."""
    return (x.contiguous().view(torch.int32) & ~0xff).view(torch.float32)


def one_each(tokens, inputs, first, seed):
    """(x, where): x [tokens, inputs] with one element of every token, at where[t]."""
    where = (first + torch.arange(tokens)) % inputs
    x = torch.zeros(tokens, inputs)
    x[torch.arange(tokens), where] = all_bits((tokens,), torch.Generator().manual_seed(seed))
    return x, where


def product(x, where, held):
    """(result, limit) of such tokens with weights [outputs, inputs] in fp64: one rounding of the product, and one, half a step, of its multiplication by
    the scale: less than 2^-22."""
    want = x[torch.arange(len(where)), where].double().unsqueeze(1) * held[:, where].T
    return want, want.abs() * 2.0 ** -22


def queries(tokens, heads, dim, first):
    """[tokens, heads, dim] with one element of every head, at all places of a head in turn, of size 8 to 64 so that scores are large."""
    q = torch.zeros(tokens * heads, dim)
    where = (first + torch.arange(tokens * heads)) % dim
    q[torch.arange(tokens * heads), where] = 8 * all_bits((tokens * heads,), torch.Generator().manual_seed(first + 1))
    return q.view(tokens, heads, dim)


def weigh(q, positions, keys):
    """(totals, limit) [kv_heads, count] of one sequence, scores q k.  A score is off by its product's rounding (2^-23), that of its multiplication by the scale, of
    the scale by log2 e, of that constant, and by what its difference to the largest one is rounded (2^-24 each, of a number that is no larger than twice the largest score): e = 7 *
    2^-24 of the largest score; a weight by the factor exp(2 e).  Exponentials and their arguments are good to 2^-21 of a weight, the sum over 128 tokens at most (16 roundings in
    a row) and the division to 2^-20 and 2^-24, rows are added in fp32."""
    n, heads, _ = q.shape
    count, kv_heads, _ = keys.shape
    totals, limit = torch.zeros(kv_heads, count, dtype=torch.float64), torch.zeros(kv_heads, count, dtype=torch.float64)
    rows = n * heads // kv_heads
    for i, position in enumerate(positions):
        for h in range(heads):
            s = keys[:position + 1, h // (heads // kv_heads)] @ q[i, h].double()
            weight = torch.softmax(s, 0)
            totals[h // (heads // kv_heads), :position + 1] += weight
            limit[h // (heads // kv_heads), :position + 1] += weight * (torch.expm1(14 * 2.0 ** -24 * s.abs().max()) + 2.0 ** -19 + rows * 2.0 ** -24)
    return totals, limit + 2.0 ** -100
