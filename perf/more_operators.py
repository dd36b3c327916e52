"""What a model that generates from an attention cache in 4 bits needs around that cache, as cases whose speed can be measured.

The cache is the one of operators.py: vectors of a head in segments of `blocksize`, an fp32 scale (largest magnitude over 6) and
4-bit floating numbers, tokens in pages.  Five calls:

  product  x W' + bias with weights W [outputs, inputs] in the same 4-bit numbers, a scale for `blocksize` inputs of an output
  rotary   queries and keys turned by their positions, forwards and backwards: element pairs (a, b) of the first `dims` elements of a
           head become (a c - b s, b c + a s), c and s the fp32 numbers nearest to magnitude * cos and sin (position * frequency), each
           product rounded once; the gradient is turned back
  write    queries turned, keys turned and encoded into the cache, values encoded: the pass returns the queries and what the
           cache then stands for
  weigh    the weights softmax(scale q k) that the new tokens give the tokens they see, added up per token and head of the cache
           over queries and over the query heads that share the head
  evict    of every sequence and head the `keep` tokens are kept whose sum of weights is largest (ties to the earlier token), the first
           `sinks` and the last `recent` among them in any case; in their order they move to the front; the pass returns what the
           cache then stands for, the sums and the new lengths

`run` computes them in elementary torch operations, or where `own` is true by the framework's calls.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


def _product(name, dtype, tokens, inputs, outputs, blocksize=64, bias=False):
    return dict(name=name, call="product", dtype=dtype, tokens=tokens, inputs=inputs, outputs=outputs, blocksize=blocksize, bias=bias)


def _rotary(name, dtype, batch, tokens, heads, kv_heads, head_dim, dims, interleaved=False, scaling="none", first=0):
    """first: the position of a sequence's first token."""
    return dict(name=name, call="rotary", dtype=dtype, batch=batch, tokens=tokens, heads=heads, kv_heads=kv_heads, head_dim=head_dim, dims=dims,
                interleaved=interleaved, scaling=scaling, first=first)


def _cached(name, call, dtype, kv_heads, head_dim, blocksize, page_size, batch, shortest, longest, new=1, group=1, window=0, sinks=0, keep=0, recent=0,
            dims=0, interleaved=False, scaling="none", moved=False):
    """new: 0 for all tokens of every sequence, 1 for the last one, more for up to so many; group: query heads per key head; moved: a
    token's position is not its place in the cache (tokens have been evicted)."""
    return dict(name=name, call=call, dtype=dtype, kv_heads=kv_heads, head_dim=head_dim, blocksize=blocksize, page_size=page_size, batch=batch,
                shortest=shortest, longest=longest, new=new, group=group, window=window, sinks=sinks, keep=keep, recent=recent, dims=dims,
                interleaved=interleaved, scaling=scaling, moved=moved)


def listed():
    return [
        # one token through a projection of a layer of width 768: nothing but latency
        _product("product token", "bfloat16", 1, 768, 2304, bias=True),
        # one token through the widest matrix of a large model: all of the time is reading it
        _product("product wide", "bfloat16", 1, 8192, 28672, 128),
        # a step of an ordinary batch of sequences
        _product("product step", "bfloat16", 32, 4096, 14336),
        # a few tokens in 32 bits, sizes that no tile divides
        _product("product in 32 bits", "float32", 5, 1000, 5003, bias=True),
        # prompts: all of the time is arithmetic
        _product("product prompts", "bfloat16", 6000, 4096, 11008),
        # a step of training: whole sequences, grouped heads
        _rotary("rotary training", "bfloat16", 8, 2048, 32, 8, 128, 128),
        # part of a small model's heads, neighbours paired, far positions of a stretched context
        _rotary("rotary part", "float32", 2, 197, 12, 12, 80, 32, True, "parts", 100000),
        # a step of generation
        _cached("write step", "write", "bfloat16", 8, 128, 64, 64, 32, 100, 8000, 1, 4, dims=128, moved=True),
        # prompts of all lengths as they come in
        _cached("write prompts", "write", "bfloat16", 8, 128, 64, 64, 9, 1, 3500, 0, 4, dims=128),
        # weights of a step of generation, sequences of very different lengths
        _cached("weigh step", "weigh", "bfloat16", 8, 128, 64, 64, 32, 100, 8000, 1, 4),
        # weights that the last tokens of long prompts give, to choose what is kept of them
        _cached("weigh window", "weigh", "bfloat16", 8, 128, 64, 64, 4, 9000, 32768, 32, 4),
        # the cache of a batch cut down
        _cached("evict batch", "evict", "bfloat16", 8, 128, 64, 64, 24, 1000, 12000, keep=2048, recent=128, sinks=4),
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    call = rng.choice(["product", "product", "product", "rotary", "write", "weigh", "weigh", "evict"])
    dtype = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])
    if call == "product":
        inputs, outputs = (rng.choice([n, n, 64 * max(1, n // 64)]) for n in (_log_uniform(rng, 64, 16384), _log_uniform(rng, 16, 32768)))
        most = 2.0e11 / (inputs * outputs) / (1 if dtype == "bfloat16" else 8)
        tokens = _log_uniform(rng, 1, max(2, min(8192, most)))
        if rng.random() < 0.4:
            tokens = rng.choice([1, 1, 2, 4, 8, 16, 17, 33, 64])
        return _product(None, dtype, tokens, inputs, outputs, rng.choice([64, 64, 128, 256]), rng.random() < 0.3)
    head_dim = rng.choice([64, 64, 72, 80, 96, 112, 128, 128, 128, 192, 256, 2 * _log_uniform(rng, 17, 128)])
    dims = rng.choice([head_dim, head_dim, 2 * max(1, head_dim // 4), 2 * _log_uniform(rng, 1, head_dim // 2)])
    kv_heads, group = _log_uniform(rng, 1, 16), rng.choice([1, 2, 3, 4, 4, 5, 6, 7, 8, 8, 16])
    interleaved, scaling = rng.random() < 0.4, rng.choice(["none", "none", "all", "base", "parts"])
    if call == "rotary":
        batch = _log_uniform(rng, 1, 16)
        most = 4.0e7 / (batch * kv_heads * (group + 1) * head_dim)
        return _rotary(None, dtype, batch, _log_uniform(rng, 1, max(2, min(8192, most))), kv_heads * group, kv_heads, head_dim, dims, interleaved, scaling,
                       rng.choice([0, 0, _log_uniform(rng, 1, 500000)]))
    page_size, blocksize, batch = rng.choice([16, 32, 64, 128]), rng.choice([64, 64, 128, 256]), _log_uniform(rng, 1, 48)
    each = kv_heads * max(1.0, head_dim / 128)                       # vectors of 128 of a token
    if call == "write":
        new = rng.choice([0, 0, 1, 1, _log_uniform(rng, 2, 1000)])
        longest = _log_uniform(rng, 1, min(8192, max(64, int(2.5e5 / (batch * each * (1 + group / 4))))))
        return _cached(None, call, dtype, kv_heads, head_dim, blocksize, page_size, batch, rng.choice([0, longest // 8, longest]), longest, new, group,
                       dims=dims, interleaved=interleaved, scaling=scaling, moved=rng.random() < 0.3)
    if call == "weigh":
        new = rng.choice([1, 1, 1, 0, 16, 32, _log_uniform(rng, 2, 200)])
        batch = batch if new == 1 else min(batch, 6)
        # scores in 32 bits of all pairs, and all keys decoded, have to be held by the plain form
        pairs = 1.2e8 / (batch * kv_heads * group)
        longest = int(math.sqrt(pairs)) if new == 0 else int(min(pairs / new, 1.0e6 / (batch * each)))
        longest = _log_uniform(rng, 1, min(65536, max(64, longest)))
        window, sinks = rng.choice([(0, 0), (0, 0), (_log_uniform(rng, 1, 8192), rng.choice([0, 1, 4, 16, 100]))])
        return _cached(None, call, dtype, kv_heads, head_dim, blocksize, page_size, batch, rng.choice([0, longest // 8, longest]), longest, new, group,
                       window, sinks)
    longest = _log_uniform(rng, 16, min(65536, max(64, int(1.0e6 / (batch * each)))))
    keep = _log_uniform(rng, 2, longest)
    recent = rng.choice([0, keep // 4, keep // 2])
    return _cached(None, call, dtype, kv_heads, head_dim, blocksize, page_size, batch, rng.choice([0, longest // 8, longest]), longest, keep=keep,
                   recent=recent, sinks=min(keep - recent, rng.choice([0, 1, 4])))


# ------------------------------------------------------------------------------------------------ what a case holds
def _spread(low, high, at):
    return low + int(round((high - low) * ((0.5 + 0.6180339887498949 * at) % 1.0)))


def _counts(case):
    """Tokens of every sequence and how many of them the call is about: the first is the longest, others are spread evenly."""
    lengths = [case["longest"]] + [_spread(case["shortest"], case["longest"], b) for b in range(1, case["batch"])]
    if case["shortest"] == 0:
        lengths = [0 if b % 5 == 3 else n for b, n in enumerate(lengths)]
    if case["new"] == 0:
        return lengths, list(lengths)
    if case["new"] == 1:
        return lengths, [1] * case["batch"]
    return lengths, [min(n, 1 if b % 3 == 2 else _spread(1, case["new"], 2 * b + 1)) for b, n in enumerate(lengths)]


def _frequencies(case):
    """Of the pairs of `dims` elements, for position * frequency, in 64 bits on the host, and the magnitude of what is turned: as a
    model was trained, all of them slower by 8, by a larger base, or only those slower that turn less than 1 to 32 times in 4096
    places (with a magnitude of 0.1 ln 8 + 1)."""
    dims, base, factor = case["dims"], 10000.0, 8.0
    if case["scaling"] == "base":
        base *= factor ** (dims / max(1, dims - 2))
    speed = [base ** (-2.0 * i / dims) for i in range(dims // 2)]
    if case["scaling"] == "all":
        speed = [f / factor for f in speed]
    if case["scaling"] == "parts":
        kept = [min(1.0, max(0.0, (4096 * f / (2 * math.pi) - 1.0) / (32.0 - 1.0))) for f in speed]
        speed = [f * k + f / factor * (1 - k) for f, k in zip(speed, kept)]
    return speed, 0.1 * math.log(factor) + 1.0 if case["scaling"] == "parts" else 1.0


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    if case["call"] == "product":
        tokens, inputs, outputs = case["tokens"], case["inputs"], case["outputs"]
        weights = outputs * (inputs / 2 + 4 * math.ceil(inputs / case["blocksize"]))
        return {"bytes": weights + tokens * (inputs + outputs) * size + 4 * outputs * case["bias"], "flops": 2 * tokens * inputs * outputs}
    if case["call"] == "rotary":
        vectors = case["batch"] * case["tokens"] * (case["heads"] + case["kv_heads"])
        # forwards and backwards: read and written once each, and the positions
        return {"bytes": 4 * vectors * case["head_dim"] * size + 4 * case["tokens"] * case["batch"], "flops": 6 * vectors * case["dims"]}
    lengths, news = _counts(case)
    heads, group, dim = case["kv_heads"], case["group"], case["head_dim"]
    half = heads * (dim / 2 + 4 * math.ceil(dim / case["blocksize"]))              # a token's keys in the cache
    rows = sum(news)
    if case["call"] == "write":
        held = sum(min(a, n) for a, n in zip(news, lengths))
        # queries in and out; keys and values in, into the cache, and as they come back
        return {"bytes": 2 * rows * heads * group * dim * size + 2 * held * heads * dim * size * 2 + 2 * held * half * 2,
                "flops": 6 * rows * heads * (group + 1) * case["dims"] / 2}
    if case["call"] == "evict":
        kept = sum(min(n, case["keep"]) for n in lengths)
        return {"bytes": 4 * heads * sum(lengths) + kept * (2 * (2 * half + 4 * heads) + 2 * heads * dim * size), "flops": heads * sum(lengths)}
    tokens = pairs = 0
    for length, new in zip(lengths, news):
        if length:
            window = case["window"] or length + 1
            low = max(0, length - new + 1 - window)
            tokens += length - low + min(case["sinks"], low)
            seen = sum(min(p + 1, window + case["sinks"]) for p in range(length - new, length))
            pairs += seen
    return {"bytes": tokens * (half + 8 * heads) + rows * heads * group * dim * size, "flops": 2 * dim * heads * group * pairs}


def _generator(seed, *more):
    for n in more:
        seed = (seed * 1000003 + n + 1) % (2 ** 62)
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(seed, at, *shape):
    return torch.randn(*shape, device="cuda", generator=_generator(seed, at))


def _weights(case, seed):
    """Rows of ordinary numbers with a few inputs that matter more, as a trained matrix has them."""
    w = _randn(seed, 1, case["outputs"], case["inputs"]) / math.sqrt(case["inputs"])
    w[:, ::61] *= 4.0
    return w.to(DTYPES[case["dtype"]])


def _keys_and_values(case, seed, rows):
    """A few channels of the keys are much larger than the rest, as they are in a trained model, a few tokens larger in all of them, and one
    head's values are small."""
    heads, dim, dtype = case["kv_heads"], case["head_dim"], DTYPES[case["dtype"]]
    keys, values = _randn(seed, 1, rows, heads, dim), _randn(seed, 2, rows, heads, dim)
    keys[:, :, ::31] *= 6.0
    keys[::97] *= 1.5
    values[:, 0] *= 0.01
    return keys.to(dtype), values.to(dtype)


def _vectors(case, seed, at, *shape):
    return _randn(seed, at, *shape).to(DTYPES[case["dtype"]])


def _starts(news):
    return torch.tensor([0] + torch.tensor(news).cumsum(0).tolist(), dtype=torch.int32, device="cuda")


def _places(case, seed):
    """Pages of all sequences, in an order that has nothing to do with the sequences."""
    lengths, news = _counts(case)
    width = max(1, -(-max(lengths) // case["page_size"]))
    pages = case["batch"] * width
    order = torch.randperm(pages, device="cuda", generator=_generator(seed, 3)).to(torch.int32)
    return pages, order.view(case["batch"], width), torch.tensor(lengths, dtype=torch.int32, device="cuda"), None if case["new"] == 1 else _starts(news)


def _sums(case, seed, capacity):
    """Sums of weights as they come together: most tokens have hardly any, a few nearly all, and some none at all."""
    u = torch.rand(case["batch"], case["kv_heads"], capacity, device="cuda", generator=_generator(seed, 6))
    return torch.where(u < 0.1, torch.zeros_like(u), 5.0 * u ** 8)


def _framework(name):
    for path in (os.getcwd(), os.path.join(os.getcwd(), "low-bit-shampoo_amd")):
        if path not in sys.path:
            sys.path.insert(0, path)
    import importlib
    return importlib.import_module(name)


def prepare(case, seed):
    state = {"case": case}
    dtype = DTYPES[case["dtype"]]
    if case["call"] == "product":
        w = _weights(case, seed)
        state["x"] = _vectors(case, seed, 2, case["tokens"], case["inputs"])
        state["bias"] = _randn(seed, 3, case["outputs"]) if case["bias"] else None
        if own:
            state["weights"] = _framework("qtensor.linear").QTensorLinear(case["inputs"], case["outputs"], blocksize=case["blocksize"])
            state["weights"].quantize(w)
        else:
            state["codes"], state["scales"] = _encode(w, case["blocksize"])
        return state
    if case["dims"]:
        speed, magnitude = _frequencies(case)
        if own:
            state["rotary"] = _framework("qtensor.rotary").Rotary(case["dims"], frequencies=speed, magnitude=magnitude, interleaved=case["interleaved"])
        else:
            state["speed"], state["magnitude"] = torch.tensor(speed, dtype=torch.float64, device="cuda"), magnitude
    if case["call"] == "rotary":
        for at, name, heads in ((1, "q", case["heads"]), (2, "k", case["kv_heads"])):
            shape = (case["batch"], case["tokens"], heads, case["head_dim"])
            state[name], state["d" + name] = _vectors(case, seed, at, *shape).requires_grad_(own), _vectors(case, seed, at + 2, *shape)
        state["positions"] = case["first"] + torch.arange(case["tokens"], dtype=torch.int32, device="cuda")
        return state
    lengths, news = _counts(case)
    pages, state["table"], state["lengths"], state["starts"] = _places(case, seed)
    if own:
        cache = _framework("qtensor.cache").QTensorCache(pages, case["kv_heads"], case["head_dim"], page_size=case["page_size"], blocksize=case["blocksize"])
    else:
        cache = _PlainCache(case, pages)
    state["cache"] = cache
    if case["call"] == "write":
        state["k"], state["v"] = _keys_and_values(case, seed, sum(news))
        state["q"] = _vectors(case, seed, 4, sum(news), case["kv_heads"] * case["group"], case["head_dim"])
        state["positions"] = _moved(case) if case["moved"] else None
        return state
    keys, values = _keys_and_values(case, seed, sum(lengths))
    if own:
        cache.write(keys, values, state["table"], state["lengths"], _starts(lengths))
    else:
        cache.write(keys, values, cache.slots(state["table"], *_of_sequences(lengths, lengths)))
    capacity = state["table"].shape[1] * case["page_size"]
    if case["call"] == "weigh":
        state["q"] = _vectors(case, seed, 4, sum(news), case["kv_heads"] * case["group"], case["head_dim"])
        state["sums"] = torch.zeros(case["batch"], case["kv_heads"], capacity, device="cuda")
    else:
        state["sums"] = _sums(case, seed, capacity)
        kept = [min(n, case["keep"]) for n in lengths]
        state["kept"], state["rows"] = _starts(kept), sum(kept)
    return state


# ------------------------------------------------------------------------------------------------ the plain form
def _encode(x, blocksize):
    """(codes [.., ceil(dim / 2)], scales [.., segments]) of vectors."""
    dim = x.shape[-1]
    segments = -(-dim // blocksize)
    padded = torch.nn.functional.pad(x.float(), (0, segments * blocksize - dim)).unflatten(-1, (segments, blocksize))
    top = padded.abs().amax(-1)
    scales = top / torch.full_like(top, 6.0)
    held = padded / torch.where(scales > 0, scales, torch.ones_like(scales)).unsqueeze(-1)
    size = held.abs()
    codes = ((size > 0.25).to(torch.uint8) + (size >= 0.75) + (size > 1.25) + (size >= 1.75) + (size > 2.5) + (size >= 3.5)
             + (size > 5.0))
    codes = torch.where(held < 0, codes + 8, codes).flatten(-2)[..., :dim + dim % 2]
    if codes.shape[-1] % 2:
        codes = torch.nn.functional.pad(codes, (0, 1))
    return codes[..., 0::2] | (codes[..., 1::2] << 4), scales


def _decode(codes, scales, dim, blocksize):
    numbers = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    each = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)[..., :dim].int()
    return numbers[each] * scales.repeat_interleave(blocksize, -1)[..., :dim]


def _of_sequences(lengths, news):
    """(sequence, place) of the last `news` tokens of every sequence, packed; places below 0 where there are not so many."""
    b = torch.arange(len(news), device="cuda").repeat_interleave(torch.tensor(news, device="cuda"))
    end = torch.tensor(news, device="cuda").cumsum(0)
    return b, torch.arange(b.numel(), device="cuda") - end[b] + torch.tensor(lengths, device="cuda")[b]


def _moved(case):
    return (3 * _of_sequences(*_counts(case))[1] + 7).to(torch.int32)


class _PlainCache:
    def __init__(self, case, pages):
        self.case = case
        heads, dim = case["kv_heads"], case["head_dim"]
        slots = pages * case["page_size"]
        self.codes = torch.zeros(2, slots, heads, -(-dim // 2), dtype=torch.uint8, device="cuda")
        self.scales = torch.zeros(2, slots, heads, -(-dim // case["blocksize"]), device="cuda")

    def slots(self, table, b, places):
        size = self.case["page_size"]
        return table.long()[b, places // size] * size + places % size

    def write(self, keys, values, slots):
        for i, x in enumerate((keys, values)):
            codes, scales = _encode(x, self.case["blocksize"])
            self.codes[i, slots] = codes
            self.scales[i, slots] = scales

    def read(self, i, slots):
        return _decode(self.codes[i, slots], self.scales[i, slots], self.case["head_dim"], self.case["blocksize"])


def _turn(x, positions, state, back=False):
    """x [.., tokens, heads, head_dim]; positions [tokens]: the angles in 64 bits, the rest in 32."""
    case, dims = state["case"], state["case"]["dims"]
    angle = positions.double()[:, None, None] * state["speed"]
    c, s = ((state["magnitude"] * f(angle)).float() for f in (torch.cos, torch.sin))
    x = x.float()
    turned, rest = x[..., :dims], x[..., dims:]
    a, b = (turned[..., 0::2], turned[..., 1::2]) if case["interleaved"] else (turned[..., :dims // 2], turned[..., dims // 2:])
    if back:
        s = -s
    first, second = a * c - b * s, b * c + a * s
    both = torch.stack((first, second), -1).flatten(-2) if case["interleaved"] else torch.cat((first, second), -1)
    return torch.cat((both, rest), -1).to(DTYPES[case["dtype"]])


def _plain_write(state):
    case, cache = state["case"], state["cache"]
    lengths, news = _counts(case)
    b, places = _of_sequences(lengths, news)
    there = places >= 0
    positions = places if state["positions"] is None else state["positions"]
    q, k = (_turn(state[n], positions, state) * there[:, None, None] for n in ("q", "k"))
    rows = torch.arange(b.numel(), device="cuda") if min(lengths) else torch.nonzero(there)[:, 0]
    slots = cache.slots(state["table"], b[rows], places[rows])
    cache.write(k[rows], state["v"][rows], slots)
    out = [torch.zeros_like(k), torch.zeros_like(k)]
    out[0][rows], out[1][rows] = (cache.read(i, slots).to(k.dtype) for i in range(2))
    return q, out[0], out[1]


def _plain_weigh(state):
    case, cache = state["case"], state["cache"]
    heads, group, dim, window, sinks = case["kv_heads"], case["group"], case["head_dim"], case["window"], case["sinks"]
    lengths, news = _counts(case)
    b, places = _of_sequences(lengths, news)
    most, capacity = max(news), state["sums"].shape[-1]
    nth = torch.arange(b.numel(), device="cuda") - state["starts"].long()[b] if state["starts"] is not None else torch.zeros_like(b)
    # every sequence as long as the longest, with as many queries as the one that has most
    at = torch.full((case["batch"], most), -1, device="cuda")
    at[b, nth] = places
    q = torch.zeros(case["batch"], most, heads, group, dim, device="cuda")
    q[b, nth] = state["q"].float().unflatten(1, (heads, group))
    t = torch.arange(capacity, device="cuda")
    keys = cache.read(0, (state["table"].long()[:, t // case["page_size"]] * case["page_size"] + t % case["page_size"]).flatten())
    keys = keys.view(case["batch"], capacity, heads, dim).permute(0, 2, 3, 1).contiguous()
    scores = torch.matmul(q.permute(0, 2, 1, 3, 4).reshape(case["batch"], heads, most * group, dim), keys) * (1.0 / math.sqrt(dim))
    hidden = t > at[:, :, None]
    if window:
        hidden |= (t <= at[:, :, None] - window) & (t >= sinks)
    scores = scores.view(case["batch"], heads, most, group, capacity).masked_fill(hidden[:, None, :, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - torch.where(top > -math.inf, top, torch.zeros_like(top)))
    weights = weights / weights.sum(-1, keepdim=True).clamp(min=1e-30)
    state["sums"] += weights.sum((2, 3))
    return state["sums"]


def _plain_evict(state):
    case, cache, sums = state["case"], state["cache"], state["sums"]
    t = torch.arange(sums.shape[-1], device="cuda")
    length = state["lengths"].long()[:, None, None]
    kept_anyhow = (t < case["sinks"]) | (t >= length - case["recent"])
    order = torch.where(t >= length, -math.inf, torch.where(kept_anyhow, math.inf, sums))
    chosen = torch.sort(order, dim=-1, descending=True, stable=True).indices[..., :case["keep"]]
    count = length.clamp(max=case["keep"])
    nth = torch.arange(chosen.shape[-1], device="cuda")
    chosen = torch.where(nth < count, chosen, sums.shape[-1]).sort(-1).values
    b, h, nth = torch.nonzero((nth < count).expand_as(chosen), as_tuple=True)
    source = chosen[b, h, nth]
    to, come = cache.slots(state["table"], b, nth), cache.slots(state["table"], b, source)
    cache.codes[:, to, h] = cache.codes[:, come, h]
    cache.scales[:, to, h] = cache.scales[:, come, h]
    sums[b, h, nth] = sums[b, h, source]
    lengths = state["lengths"].clamp(max=case["keep"])
    slots = cache.slots(state["table"], *_of_sequences(*[[min(n, case["keep"]) for n in _counts(case)[0]]] * 2))
    return (*(cache.read(i, slots).to(DTYPES[case["dtype"]]) for i in range(2)), sums, lengths)


def run(state):
    case = state["case"]
    if own:
        return _own(state)
    if case["call"] == "product":
        w = _decode(state["codes"], state["scales"], case["inputs"], case["blocksize"])
        out = torch.matmul(state["x"].float(), w.T)
        return (out + state["bias"] if case["bias"] else out).to(DTYPES[case["dtype"]])
    if case["call"] == "rotary":
        return tuple(_turn(state[n], state["positions"], state, n[0] == "d") for n in ("q", "k", "dq", "dk"))
    return {"write": _plain_write, "weigh": _plain_weigh, "evict": _plain_evict}[case["call"]](state)


# ------------------------------------------------------------------------------------------------ the framework's calls
def _own(state):
    case = state["case"]
    if case["call"] == "product":
        return state["weights"].product(state["x"], state["bias"])
    if case["call"] == "rotary":
        q, k = state["rotary"].turn(state["q"], state["k"], state["positions"])
        dq, dk = torch.autograd.grad((q, k), (state["q"], state["k"]), (state["dq"], state["dk"]))
        return q.detach(), k.detach(), dq, dk
    cache, where = state["cache"], (state["table"], state["lengths"], state["starts"])
    dtype = DTYPES[case["dtype"]]
    if case["call"] == "write":
        q = cache.write_turned(state["rotary"], state["q"], state["k"], state["v"], *where, positions=state["positions"])
        return (q, *cache.read(*where, tokens=state["q"].shape[0], dtype=dtype))
    if case["call"] == "weigh":
        return cache.weigh(state["sums"], state["q"], *where, window=case["window"] or None, sinks=case["sinks"])
    lengths = cache.evict(state["sums"], state["table"], state["lengths"], case["keep"], recent=case["recent"], sinks=case["sinks"])
    return (*cache.read(state["table"], lengths, state["kept"], tokens=state["rows"], dtype=dtype), state["sums"], lengths)


# ------------------------------------------------------------------------------------------------ in 64 bits
def _held(x, blocksize):
    """What 4 bits stand for: scales and quotients are numbers of 32 bits by definition, the rest is exact."""
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for first in range(0, x.shape[-1], blocksize):
        piece = x[..., first:first + blocksize].double()
        scale = (piece.abs().amax(-1, keepdim=True) / 6.0).float().double()
        part = torch.where(scale > 0, piece / scale, torch.zeros_like(piece)).float().double()
        size = part.abs().clamp(max=6.0)
        step = torch.where(size < 2, 0.5, torch.where(size < 4, 1.0, 2.0)).double()
        out[..., first:first + blocksize] = torch.round(size / step) * step * part.sign() * scale
    return out


def _turned(case, x, positions, sign=1.0):
    """By complex numbers, cosines and sines as the fp32 numbers they are by definition."""
    speed, magnitude = _frequencies(case)
    angle = positions.to("cuda", torch.float64)[:, None, None] * torch.tensor(speed, dtype=torch.float64, device="cuda")
    by = torch.complex((magnitude * angle.cos()).float().double(), sign * (magnitude * angle.sin()).float().double())
    out, n = x.double().clone(), case["dims"]
    at = (slice(0, n, 2), slice(1, n, 2)) if case["interleaved"] else (slice(0, n // 2), slice(n // 2, n))
    z = torch.complex(out[..., at[0]], out[..., at[1]]) * by
    out[..., at[0]], out[..., at[1]] = z.real, z.imag
    return out


def exact(case, seed):
    if case["call"] == "product":
        out = _vectors(case, seed, 2, case["tokens"], case["inputs"]).double() @ _held(_weights(case, seed), case["blocksize"]).T
        return out + _randn(seed, 3, case["outputs"]).double() if case["bias"] else out
    if case["call"] == "rotary":
        positions = case["first"] + torch.arange(case["tokens"])
        shapes = [(case["batch"], case["tokens"], n, case["head_dim"]) for n in (case["heads"], case["kv_heads"])]
        return tuple(_turned(case, _vectors(case, seed, at, *shapes[(at - 1) % 2]), positions, 1.0 if at < 3 else -1.0) for at in (1, 2, 3, 4))
    lengths, news = _counts(case)
    heads, group, dim = case["kv_heads"], case["group"], case["head_dim"]
    if case["call"] == "write":
        keys, values = _keys_and_values(case, seed, sum(news))
        q = _vectors(case, seed, 4, sum(news), heads * group, dim)
        places = torch.tensor([n - a + i for n, a in zip(lengths, news) for i in range(a)], device="cuda")
        positions = 3 * places + 7 if case["moved"] else places
        there = (places >= 0)[:, None, None]
        turned = _turned(case, keys, positions).float().to(keys.dtype)      # (what is encoded has the type of the keys)
        out = (_turned(case, q, positions), _held(turned, case["blocksize"]), _held(values, case["blocksize"]))
        # (a key that lies next to a border of two numbers may go to either: those are compared with the plain form's alone)
        return out[0] * there, None, out[2] * there
    keys, values = _keys_and_values(case, seed, sum(lengths))
    width = max(1, -(-max(lengths) // case["page_size"])) * case["page_size"]
    first = [sum(lengths[:b]) for b in range(len(lengths))]
    if case["call"] == "evict":
        sums = _sums(case, seed, width)
        got = [torch.zeros(0, heads, dim, dtype=torch.float64, device="cuda")] * 2
        for b, n in enumerate(lengths):
            kept = [i for i in range(n) if i < case["sinks"] or i >= n - case["recent"]]
            rows, count = [], min(n, case["keep"])
            for h in range(heads):
                other = sums[b, h, :n].double().clone()
                other[kept] = math.inf
                at = torch.argsort(other, descending=True, stable=True)[:count].sort().values
                rows.append(at + first[b])
                sums[b, h, :count] = sums[b, h][at].clone()
            if count:
                rows = torch.stack(rows, 1)[:, :, None].expand(-1, -1, dim)
                got = [torch.cat((g, _held(x.gather(0, rows), case["blocksize"]))) for g, x in zip(got, (keys, values))]
        return (*got, sums.double(), None)
    q = _vectors(case, seed, 4, sum(news), heads * group, dim).double()
    out = torch.zeros(case["batch"], heads, width, dtype=torch.float64, device="cuda")
    at = 0
    for b, (n, new) in enumerate(zip(lengths, news)):
        if n:
            held = _held(keys[first[b]:first[b] + n], case["blocksize"])
            i, j = torch.arange(n - new, n, device="cuda")[:, None], torch.arange(n, device="cuda")[None, :]
            see = j <= i
            if case["window"]:
                see = see & ((i - j < case["window"]) | (j < case["sinks"]))
            for h in range(heads * group):
                s = (q[at:at + new, h] @ held[:, h // group].T) / math.sqrt(dim)
                out[b, h // group, :n] += torch.softmax(s.masked_fill(~see, -math.inf), -1).sum(0)
        at += new
    return out
