"""A layer of a model as it generates, everything of it held in 4 bits: projections (qtensor.linear), rotary positions on the way into the
cache, attention, weights, eviction (qtensor.cache, qtensor.rotary).  Every stage is held to its definition on what the stage before gave."""
import pytest
import torch

from oracle import cache_ref as C
from oracle import evict_ref as E
from oracle import linear_ref as L
from oracle import rotary_ref as R

pytestmark = pytest.mark.gpu

WIDTH, HEADS, KV, DIM, KEEP = 256, 8, 2, 64, 40


class Layer:
    def __init__(self, batch, room, dtype, seed=0):
        from qtensor.cache import QTensorCache
        from qtensor.linear import QTensorLinear
        from qtensor.rotary import Rotary
        g = torch.Generator().manual_seed(seed)
        self.dtype = dtype
        self.w = {"in": torch.randn((HEADS + 2 * KV) * DIM, WIDTH, generator=g) / 16, "out": torch.randn(WIDTH, HEADS * DIM, generator=g) / 22}
        self.held = {n: QTensorLinear(w.shape[1], w.shape[0]).quantize(w.to(dtype).cuda()) for n, w in self.w.items()}
        self.rotary = Rotary(DIM, base=1000.0)
        self.cache = QTensorCache(batch * room, KV, DIM, page_size=16)
        self.table = torch.randperm(batch * room, generator=g).view(batch, room).to(torch.int32).cuda()
        self.totals = self.cache.totals(self.table)

    def __call__(self, x, lengths, starts, positions):
        """(result, what the stages gave)"""
        mixed = self.held["in"].product(x).unflatten(-1, (-1, DIM))
        q, k, v = mixed.split((HEADS, KV, KV), 1)                       # (slices of one tensor)
        turned = self.cache.write_turned(self.rotary, q, k, v, self.table, lengths, starts, positions=positions)
        out = self.cache.attend(turned, self.table, lengths, starts)
        self.cache.weigh(self.totals, turned, self.table, lengths, starts)
        return self.held["out"].product(out.flatten(1)), (mixed, turned, out)


def within(got, want, limit):
    assert bool(((got.double().cpu() - want).abs() <= limit).all()), float(((got.double().cpu() - want).abs() / limit.clamp(min=1e-300)).max())


def check(layer, x, stages, y, lengths, news, positions, held_k, held_v):
    """held_k, held_v: per sequence, what its cache stood for before; returns them as they are now."""
    mixed, turned, out = stages
    dtype = layer.dtype
    for name, given, got in (("in", x.cpu(), mixed.flatten(1)), ("out", out.flatten(1).cpu(), y)):
        want, size = L.product(given, layer.w[name].to(dtype), 64)
        within(got, want, L.bounds(dtype, want, size, given.shape[1], 64))
    want, size = R.turned(mixed[:, :HEADS].cpu(), positions, layer.rotary.frequencies.cpu(), DIM)
    within(turned, want, R.bounds(dtype, want, size))
    keys, _ = layer.rotary.turn(mixed[:, HEADS:HEADS + KV], None, positions.cuda())
    at = 0
    for b, (n, new) in enumerate(zip(lengths, news)):
        held_k[b] = torch.cat([held_k[b], C.held(keys[at:at + new].cpu(), 64)])
        held_v[b] = torch.cat([held_v[b], C.held(mixed[at:at + new, HEADS + KV:].cpu(), 64)])
        want, size, spread = C.attend(turned[at:at + new].cpu(), range(n - new, n), held_k[b], held_v[b], 0.125)
        within(out[at:at + new], want, C.bounds(dtype, want, size, spread, DIM))
        at += new
    return held_k, held_v


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_prompts_steps_and_eviction(dtype):
    batch, room = 3, 6
    prompts = [70, 33, 1]
    layer = Layer(batch, room, dtype)
    g = torch.Generator().manual_seed(5)
    lengths = torch.tensor(prompts, dtype=torch.int32).cuda()
    starts = torch.tensor([0, 70, 103, 104], dtype=torch.int32).cuda()
    x = torch.randn(104, WIDTH, generator=g).to(dtype).cuda()
    positions = torch.cat([torch.arange(n) for n in prompts])
    y, stages = layer(x, lengths, starts, None)
    none = torch.zeros(0, KV, DIM, dtype=torch.float64)
    held_k, held_v = check(layer, x, stages, y, prompts, prompts, positions, [none] * 3, [none] * 3)
    sums = [E.weigh(stages[1][a:a + n].cpu(), range(n), held_k[b], 0.125) for b, (a, n) in enumerate(((0, 70), (70, 33), (103, 1)))]
    for b, (want, spread) in enumerate(sums):
        within(layer.totals[b, :, :prompts[b]], want, E.bound(DIM, prompts[b] * HEADS // KV, want, spread))

    # cut down: the tokens that stay by the totals that the GPU has
    totals = layer.totals.cpu()
    kept = [[E.evict(totals[b, h].tolist(), n, KEEP, recent=8, sinks=2)[0] for h in range(KV)] for b, n in enumerate(prompts)]
    lengths.copy_(layer.cache.evict(layer.totals, layer.table, lengths, KEEP, recent=8, sinks=2))
    assert lengths.tolist() == [40, 33, 1]
    for b in range(batch):
        held_k[b], held_v[b] = (torch.stack([t[b][kept[b][h], h] for h in range(KV)], 1) for t in (held_k, held_v))
        layer.totals[b, :, int(lengths[b]):] = 0

    # steps, captured: every one a token of each sequence, at its own position
    at = torch.tensor(prompts, device="cuda")
    given = torch.randn(batch, WIDTH, generator=g).to(dtype).cuda()
    graph = torch.cuda.CUDAGraph()
    lengths += 1
    state = [t.clone() for t in (layer.cache.codes, layer.cache.scales, layer.totals)]
    layer(given, lengths, None, at)                     # (once before it is captured, and taken back)
    for t, kept_state in zip((layer.cache.codes, layer.cache.scales, layer.totals), state):
        t.copy_(kept_state)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        y, stages = layer(given, lengths, None, at)
    for step in range(3):
        if step:
            lengths += 1
            at += 1
            given.copy_(torch.randn(batch, WIDTH, generator=g).to(dtype))
        before = layer.totals.clone()
        graph.replay()
        torch.cuda.synchronize()
        held_k, held_v = check(layer, given, stages, y, lengths.tolist(), [1] * batch, at.cpu(), held_k, held_v)
        for b, n in enumerate(lengths.tolist()):
            want, spread = E.weigh(stages[1][b:b + 1].cpu(), [n - 1], held_k[b], 0.125)
            rise = before[b, :, :n].double().cpu() + want
            within(layer.totals[b, :, :n], rise, E.bound(DIM, HEADS // KV, want, spread) + 2.0 ** -23 * rise)
