"""A small language model from training to answering: low-bit Shampoo trains it, then it generates with its attention cache held
in 4 bits (qtensor.cache).

    python examples/generate.py [--steps 150] [--new 48]

The text is synthetic: a random passage of PERIOD tokens, repeated; a model that has learnt it looks back one period.  Training runs in
fp32 over whole sequences.  Serving takes prompts of different lengths in one call (every layer writes its keys and values, then
attends), then one token of each sequence at a time, a step that is captured in a graph and replayed: what changes from step to step
(tokens, lengths) lives on the GPU."""
import argparse
import math
import sys
import time
from pathlib import Path

import torch
from torch import nn

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "low-bit-shampoo_amd"))
from optimizers.shampoo1 import ShampooAdamW  # noqa: E402
from qtensor.cache import QTensorCache  # noqa: E402

VOCABULARY, PERIOD, LONGEST = 32, 12, 128


class Layer(nn.Module):
    def __init__(self, width, heads, kv_heads, head_dim):
        super().__init__()
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        self.before, self.between = nn.LayerNorm(width), nn.LayerNorm(width)
        self.project = nn.Linear(width, (heads + 2 * kv_heads) * head_dim, bias=False)
        self.back = nn.Linear(heads * head_dim, width, bias=False)
        self.up, self.down = nn.Linear(width, 4 * width), nn.Linear(4 * width, width)

    def forward(self, x, attention):
        """x [.., width]; attention: (q, k, v) -> result, each [.., heads, head_dim]."""
        parts = self.project(self.before(x)).unflatten(-1, (-1, self.head_dim))
        q, k, v = parts.split((self.heads, self.kv_heads, self.kv_heads), -2)
        x = x + self.back(attention(q, k, v).flatten(-2))
        return x + self.down(torch.nn.functional.gelu(self.up(self.between(x))))


class Model(nn.Module):
    def __init__(self, width=128, layers=2, heads=4, kv_heads=2, head_dim=64):
        super().__init__()
        self.tokens, self.places = nn.Embedding(VOCABULARY, width), nn.Embedding(LONGEST, width)
        self.layers = nn.ModuleList(Layer(width, heads, kv_heads, head_dim) for _ in range(layers))
        self.last, self.head = nn.LayerNorm(width), nn.Linear(width, VOCABULARY, bias=False)

    def forward(self, tokens, positions, attentions):
        x = self.tokens(tokens) + self.places(positions)
        for layer, attention in zip(self.layers, attentions):
            x = layer(x, attention)
        return self.head(self.last(x))


def whole(q, k, v):
    """Attention over whole sequences [batch, tokens, heads, head_dim], for training."""
    group = q.shape[2] // k.shape[2]
    q, k, v = (t.repeat_interleave(n, 2).transpose(1, 2) for t, n in ((q, 1), (k, group), (v, group)))
    scores = q @ k.transpose(-1, -2).contiguous() / math.sqrt(q.shape[-1])
    ahead = torch.ones(scores.shape[-2:], dtype=torch.bool, device=q.device).triu(1)
    return (torch.softmax(scores.masked_fill(ahead, -math.inf), -1) @ v.contiguous()).transpose(1, 2)


def text(batch, length, generator):
    passage = torch.randint(VOCABULARY, (batch, PERIOD), generator=generator, device=generator.device)
    return passage.repeat(1, -(-length // PERIOD))[:, :length]


def train(model, steps, batch=64, length=LONGEST, seed=0):
    """Losses of the first and the last step."""
    generator = torch.Generator(device="cuda").manual_seed(seed)
    optimizer = ShampooAdamW(model.parameters(), lr=2e-3, prec_bits=4, start_prec_step=1, stat_compute_steps=10, prec_compute_steps=50, fused=True)
    positions = torch.arange(length - 1, device="cuda")
    losses = []
    for _ in range(steps):
        x = text(batch, length, generator)
        logits = model(x[:, :-1], positions, [whole] * len(model.layers))
        loss = torch.nn.functional.cross_entropy(logits[:, PERIOD:].flatten(0, 1), x[:, PERIOD + 1:].flatten())
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
    return float(losses[0]), float(losses[-1])


class Server:
    """Generates for a batch of sequences: a cache per layer, pages handed out in front."""

    def __init__(self, model, batch, dtype=torch.bfloat16, page_size=16):
        first = model.layers[0]
        width = -(-LONGEST // page_size)
        self.model, self.dtype = model, dtype
        self.caches = [QTensorCache(batch * width, first.kv_heads, first.head_dim, page_size=page_size) for _ in model.layers]
        self.table = torch.arange(batch * width, dtype=torch.int32, device="cuda").view(batch, width)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device="cuda")

    def _run(self, tokens, positions, starts):
        def through(cache):
            def attention(q, k, v):
                q, k, v = (t.to(self.dtype) for t in (q, k, v))
                cache.write(k, v, self.table, self.lengths, starts)
                return cache.attend(q, self.table, self.lengths, starts).float()
            return attention
        return self.model(tokens, positions, [through(c) for c in self.caches])

    @torch.no_grad()
    def prompts(self, sequences):
        """Logits of the token behind every prompt (lists of tokens), all prompts in one call."""
        counts = torch.tensor([len(s) for s in sequences])
        starts = torch.cat([torch.zeros(1, dtype=torch.long), counts.cumsum(0)])
        positions = torch.cat([torch.arange(n) for n in counts]).cuda()
        self.lengths.copy_(counts)
        logits = self._run(torch.cat(sequences).cuda(), positions, starts.to(torch.int32).cuda())
        return logits[starts[1:].cuda() - 1]

    @torch.no_grad()
    def step(self, tokens):
        """Logits behind one more token of each sequence."""
        self.lengths += 1
        return self._run(tokens, self.lengths.long() - 1, None)

    @torch.no_grad()
    def generate(self, sequences, new, captured=True):
        """`new` tokens behind each prompt, the likeliest each time: [batch, new]."""
        shortest, longest = min(len(s) for s in sequences), max(len(s) for s in sequences)
        if new < 1 or shortest < 1 or longest + new - 1 > LONGEST:
            raise ValueError(f"{new} tokens behind prompts of {shortest} to {longest}: at least one of each, and {LONGEST} with all but the last new one")
        token = self.prompts(sequences).argmax(-1)
        out = [token.clone()]
        if new > 1:
            token = self.step(token).argmax(-1)
            out.append(token.clone())
        if captured and new > 2:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):           # (recorded, not run)
                token.copy_(self.step(token).argmax(-1))
        for _ in range(new - 2):
            if captured:
                graph.replay()
            else:
                token.copy_(self.step(token).argmax(-1))
            out.append(token.clone())
        return torch.stack(out, 1)


def main():
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--steps", type=int, default=150)
    parser.add_argument("--new", type=int, default=48)
    arguments = parser.parse_args()
    torch.manual_seed(0)
    model = Model().cuda()
    first, last = train(model, arguments.steps)
    print(f"loss {first:.3f} -> {last:.3f} in {arguments.steps} steps")
    x = text(8, LONGEST, torch.Generator(device="cuda").manual_seed(1))
    counts = [24 + 5 * b for b in range(8)]
    new = min(arguments.new, LONGEST - max(counts))
    server = Server(model, 8)
    begin = time.perf_counter()
    got = server.generate([x[b, :n].cpu() for b, n in enumerate(counts)], new)
    torch.cuda.synchronize()
    took = time.perf_counter() - begin
    want = torch.stack([x[b, n:n + new] for b, n in enumerate(counts)])
    held = server.caches[0].codes.numel() + 4 * server.caches[0].scales.numel()
    print(f"{new} tokens behind each of 8 prompts in {1e3 * took:.0f} ms (the graph's capture included), {float((got == want).float().mean()):.1%} as "
          f"the text goes on; {held / server.caches[0].scales.numel() / 64 * 8:.2f} bits per element of the cache")


if __name__ == "__main__":
    main()
