"""The example that trains a small model and generates with its attention cache in 4 bits: every attention it runs against the
definition, over what the cache holds at that moment; replayed steps against steps run one by one."""
import importlib.util
from pathlib import Path

import pytest
import torch

from oracle import cache_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    import qtensor.functional as F
    assert torch.cuda.is_available() and F.lib is not None
    spec = importlib.util.spec_from_file_location("generate_example", Path(__file__).resolve().parents[1] / "examples" / "generate.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.fixture(scope="module")
def model(example):
    torch.manual_seed(0)
    model = example.Model().cuda()
    first, last = example.train(model, 30)
    assert last < first
    return model


def prompts(example):
    x = example.text(5, example.LONGEST, torch.Generator(device="cuda").manual_seed(1)).cpu()
    return [x[b, :n] for b, n in enumerate((1, 40, 17, 100, 2))]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_every_attention_of_prompts_and_steps(example, model, dtype):
    server = example.Server(model, 5, dtype)
    seen = []
    for cache in server.caches:
        def checked(q, table, lengths, starts=None, cache=cache, real=cache.attend):
            out = real(q, table, lengths, starts)
            counts = lengths.tolist()
            ends = torch.tensor([sum(counts[:b]) for b in range(6)], dtype=torch.int32).cuda()
            keys, values = (t.cpu().double() for t in cache.read(table, lengths, ends, tokens=sum(counts)))
            at = list(range(6)) if starts is None else starts.tolist()
            for b, n in enumerate(counts):
                rows, kept, new = slice(at[b], at[b + 1]), slice(int(ends[b]), int(ends[b + 1])), at[b + 1] - at[b]
                want, size, spread = R.attend(q[rows].cpu(), range(n - new, n), keys[kept], values[kept], cache.head_dim ** -0.5)
                limit = R.bounds(dtype, want, size, spread, cache.head_dim)
                if dtype == torch.bfloat16:         # (many queries: three roundings of 2^-12 in a product)
                    limit = limit + size * 6 * 2.0 ** -12 * spread
                assert ((out[rows].cpu().double() - want).abs() <= limit).all()
            seen.append(q.shape[0])
            return out
        cache.attend = checked
    token = server.prompts(prompts(example)).argmax(-1)
    for _ in range(3):
        token = server.step(token).argmax(-1)
    assert seen == [160, 160] + [5] * 6 and server.lengths.tolist() == [4, 43, 20, 103, 5]


def test_replayed_steps_are_the_steps(example, model):
    runs = [example.Server(model, 5).generate(prompts(example), 20, captured=c) for c in (False, True, True)]
    assert runs[0].shape == (5, 20) and torch.equal(runs[0], runs[1]) and torch.equal(runs[0], runs[2])
