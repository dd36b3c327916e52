"""The example that generates, with its projections held in 4 bits too: every product it runs against the definition, replayed steps against
steps run one by one."""
import importlib.util
from pathlib import Path

import pytest
import torch

from oracle import linear_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("generate_example", Path(__file__).resolve().parents[1] / "examples" / "generate.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_every_product_of_prompts_and_steps(example):
    torch.manual_seed(0)
    model = example.Model().cuda()
    server = example.Server(model, 3, held=True)
    x = example.text(3, example.LONGEST, torch.Generator(device="cuda").manual_seed(1)).cpu()
    prompts = [x[b, :n] for b, n in enumerate((1, 60, 17))]
    linear = [m for m in model.modules() if isinstance(m, torch.nn.Linear)]
    held = [m for m in server.model.modules() if isinstance(m, example.Held)]
    assert len(held) == len(linear) == 9 and not any(isinstance(m, torch.nn.Linear) for m in server.model.modules())
    seen = []
    for was, now in zip(linear, held):
        def checked(given, bias, was=was, real=now.weights.product):
            got = real(given, bias)
            want, size = R.product(given.flatten(0, -2).cpu(), was.weight.detach().cpu(), 64, None if was.bias is None else was.bias.detach().cpu())
            limit = R.bounds(given.dtype, want, size, was.in_features, 64)
            assert bool(((got.flatten(0, -2).double().cpu() - want).abs() <= limit).all())
            seen.append(got.shape[0])
            return got
        now.weights.product = checked
    token = server.prompts(prompts).argmax(-1)
    server.step(token)
    assert seen == [78] * 9 + [3] * 9


def test_replayed_steps_are_the_steps(example):
    torch.manual_seed(0)
    model = example.Model().cuda()
    x = example.text(3, example.LONGEST, torch.Generator(device="cuda").manual_seed(1)).cpu()
    prompts = [x[b, :n] for b, n in enumerate((1, 60, 17))]
    runs = [example.Server(model, 3, held=True).generate(prompts, 12, captured=c) for c in (False, True)]
    assert runs[0].shape == (3, 12) and torch.equal(runs[0], runs[1])
