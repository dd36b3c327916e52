"""How many tokens the example that generates with its attention cache in 4 bits returns, and what it refuses."""
import importlib.util
from pathlib import Path

import pytest
import torch

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
    return example.Model().cuda()


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("new", [1, 2, 3, 7])
def test_as_many_tokens_as_asked_for(example, model, new, captured):
    prompts = [torch.arange(n) % example.VOCABULARY for n in (5, 1, 30)]
    whole = example.Server(model, 3).generate(prompts, 9, captured=False)
    got = example.Server(model, 3).generate(prompts, new, captured=captured)
    assert got.shape == (3, new) and torch.equal(got, whole[:, :new])


def test_places_up_to_the_last_one_and_refusals(example, model):
    prompt = torch.zeros(example.LONGEST - 2, dtype=torch.long)
    server = example.Server(model, 2)
    assert server.generate([prompt, prompt[:3]], 3).shape == (2, 3) and int(server.lengths.max()) == example.LONGEST
    for prompts, new in (([prompt, prompt[:3]], 4), ([prompt, prompt[:0]], 1), ([prompt, prompt], 0)):
        with pytest.raises(ValueError):
            example.Server(model, 2).generate(prompts, new)
