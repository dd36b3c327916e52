"""The 4-bit attention cache where no GPU is involved: its construction, its refusal to compute elsewhere, the oracle's own pins."""
import math

import pytest
import torch

from oracle import cache_ref as R


def test_construction_and_its_refusals():
    from qtensor.cache import QTensorCache
    c = QTensorCache(3, 2, 80, page_size=32, blocksize=64, device="cpu")
    assert c.codes.shape == (2, 3, 2, 32, 48) and c.scales.shape == (2, 3, 2, 2, 32) and c.codes.dtype == torch.uint8
    for bad in (dict(blocksize=32), dict(page_size=8), dict(page_size=48), dict(page_size=8192), dict(head_dim=0), dict(head_dim=257),
                dict(kv_heads=0), dict(pages=0)):
        args = dict(pages=3, kv_heads=2, head_dim=80, device="cpu")
        args.update(bad)
        with pytest.raises(ValueError):
            QTensorCache(**args)


def test_no_cpu_fallback():
    from qtensor.cache import QTensorCache
    c = QTensorCache(3, 2, 64, device="cpu")
    x = torch.zeros(1, 2, 64)
    table, lengths = torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    for call in (lambda: c.write(x, x, table, lengths), lambda: c.read(table, lengths), lambda: c.attend(x, table, lengths)):
        with pytest.raises(RuntimeError):
            call()


def test_the_oracle_holds_the_nearest_numbers():
    """Brute force over the sixteen numbers; ties go to the code without a last bit."""
    numbers = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
    x = torch.randn(200, 64, generator=torch.Generator().manual_seed(0))
    x[:8, 0] = 6.0
    x[:8, 1:8] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    x[:8] = x[:8].clamp(-6, 6)
    got = R.held(x, 64)
    scale = (x.double().abs().amax(-1, keepdim=True) / 6).float().double()
    part = (x.double() / scale).float().double()
    off = (part.abs().unsqueeze(-1) - numbers).abs()
    best = off.min(-1, keepdim=True).values
    for i in range(200):
        for d in range(64):
            near = [c for c in range(8) if off[i, d, c] == best[i, d, 0]]
            want = numbers[[c for c in near if c % 2 == 0][0] if len(near) > 1 else near[0]] * scale[i, 0]
            assert got[i, d].abs() == want
    assert torch.equal(got.sign() * (got != 0), x.double().sign() * (got != 0))
    assert torch.isnan(R.held(torch.tensor([[math.nan, 1.0]]), 64)).all()


def test_the_oracle_attends_to_what_is_seen():
    assert R.seen(5, 8).tolist() == [True] * 6 + [False] * 2
    assert R.seen(5, 8, 2, 1).tolist() == [True, False, False, False, True, True, False, False]
    k = torch.zeros(4, 1, 2, dtype=torch.float64)
    v = torch.arange(8.0, dtype=torch.float64).view(4, 1, 2)
    out, size, _ = R.attend(torch.ones(2, 2, 2), [-1, 3], k, v, 1.0, 2, 1)
    assert not out[0].any() and torch.allclose(out[1, 0], (v[0, 0] + v[2, 0] + v[3, 0]) / 3)
    assert torch.allclose(size[1, 1], torch.tensor([(1.0 + 5.0 + 7.0) / 3], dtype=torch.float64))


def test_tensors_that_are_not_the_caches_are_refused():
    """Kernels go by the cache's numbers: a tensor of another size in the place of its own would be read past its end."""
    from qtensor.cache import QTensorCache

    def cache():
        return QTensorCache(3, 2, 80, page_size=32, blocksize=64, device="cpu")
    assert cache()._ref().pages == 3
    for name in ("codes", "scales"):
        for change in (lambda t: t[:, :2], lambda t: t[:, :2].contiguous(), lambda t: t.double(), lambda t: t[..., ::2], lambda t: t.flatten(),
                       lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)):
            c = cache()
            setattr(c, name, change(getattr(c, name)))
            with pytest.raises(ValueError):
                c._ref()
    c = cache()
    c.pages = 4
    with pytest.raises(ValueError):
        c._ref()
