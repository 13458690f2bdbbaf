"""Dropout against its generator in Python's whole numbers, and its refusals, on the CPU."""
import math

import pytest
import torch

import bit_reproducible_training_amd as rg
from test_attention import philox


def kept(n, p, seed):
    out = []
    for group in range((n + 3) // 4):
        out += [w >= int(p * 2 ** 32) for w in philox(group % 2 ** 32, group >> 32, 0, 0, seed % 2 ** 64)]
    return torch.tensor(out[:n], dtype=torch.bool)


def test_the_generator_is_philox():
    """The generator's published answers for counters and keys of zeros and of ones."""
    assert philox(0, 0, 0, 0, 0) == (0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8)
    ones = 2 ** 32 - 1
    assert philox(ones, ones, ones, ones, 2 ** 64 - 1) == (0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd)


@pytest.mark.parametrize("shape,p,seed", [((7,), 0.5, 0), ((33, 5), 0.1, 2 ** 63 + 5), ((1,), 0.9, -1), ((2, 3, 1001), 0.25, 77),
                                          ((0, 4), 0.5, 1), ((5,), 0.0, 3)])
def test_values_and_gradient(shape, p, seed):
    x, dy = torch.randn(shape), torch.randn(shape)
    leaf = x.clone().requires_grad_()
    y = rg.dropout(leaf, p, seed=seed)
    mask = kept(x.numel(), p, seed).view(shape)
    factor = torch.tensor(1.0 / (1.0 - p))
    assert torch.equal(y, torch.where(mask, x * factor, 0.0))
    assert torch.equal(torch.autograd.grad(y, leaf, dy)[0], torch.where(mask, dy * factor, 0.0))
    assert torch.equal(rg.dropout(x, p, seed=torch.tensor([seed % 2 ** 63])), rg.dropout(x, p, seed=seed % 2 ** 63))


def test_place_counts_and_not_memory():
    x = torch.randn(6, 10)
    assert torch.equal(rg.dropout(x.t().contiguous().t(), 0.5, seed=9), rg.dropout(x, 0.5, seed=9))
    assert torch.equal(rg.dropout(x[:, ::2], 0.5, seed=9), rg.dropout(x[:, ::2].contiguous(), 0.5, seed=9))


def test_dropped_values_do_not_matter():
    x = torch.full((64,), math.nan)
    y = rg.dropout(x, 0.5, seed=4)
    mask = kept(64, 0.5, 4)
    assert torch.equal(y.isnan(), mask) and torch.all(y[~mask] == 0)


def test_the_rate():
    """Of 2^16 draws of probability p, within 5 standard deviations."""
    for p in (0.01, 0.3, 0.9):
        n = 1 << 16
        dropped = (rg.dropout(torch.ones(n), p, seed=11) == 0).sum().item()
        assert abs(dropped - n * p) <= 5 * math.sqrt(n * p * (1 - p))


def test_the_module():
    m, x = rg.Dropout(0.5), torch.ones(50)
    torch.manual_seed(1)
    a, b = m(x), m(x)
    torch.manual_seed(1)
    assert torch.equal(m(x), a) and not torch.equal(a, b)
    assert torch.equal(m(x, seed=3), rg.dropout(x, 0.5, seed=3))
    assert m.eval()(x) is x and rg.Dropout(0.0)(x) is x
    # under checkpointing the second pass drops what the first did
    m.train()
    w = torch.ones(50, requires_grad=True)
    torch.utils.checkpoint.checkpoint(lambda v: m(v) * w, x, use_reentrant=False).sum().backward()
    torch.manual_seed(5)
    w.grad = None
    y = torch.utils.checkpoint.checkpoint(lambda v: m(v) * w, x, use_reentrant=False)
    y.sum().backward()
    assert torch.equal(w.grad, y.detach())


def test_a_seed_changed_after_the_forward_pass():
    x, seed = torch.ones(100, requires_grad=True), torch.tensor([6])
    y = rg.dropout(x, 0.5, seed=seed)
    seed.add_(1)
    assert torch.equal(torch.autograd.grad(y.sum(), x)[0], y.detach())


def test_refusals():
    x = torch.ones(4)
    for p in (1.0, -0.1, math.nan):
        with pytest.raises(ValueError):
            rg.dropout(x, p, seed=1)
    with pytest.raises(ValueError):
        rg.Dropout(1.0)
    with pytest.raises(ValueError, match="float32"):
        rg.dropout(x.double(), 0.5, seed=1)
    for seed in (torch.tensor([1, 2]), torch.tensor([1.0]), torch.tensor([1], dtype=torch.int32)):
        with pytest.raises(ValueError, match="seed"):
            rg.dropout(x, 0.5, seed=seed)
    with pytest.raises(ValueError):
        rg.dropout(torch.ones(4, device="meta"), 0.5, seed=1)
    leaf = x.clone().requires_grad_()
    (g,) = torch.autograd.grad(rg.dropout(leaf, 0.5, seed=1).sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable"):
        g.sum().backward()
