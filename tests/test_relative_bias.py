"""The bias of relative positions and its gradient against the formula, and its refusals, on the CPU."""
import math

import pytest
import torch

import bit_reproducible_training_amd as rg

EPS32 = 2.0 ** -24


def bucket(relative, buckets, max_distance, both):
    """The definition, a step's end decided in whole numbers."""
    side = buckets // 2 if both else buckets
    at = side if both and relative > 0 else 0
    n = abs(relative) if both else max(0, -relative)
    exact = side // 2
    if n < exact:
        return at + n
    steps, t = side - exact, 0
    while t + 1 < steps and n ** steps * exact ** (t + 1) >= max_distance ** (t + 1) * exact ** steps:
        t += 1
    return at + exact + t


def check(device, buckets, max_distance, both, tq, tk, start, heads=3):
    g = torch.Generator().manual_seed(tq * 1000 + tk)
    table, dy = torch.randn(buckets, heads, generator=g), torch.randn(heads, tq, tk, generator=g)
    kw = dict(max_distance=max_distance, bidirectional=both, query_start=start)
    leaf = table.to(device).requires_grad_()
    dense = rg.relative_position_bias(leaf, tq, tk, **kw)
    strip = rg.relative_position_bias(leaf, tq, tk, dense=False, **kw)
    which = [bucket(r - start, buckets, max_distance, both) for r in range(-(tq - 1), tk)]
    place = torch.arange(tk)[None, :] - torch.arange(tq)[:, None] + tq - 1
    assert torch.equal(strip.cpu(), table[which].t()) if which else strip.numel() == 0
    if dense.numel():
        assert torch.equal(dense.cpu(), table[torch.tensor(which)[place]].permute(2, 0, 1))
    d_strip = torch.randn(strip.shape, generator=g)
    got = torch.autograd.grad(dense, leaf, dy.to(device))[0].cpu(), torch.autograd.grad(strip, leaf, d_strip.to(device))[0].cpu()
    for mine, up, index in ((got[0], dy.flatten(1), torch.tensor(which)[place].flatten() if tq and tk else None),
                            (got[1], d_strip, torch.tensor(which) if which else None)):
        want, size = torch.zeros(buckets, heads).double(), torch.zeros(buckets, heads).double()
        if index is not None:
            want.index_add_(0, index, up.t().double())
            size.index_add_(0, index, up.t().double().abs())
        # a term passes a run's additions (64), the runs', a strand's and the tree's
        steps = 64 + tq / 64 + (tq + tk) / 256 + 10
        assert torch.all((mine.double() - want).abs() <= steps * EPS32 * size)
    return dense.detach().cpu(), strip.detach().cpu(), *got


CASES = [(32, 128, True, 40, 300, 0), (32, 128, False, 300, 300, 0), (8, 20, True, 1, 513, 512), (2, 2, False, 7, 5, 3),
         (4, 3, True, 130, 2, -9), (1026, 1000, True, 3, 1200, 600), (6, 2 ** 31 - 1, False, 1, 1, 10 ** 9),
         (10, 6, True, 200, 1, 0), (32, 128, True, 0, 5, 0), (32, 128, True, 5, 0, 0), (16, 9, False, 1, 1, 0)]


@pytest.mark.parametrize("c", CASES)
def test_values_and_gradient_are_the_formula(c):
    check("cpu", *c)


def test_steps_that_end_exactly():
    """8 buckets of a side with 8 = 128^(1/..): distances 8 2^(t/2) end steps exactly where t is even."""
    strip = rg.relative_position_bias(torch.arange(32.0)[:, None], 200, 1, dense=False)[0].flip(0)
    assert [strip[n].item() for n in (7, 8, 11, 12, 15, 16, 31, 32, 63, 64, 90, 91, 199)] == \
        [7, 8, 8, 9, 9, 10, 11, 12, 13, 14, 14, 15, 15]


def test_in_an_attention_and_shared_by_layers():
    module = rg.RelativePositionBias(2, num_buckets=8, max_distance=16, bidirectional=False)
    q, k = torch.randn(1, 5, 2, 4), torch.randn(1, 7, 2, 4)
    bias = module(5, 7, query_start=2)
    (rg.attention(q, k, k, relative_bias=bias) + rg.attention(k[:, :5], k, k, relative_bias=bias)).sum().backward()
    shared = module.weight.grad.clone()
    module.weight.grad = None
    rg.attention(q, k, k, relative_bias=module(5, 7, query_start=2)).sum().backward()
    rg.attention(k[:, :5], k, k, relative_bias=module(5, 7, query_start=2)).sum().backward()
    assert torch.allclose(module.weight.grad, shared, rtol=1e-4, atol=1e-6)
    assert torch.equal(module.dense(5, 7, 2)[:, 1, 3], bias[:, 3 - 1 + 4])


def test_refusals():
    f, t = rg.relative_position_bias, torch.zeros(8, 2)
    for bad in (dict(table=torch.zeros(8)), dict(table=torch.zeros(7, 2)), dict(table=torch.zeros(2, 2)), dict(table=torch.zeros(1, 2), bidirectional=False),
                dict(table=torch.zeros(1028, 2)), dict(max_distance=2), dict(max_distance=2 ** 31), dict(q_len=-1), dict(k_len=2 ** 22 + 1),
                dict(query_start=2 ** 33), dict(table=torch.zeros(8, 0)), dict(table=t.double()), dict(table=torch.zeros(8, 4097))):
        with pytest.raises(ValueError):
            f(**{**dict(table=t, q_len=3, k_len=3), **bad})
    with pytest.raises(ValueError):
        rg.RelativePositionBias(2, num_buckets=7)
    leaf = t.clone().requires_grad_()
    (g,) = torch.autograd.grad(f(leaf, 3, 3).sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable"):
        g.sum().backward()
    assert not math.isnan(f(t, 3, 3).sum())
