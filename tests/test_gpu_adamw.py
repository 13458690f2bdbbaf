"""The AdamW step on the GPU against the CPU's: the same bits, whatever the sizes, alignment, number of
tensors and stream."""
import math

import pytest
import torch

import bit_reproducible_training_amd as rg
from test_adamw import SETTINGS, check_step, tensors

pytestmark = pytest.mark.gpu


def same(a, b):
    return all(torch.equal(x.cpu().view(torch.int32), y.cpu().view(torch.int32)) for x, y in zip(a, b))


SIZES = [[(1,)], [(255,), (256,), (257,)], [(4096,), (4095,), (4097,), (0,), (16384 + 3,)],
         [(1 + (i * 37) % 700,) for i in range(230)], [(1025, 1023), (3,)]]


@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: "%dx%s" % (len(s), s[0]))
def test_step_gives_the_cpu_bits(sizes):
    cpu = tensors(sizes, len(sizes))
    before = tuple([t.clone() for t in ts] for ts in cpu)
    gpu = tuple([t.cuda() for t in ts] for ts in cpu)
    for step in (1, 7):
        rg.adamw_step(*cpu, step=step, **SETTINGS)
        rg.adamw_step(*gpu, step=step, **SETTINGS)
        if step == 1:
            check_step(before, (gpu[0], gpu[2], gpu[3]), 1, SETTINGS)
    assert all(same(a, b) for a, b in zip(cpu, gpu))


@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: "%dx%s" % (len(s), s[0]))
def test_step8_gives_the_cpu_bits(sizes):
    p, g, _, _ = tensors(sizes, 20 + len(sizes))
    q, h = [t.cuda() for t in p], [t.cuda() for t in g]
    a, b = rg.adamw8_state(p), rg.adamw8_state(q)
    for step in (1, 2, 3, 100):
        rg.adamw8_step(p, g, *a, step=step, **SETTINGS)
        rg.adamw8_step(q, h, *b, step=step, **SETTINGS)
    assert same(p, q)
    assert all(torch.equal(x, y.cpu()) for x, y in zip(a, b))
    assert same(rg.adamw8_values(*a), rg.adamw8_values(*b))


@pytest.mark.parametrize("shift", [1, 2, 3])
def test_tensors_off_16_bytes_and_out_of_step_with_each_other(shift):
    """Views of flat buffers at odd places; the values around them stay."""
    n = 9000
    cpu = tensors([(n + 8,)] * 4, shift)
    gpu = tuple([t.cuda() for t in ts] for ts in cpu)
    views = lambda ts, k: [t[k:k + n] for t in ts]  # noqa: E731
    rg.adamw_step(views(cpu[0], shift), views(cpu[1], 0), views(cpu[2], shift), views(cpu[3], 4), step=3)
    rg.adamw_step(views(gpu[0], shift), views(gpu[1], 0), views(gpu[2], shift), views(gpu[3], 4), step=3)
    assert all(same(a, b) for a, b in zip(cpu, gpu))
    a, b = rg.adamw8_state(views(cpu[0], 0)), rg.adamw8_state(views(gpu[0], 0))
    rg.adamw8_step(views(cpu[0], shift), views(cpu[1], 1), *a, step=3)
    rg.adamw8_step(views(gpu[0], shift), views(gpu[1], 1), *b, step=3)
    assert same(cpu[0], gpu[0]) and all(torch.equal(x, y.cpu()) for x, y in zip(a, b))


def test_extreme_values_give_the_cpu_bits():
    """Zeros, subnormal numbers, infinities, NaN and squares past the range, beside ordinary ones."""
    special = [0.0, -0.0, 1e-45, -1e-40, 1e-38, 3e38, -3e38, math.inf, -math.inf, math.nan, 1e20, 1e-20]
    g = torch.tensor(special * 90 + [1.0] * 64)
    p, m = torch.linspace(-2, 2, g.numel()), g.roll(5) * 0.5
    v = g.roll(9).abs()
    cpu, gpu = [[p.clone()], [g], [m.clone()], [v.clone()]], [[p.cuda()], [g.cuda()], [m.cuda()], [v.cuda()]]
    rg.adamw_step(*cpu, step=2)
    rg.adamw_step(*gpu, step=2)
    for a, b in zip(cpu, gpu):
        a, b = a[0], b[0].cpu()
        nan = a.isnan()
        assert torch.equal(nan, b.isnan())
        assert torch.equal(a[~nan].view(torch.int32), b[~nan].view(torch.int32))
    p, q = [p.clone()], [p.cuda()]
    a, b = rg.adamw8_state(p), rg.adamw8_state(q)
    for step in (1, 2):
        rg.adamw8_step(p, [g], *a, step=step)
        rg.adamw8_step(q, [g.cuda()], *b, step=step)
    assert all(torch.equal(x, y.cpu()) for x, y in zip(a, b))
    assert torch.equal(p[0].isnan(), q[0].cpu().isnan())


def test_step_runs_on_the_current_stream_and_in_a_graph():
    p, g, m, v = tensors([(100000,), (33,)], 8, "cuda")
    want = tuple([t.clone() for t in ts] for ts in (p, m, v))
    for _ in range(3):
        rg.adamw_step(want[0], g, want[1], want[2], step=4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        rg.adamw_step(p, g, m, v, step=4)
        with torch.cuda.graph(graph, stream=side):
            rg.adamw_step(p, g, m, v, step=4)
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
    assert same(p, want[0]) and same(m, want[1]) and same(v, want[2])


def test_tensors_on_two_devices_are_refused():
    p, g, m, v = tensors([(10,)], 1, "cuda")
    with pytest.raises(ValueError):
        rg.adamw_step(p, [g[0].cpu()], m, v, step=1)
    with pytest.raises(ValueError):
        rg.adamw_step(p + [torch.zeros(3)], g + [torch.zeros(3)], m + [torch.zeros(3)], v + [torch.zeros(3)], step=1)


@pytest.mark.parametrize("count", [3, 127, 128, 129, 300])
def test_moments_in_one_row_or_apart_take_the_same_step(count):
    sizes = [(1 + (37 * i) % 700,) for i in range(count)]
    p, g, _, _ = tensors(sizes, count, "cuda")
    q = [t.clone() for t in p]
    row = rg.adamw8_state(p)
    apart = [[torch.zeros(len_, dtype=torch.uint8, device="cuda") for len_ in lens]
             for lens in ([-(-t.numel() // 256) * k for t in p] for k in (256, 1, 256, 1))]
    for step in (1, 2):
        rg.adamw8_step(p, g, *row, step=step)
        rg.adamw8_step(q, g, *apart, step=step)
    assert same([t.cpu() for t in p], q)
    assert all(torch.equal(a, torch.cat(b)) for a, b in zip(row, apart))
