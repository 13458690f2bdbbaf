"""Attention, the bias of relative positions and dropout on the GPU against the CPU's: the same bits, for every class of sizes,
mask and alignment, and under graphs and streams."""
import math

import pytest
import torch

import bit_reproducible_training_amd as rg
import test_relative_bias as bias_cases
from test_attention import CASES, case, check, gradients
from test_gpu_norm import assert_same

pytestmark = pytest.mark.gpu


def cuda(t):
    return {n: v.cuda() if isinstance(v, torch.Tensor) else v for n, v in t.items()}


def compare(t, s, dy):
    got = gradients(cuda(t), cuda(s), dy.cuda())
    assert_same(got, gradients(t, s, dy))
    with torch.no_grad():
        assert torch.equal(rg.attention(**cuda(t), **cuda(s)).nan_to_num(7.0), got["y"].nan_to_num(7.0))
    return got


@pytest.mark.parametrize("c", CASES)
def test_the_formula(c):
    t, s, dy = case(*c, seed=sum(c[:6]))
    check(compare(t, s, dy), t, s, dy)


@pytest.mark.parametrize("d", [1, 2, 7, 8, 31, 32, 33, 48, 64, 65, 80, 96, 97, 127, 128])
def test_gives_the_cpu_bits_at_every_size(d):
    for c in ((2, 2, 1, 70, 133, d, False, True, None, True, 0.0), (1, 2, 2, 140, 140, d, True, False, None, False, 0.2),
              (1, 2, 1, 3, 300, d, False, False, "pairs", False, 0.1)):
        print(c, flush=True)
        compare(*case(*c))


@pytest.mark.parametrize("tq,tk", [(1, 1), (1, 255), (1, 256), (1, 257), (1, 1500), (2, 64), (8, 65), (9, 700), (31, 128), (32, 129),
                                   (33, 1), (64, 256), (65, 513), (127, 127), (128, 384), (129, 31), (255, 256), (256, 257),
                                   (257, 1030), (600, 96), (1100, 40)])
def test_gives_the_cpu_bits_at_every_length(tq, tk):
    for c in ((1, 2, 1, tq, tk, 20, False, False, None, False, 0.0), (2, 2, 2, tq, tk, 64, True, True, "pairs", True, 0.1)):
        print(c, flush=True)
        compare(*case(*c))


@pytest.mark.parametrize("h,kvh", [(1, 1), (8, 1), (12, 3), (6, 6), (40, 2), (128, 1), (129, 1)])
def test_shared_heads(h, kvh):
    for tq, tk in ((1, 520), (3, 300), (5, 300), (90, 90)):
        compare(*case(2, h, kvh, tq, tk, 16, True, True, "keys", True, 0.1))


def test_many_items_and_long_rows():
    compare(*case(40, 6, 6, 20, 33, 32, False, True, None, False, 0.0))
    compare(*case(1, 1, 1, 700, 2100, 64, True, False, None, True, 0.0))
    compare(*case(1, 1, 1, 2100, 300, 64, False, False, None, True, 0.1))
    compare(*case(1, 2, 2, 1, 9000, 64, False, False, None, True, 0.0))


def test_a_scale_and_a_late_start():
    for start in (-200, -5, 0, 37, 200):
        t, s, dy = case(2, 2, 2, 150, 100, 12)
        s.update(scale=-0.7, causal=True, query_start=start)
        compare(t, s, dy)


@pytest.mark.parametrize("hidden", [math.nan, math.inf, torch.finfo(torch.float32).min])
@pytest.mark.parametrize("d", [8, 64, 128])
def test_what_is_masked_reaches_nothing(hidden, d):
    for kind in ("causal", "pairs", "lengths"):
        t, s, dy = case(2, 2, 1, 200, 200, d, causal=kind == "causal", bias=True, drop=0.1)
        if kind == "lengths":
            s["key_lengths"] = torch.tensor([150, 0])
            t["k"][0, 150:], t["v"][0, 150:], t["k"][1], t["v"][1] = hidden, hidden, hidden, hidden
            got = compare(t, s, dy)
            assert got["y"].isfinite().all() and torch.all(got["y"][1] == 0) and torch.all(got["dk"][0, 150:] == 0)
            continue
        if kind == "pairs":
            s["mask"] = torch.ones(200, 200, dtype=torch.bool)
            s["mask"][:150, 150:] = False
        want = gradients(cuda(t), cuda(s), dy.cuda())
        t["v"][:, 160], t["k"][:, 170] = hidden, hidden
        got = compare(t, s, dy)
        assert torch.equal(got["y"][:, :150], want["y"][:, :150]) and torch.equal(got["dq"][:, :150], want["dq"][:, :150])
        t, s, dy = case(2, 2, 1, 200, 200, d, causal=True, drop=0.1)
        want = gradients(cuda(t), cuda(s), dy.cuda())
        t["q"][:, 40], dy[:, 41] = hidden, hidden
        got = compare(t, s, dy)
        for n in ("dk", "dv"):
            assert torch.equal(got[n][:, 42:], want[n][:, 42:]), n


def test_visible_nans_and_large_scores():
    t, s, dy = case(1, 2, 2, 80, 300, 16, bias=True)
    t["v"][0, 7, 0, 3], t["q"][0, 9], t["k"][0, 250, 1, 2] = math.nan, math.inf, -math.inf
    compare(t, s, dy)
    t, s, dy = case(1, 2, 2, 80, 300, 16, bias=True)
    t["q"] *= 1e19
    t["k"] *= 1e18
    compare(t, s, dy)
    t, s, dy = case(1, 2, 2, 80, 300, 16, bias=True)
    t["relative_bias"][:, ::3] = -math.inf
    t["relative_bias"][:, 1::3] = -1e5
    compare(t, s, dy)
    t, s, dy = case(1, 2, 2, 80, 300, 16)
    for n in "qkv":
        t[n] *= 1e-21
    dy *= 1e-20
    compare(t, s, dy)


def test_any_strides():
    t, s, dy = case(2, 4, 2, 70, 130, 20, drop=0.1)
    want = gradients(t, s, dy)
    kv = torch.stack((t["k"], t["v"]), 2).cuda()
    odd = torch.zeros(2, 70, 4, 23, device="cuda")[..., 1:21]
    odd.copy_(t["q"])
    rev = t["v"].transpose(1, 2).contiguous().transpose(1, 2).cuda()
    shifted = torch.zeros(t["k"].numel() + 1, device="cuda")[1:].view(t["k"].shape).copy_(t["k"])
    for q, k, v in ((odd, kv[:, :, 0], kv[:, :, 1]), (t["q"].cuda(), shifted, rev),
                    (t["q"].permute(3, 2, 1, 0).contiguous().permute(3, 2, 1, 0).cuda(), kv[:, :, 0], rev)):
        got = gradients({"q": q, "k": k, "v": v, "relative_bias": None}, s, dy.cuda())
        assert_same(got, want)
    got = gradients({**cuda(t)}, s, dy.transpose(1, 2).contiguous().cuda().transpose(1, 2))
    assert_same(got, want)
    for b, tq, tk in ((0, 4, 5), (2, 0, 5), (2, 4, 0)):
        compare(*case(b, 2, 1, tq, tk, 8, bias=True, causal=True))
    # one sequence's keys for every item, one query for every head
    t, s, dy = case(1, 2, 2, 5, 400, 8)
    t["k"], t["v"], t["q"] = (x.cuda().expand(3, -1, -1, -1) for x in (t["k"], t["v"], t["q"]))
    y = rg.attention(**t)
    assert torch.equal(y[0], y[2])


def test_lengths_of_any_kind():
    t, s, dy = case(5, 2, 2, 40, 90, 16)
    s["key_lengths"] = torch.tensor([-4, 0, 1, 90, 10 ** 12])
    a = compare(t, s, dy)
    s["key_lengths"] = torch.tensor([-4, 0, 1, 90, 91], dtype=torch.int32)
    assert_same(compare(t, s, dy), {n: v.cpu() for n, v in a.items()})


def test_masks_of_any_strides():
    t, s, dy = case(2, 4, 2, 50, 70, 16)
    g = torch.Generator().manual_seed(8)
    full = torch.rand(2, 4, 50, 70, generator=g) < 0.5
    for m in (full, full.transpose(2, 3).contiguous().transpose(2, 3), full[:1], full[:, :, :1], full[0, 0], full[0, 0, 0], full[:, :1],
              full[..., :1], torch.rand(2, 4, 50, 140, generator=g)[..., ::2] < 0.5, torch.tensor(True)):
        s["mask"] = m
        compare(t, s, dy)


def test_seeds_in_device_memory_and_graphs():
    """A captured step replayed with other inputs and seeds, eager work in between, each replay against the eager result."""
    t, s, dy = case(2, 4, 2, 130, 300, 64, causal=True, lengths=True, bias=True, drop=0.2)
    t, s, dy = cuda(t), cuda(s), dy.cuda()
    s["seed"] = torch.tensor([5], device="cuda")
    eager = gradients(t, s, dy)
    assert_same(eager, {n: v.cpu() for n, v in gradients(t, {**s, "seed": 5}, dy).items()})
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        gradients(t, s, dy)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = gradients(t, s, dy)
        x_out = rg.dropout(t["q"], 0.5, seed=s["seed"])
    for seed in (6, 7, 8):
        s["seed"].fill_(seed)
        t["q"].normal_()
        graph.replay()
        torch.cuda.synchronize()
        got = {n: v.cpu().clone() for n, v in out.items()}
        assert_same(gradients(t, {**s, "seed": seed}, dy), got)
        assert torch.equal(x_out, rg.dropout(t["q"], 0.5, seed=seed))
    # a seed changed between the passes
    q = t["q"].requires_grad_()
    y = rg.attention(**{**t, "q": q}, **s)
    s["seed"].add_(1)
    (a,) = torch.autograd.grad(y, q, dy)
    (b,) = torch.autograd.grad(rg.attention(**{**t, "q": q}, **{**s, "seed": 8}), q, dy)
    assert torch.equal(a, b)


def test_two_streams_at_once():
    t, s, dy = case(2, 4, 2, 200, 600, 32, causal=True, bias=True, drop=0.2)
    t, s, dy = cuda(t), cuda(s), dy.cuda()
    want = gradients(t, s, dy)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(3)], []
    for _ in range(3):
        for stream in streams:
            with torch.cuda.stream(stream):
                got.append(gradients(t, s, dy))
    torch.cuda.synchronize()
    for g in got:
        assert_same(g, {n: v.cpu() for n, v in want.items()})


@pytest.mark.parametrize("c", bias_cases.CASES + [(32, 128, True, 700, 1500, 3), (32, 128, False, 65, 4099, 4034)])
def test_relative_bias(c):
    a, b = bias_cases.check("cuda", *c), bias_cases.check("cpu", *c)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("n,shift", [(1, 0), (3, 0), (4, 1), (1001, 0), (1001, 3), (4096, 2), (1 << 20, 0), ((1 << 20) + 7, 1)])
def test_dropout(n, shift):
    x = torch.randn(n + shift)[shift:]
    flat = torch.zeros(n + shift, device="cuda")[shift:].copy_(x)
    for p in (0.0, 0.3):
        leaf, up = flat.detach().requires_grad_(), torch.randn(n)
        y = rg.dropout(leaf, p, seed=n)
        assert torch.equal(y.cpu(), rg.dropout(x, p, seed=n))
        (g,) = torch.autograd.grad(y, leaf, up.cuda())
        assert torch.equal(g.cpu(), rg.dropout(up, p, seed=n))
        # a seed in device memory, changed after the forward pass
        at = torch.tensor([n], device="cuda")
        y = rg.dropout(leaf, p, seed=at)
        at.zero_()
        assert torch.equal(torch.autograd.grad(y, leaf, up.cuda())[0], g)


def test_a_block_of_the_layers():
    """Self attention, cross attention to padded states, dropout and the residual norms, as a decoder's block runs them: the CPU's bits."""
    results = []
    for device in ("cpu", "cuda"):
        torch.manual_seed(2)
        rg.guard().reset()
        own, cross = rg.Attention(48, 4, num_kv_heads=2, dropout=0.1), rg.Attention(48, 4, states_width=20, dropout=0.1)
        bias, drop = rg.RelativePositionBias(4, 8, 16, bidirectional=False), rg.Dropout(0.1)
        first, second = rg.ResidualNorm(48), rg.ResidualNorm(48)
        modules = torch.nn.ModuleList([own, cross, bias, drop, first, second]).to(device)
        x, states, up = torch.randn(3, 40, 48), torch.randn(3, 70, 20), torch.randn(3, 40, 48)
        x, states = x.to(device).requires_grad_(), states.to(device).requires_grad_()
        r, y = first(x, drop(own(x, causal=True, relative_bias=bias(40, 40))))
        r, y = second(r, drop(cross(y, states, key_lengths=torch.tensor([70, 1, 33], device=device))))
        y.backward(up.to(device))
        results.append([y.detach().cpu(), x.grad.cpu(), states.grad.cpu()] + [p.grad.cpu() for p in modules.parameters() if p.grad is not None])
        rg.guard().check()
    assert len(results[0]) > 10
    for a, b in zip(*results):
        assert torch.equal(a, b)


def test_backward_into_a_graph_beside_an_eager_one():
    """The forward pass refuses a capture while an eager graph of the same leaves is alive, whose stream the captured backward pass
    would wait for; once that is gone it is captured."""
    t, s, dy = case(1, 2, 2, 40, 60, 16, bias=True)
    t, dy = cuda(t), dy.cuda()
    leaves = {n: v.requires_grad_() for n, v in t.items()}
    table = torch.randn(8, 2, device="cuda", requires_grad=True)
    want = torch.autograd.grad(rg.attention(**leaves), list(leaves.values()), dy)
    for run, alive in ((lambda: rg.attention(**leaves), rg.attention(**leaves)),
                       (lambda: rg.dropout(leaves["q"], 0.5, seed=1), rg.dropout(leaves["q"], 0.5, seed=1)),
                       (lambda: rg.relative_position_bias(table, 3, 3, max_distance=9), rg.relative_position_bias(table, 3, 3, max_distance=9))):
        torch.cuda.synchronize()
        refused = None
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            torch.zeros(4, device="cuda").add_(1)
            try:
                run()
            except ValueError as e:
                refused = str(e)
        assert "still alive" in refused
        del alive
    del run
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(rg.attention(**leaves), list(leaves.values()), dy)
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_the_layer_refuses_a_capture_beside_an_eager_graph():
    layer = rg.Attention(16, 2).cuda()
    x = torch.randn(1, 5, 16, device="cuda")
    alive = layer(x)
    torch.cuda.synchronize()
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        torch.zeros(4, device="cuda").add_(1)
        with pytest.raises(ValueError, match="still alive"):
            layer(x)
    del alive


def test_key_blocks_in_turns_and_items_apart():
    """So many queries that their sums over key blocks are taken some key blocks at a time: each item and head as by itself."""
    torch.manual_seed(5)
    q, dy = (torch.randn(1, 8192, 16, 128, device="cuda") for _ in range(2))
    k, v = (torch.randn(1, 4096, 16, 128, device="cuda") for _ in range(2))
    bias = torch.randn(16, 8192 + 4096 - 1, device="cuda")
    s = dict(key_lengths=torch.tensor([4000], device="cuda"), causal=True, query_start=-4000)
    whole = gradients({"q": q, "k": k, "v": v, "relative_bias": bias}, s, dy)
    for h in (0, 11):
        one = gradients({"q": q[:, :, h:h + 1], "k": k[:, :, h:h + 1], "v": v[:, :, h:h + 1], "relative_bias": bias[h:h + 1]}, s,
                        dy[:, :, h:h + 1])
        for n in ("y", "dq", "dk", "dv"):
            assert torch.equal(whole[n][:, :, h], one[n][:, :, 0]), n
        assert torch.equal(whole["drelative_bias"][h], one["drelative_bias"][0])


def test_offsets_past_32_bits():
    """Items 2^32 values apart, as in a long cache."""
    t, s, dy = case(2, 4, 2, 70, 300, 16, causal=True)
    want = gradients(cuda(t), s, dy.cuda())
    room = torch.empty(2 ** 32 + 300 * 64, device="cuda")
    k, v = (room.as_strided((2, 300, 2, 16), (2 ** 32, 64, 16, 1), at) for at in (0, 32))
    k.copy_(t["k"])
    v.copy_(t["v"])
    got = gradients({"q": t["q"].cuda(), "k": k, "v": v, "relative_bias": None}, s, dy.cuda())
    assert_same(got, {n: x.cpu() for n, x in want.items()})
    one = rg.attention(t["q"][:, :1].cuda(), k, v)
    assert torch.equal(one, rg.attention(t["q"][:, :1].cuda(), t["k"].cuda(), t["v"].cuda()))


def test_shared_rows_of_strides_too_far_apart():
    """Positions more than 2^22 values apart are brought together."""
    t, s, dy = case(1, 1, 1, 3, 9, 8)
    room = torch.zeros(9 * (2 ** 22 + 4), device="cuda")
    k = room.as_strided((1, 9, 1, 8), (1, 2 ** 22 + 4, 1, 1))
    k.copy_(t["k"])
    assert torch.equal(rg.attention(t["q"].cuda(), k, t["v"].cuda()).cpu(), rg.attention(t["q"], t["k"], t["v"]))
