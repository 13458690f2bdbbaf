"""The vocabulary projection's cross entropy and its gradients on the GPU against the CPU's: the same bits."""
import math

import pytest
import torch

import bit_reproducible_training_amd as rg
from bit_reproducible_training_amd import _lib
from test_loss import case, check, results

pytestmark = pytest.mark.gpu


def assert_same(got, want):
    for name, a, b in zip(("loss", "dx", "dw"), got, want):
        a, b = a.cpu(), b.cpu()
        nan = b.isnan()
        assert torch.equal(a.isnan(), nan), name
        assert torch.equal(a[~nan].view(torch.int32), b[~nan].view(torch.int32)), name


# One word, one part and its ends, one token, sizes off every multiple, long rows, few and many tokens a word.
CASES = [(1, 1, 1, None), (1, 7, 3, None), (3, 4, 63, None), (5, 16, 64, 2), (17, 33, 65, 1), (64, 64, 1024, None),
         (130, 40, 1003, 5), (2, 768, 50257, None), (96, 128, 4099, None), (33, 100, 16385, 3), (700, 20, 130, 1),
         (1030, 65, 200, 3), (300, 1028, 77, 9),
         # few tokens: one, 8, 32 and past them, widths of each register class and past them
         (1, 33, 31, None), (8, 257, 33, 4), (9, 512, 100, 4), (32, 770, 97, 10), (33, 64, 97, 10), (31, 1024, 40, 2),
         (24, 1025, 70, 5), (64, 1024, 95, 9)]


@pytest.mark.parametrize("n,d,v,words", CASES)
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_gives_the_cpu_bits(n, d, v, words, reduction):
    x, w, t = case(n, d, v, seed=n + v, lean=3.0, ignored=range(1, n, 7), words=words)
    up = torch.randn(n, generator=torch.Generator().manual_seed(1)) if reduction == "none" else None
    got = results(x.cuda(), w.cuda(), t.cuda(), reduction, None if up is None else up.cuda())
    assert_same(got, results(x, w, t, reduction, up))
    check(got, x, w, t, reduction=reduction, up=up)


@pytest.mark.parametrize("S", [1, 2, 3])
def test_slices(S):
    x, w, t = case(70, 50, 333, seed=S)
    got = results(x.cuda(), w.cuda(), t.cuda(), "sum", slices=S)
    assert_same(got, results(x, w, t, "sum", slices=S))
    check(got, x, w, t, reduction="sum", S=S)


def test_groups_of_tokens():
    v = 2 ** 20 + 3
    n = 2 * _lib.lib.rg_loss_group_tokens(v) + 5
    x, w, t = case(n, 3, v, seed=2, std=1.0, words=40)
    assert_same(results(x.cuda(), w.cuda(), t.cuda()), results(x, w, t))


def test_parts_of_the_gradient_and_of_the_output():
    x, w, t = case(200, 40, 500, seed=3)
    want = results(x, w, t)
    x, w, t = x.cuda(), w.cuda(), t.cuda()
    leaf = x.clone().requires_grad_()
    (dx,) = torch.autograd.grad(rg.linear_cross_entropy(leaf, w, t), [leaf])
    leaf = w.clone().requires_grad_()
    (dw,) = torch.autograd.grad(rg.linear_cross_entropy(x, leaf, t), [leaf])
    with torch.no_grad():
        assert_same((rg.linear_cross_entropy(x, w, t), dx, dw), want)


def test_tokens_that_do_not_count_and_no_tokens():
    for reduction in ("mean", "sum", "none"):
        x, w, t = case(40, 12, 90, seed=4)
        t[::3], t[4], t[5] = -100, 90, -7
        assert_same(results(x.cuda(), w.cuda(), t.cuda(), reduction), results(x, w, t, reduction))
        t[:] = -100
        assert_same(results(x.cuda(), w.cuda(), t.cuda(), reduction), results(x, w, t, reduction))
        assert_same(results(x[:0].cuda(), w.cuda(), t[:0].cuda(), reduction), results(x[:0], w, t[:0], reduction))


def test_non_finite_inputs_give_the_cpu_bits():
    x, w, t = case(20, 12, 90, seed=4)
    x[3, 2], x[7, 1], w[9, 9] = math.nan, math.inf, -math.inf
    x[11], w[11] = 3e38, 3e38  # a logit past the range
    got, want = results(x.cuda(), w.cuda(), t.cuda(), "none"), results(x, w, t, "none")
    assert_same(got[:1], want[:1])


@pytest.mark.parametrize("shift", [1, 2, 3])
def test_operands_off_16_bytes(shift):
    x, w, t = case(50, 36, 200, seed=shift)

    def moved(v):
        flat = torch.empty(v.numel() + 8, device="cuda", dtype=v.dtype)
        return flat[shift:shift + v.numel()].view(v.shape).copy_(v)

    assert_same(results(moved(x), moved(w), moved(t)), results(x, w, t))


def test_scaled_losses_and_second_backwards():
    x, w, t = case(100, 30, 400, seed=6)
    want = results(x, w, t, up=torch.tensor(0.3))
    x, w, t = x.cuda().requires_grad_(), w.cuda().requires_grad_(), t.cuda()
    loss = rg.linear_cross_entropy(x, w, t)
    for _ in range(2):
        got = torch.autograd.grad(loss, (x, w), torch.tensor(0.3, device="cuda"), retain_graph=True)
        assert_same((loss, *got), want)


def test_another_stream_and_graph_replays():
    x, w, t = case(150, 64, 1000, seed=9)
    want = results(x, w, t)
    x, w, t = x.cuda(), w.cuda(), t.cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert_same(results(x, w, t), want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = results(x, w, t)
    for k in range(3):
        for v in got:
            v.fill_(math.nan)
        (torch.randn(1000, 1000, device="cuda") @ torch.randn(1000, 1000, device="cuda")).sum().item()
        graph.replay()
        torch.cuda.synchronize()
        assert_same(got, want)


def test_repeated_runs_give_the_same_bits():
    x, w, t = case(1500, 96, 3000, seed=10, words=30)
    x, w, t = x.cuda(), w.cuda(), t.cuda()
    first = results(x, w, t)
    for _ in range(5):
        assert_same(results(x, w, t), first)


def test_refuses_tensors_on_two_devices():
    x, w, t = case(6, 8, 20, device="cuda")
    for bad in ((x, w.cpu(), t), (x, w, t.cpu()), (x.cpu(), w, t)):
        with pytest.raises(ValueError):
            rg.linear_cross_entropy(*bad)


@pytest.mark.parametrize("S", [1, 2, 3])
@pytest.mark.parametrize("n", [1, 16, 17, 32, 33, 64, 65])
def test_few_tokens_of_every_width(n, S):
    for d in (1, 256, 257, 600, 1000, 1025, 1540, 1700, 2047, 2048, 2049):
        x, w, t = case(n, d, 50, seed=n + d, lean=2.0)
        with torch.no_grad():
            got = rg.linear_cross_entropy(x.cuda(), w.cuda(), t.cuda(), reduction="none", slices=S)
            want = rg.linear_cross_entropy(x, w, t, reduction="none", slices=S)
        assert torch.equal(got.cpu().view(torch.int32), want.view(torch.int32)), d


@pytest.mark.parametrize("n", [4096, 4097, 9001])
@pytest.mark.parametrize("words", [1, 700])
def test_many_tokens_of_the_same_words(n, words):
    x, w, t = case(n, 5, 700, seed=n, words=words, ignored=range(3, n, 11))
    t[5::97], t[7::101] = 700, -3
    assert_same(results(x.cuda(), w.cuda(), t.cuda()), results(x, w, t))


@pytest.mark.parametrize("below,above", [(0, 64), (64, 0), (54, 300), (4096, 0), (0, 270000)])
@pytest.mark.parametrize("n", [1, 40, 70])
def test_parts_whose_logits_are_all_minus_infinity(n, below, above):
    from test_loss import words_past_the_range

    x, w, t, _ = words_past_the_range(n, below, above)
    got = results(x.cuda(), w.cuda(), t.cuda())
    assert torch.isfinite(got[0]) and torch.isfinite(got[2]).all()
    assert_same(got, results(x, w, t))
    for t in (torch.zeros_like(t), t):
        assert_same(results(x.cuda(), -w.cuda(), t.cuda()), results(x, -w, t))


@pytest.mark.parametrize("n", [7, 300, 2100])
@pytest.mark.parametrize("d", [33, 36])
def test_hidden_states_of_tokens_that_do_not_count_reach_nothing(n, d):
    """Padding between and after the tokens, in one group and in two."""
    x, w, t = case(n, d, 90, seed=n, lean=2.0)
    keep = torch.rand(n, generator=torch.Generator().manual_seed(3)) < 0.7
    keep[0], keep[-1] = True, False
    t[~keep] = -100
    for large in (1e12, math.inf, math.nan):
        x[~keep, 1::2] = large
        got = results(x.cuda(), w.cuda(), t.cuda())
        assert_same(got, results(x, w, t))
        if n < 2048:
            part = results(x[keep].cuda(), w.cuda(), t[keep].cuda())
            assert torch.equal(got[2], part[2]) and torch.equal(got[1][keep.cuda()], part[1])


@pytest.mark.parametrize("n,d,v", [(9, 12, 90), (20, 1601, 130), (70, 30, 90), (130, 768, 333), (70, 4100, 80), (66, 4103, 70), (2100, 36, 70)])
def test_a_nan_or_infinity_gives_the_cpu_bits_everywhere(n, d, v):
    """In x and in the weight, in a token's and a word's first and last values, on every way to the logits."""
    for bad in (math.nan, math.inf, -math.inf):
        for where in ("x", "w", "x last", "w last"):
            x, w, t = case(n, d, v, seed=n, lean=2.0, ignored=(1,))
            (x if where[0] == "x" else w)[(-1, -1) if "last" in where else (2, 0)] = bad
            for reduction in ("mean", "none"):
                got, want = results(x.cuda(), w.cuda(), t.cuda(), reduction), results(x, w, t, reduction)
                assert_same(got, want)
            assert got[0].isnan().sum() == (1 if where[0] == "x" else n - 1)


def test_left_out_tokens_may_hold_anything():
    x, w, t = case(150, 64, 200, seed=2)
    want = results(x.cuda(), w.cuda(), t.where(torch.arange(150) % 3 > 0, -100).cuda())
    t[::3] = -100
    x[::3] = math.nan
    assert_same(results(x.cuda(), w.cuda(), t.cuda()), [v.cpu() for v in want])


@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_the_guard_hears_a_gradient_that_is_not_finite(reduction):
    rg.guard().reset()
    torch.manual_seed(0)
    m = rg.LinearCrossEntropy(8, 20, reduction=reduction).cuda()
    x, t = torch.randn(5, 8, device="cuda"), torch.randint(0, 20, (5,), device="cuda")
    loss = m(x, t)
    up = torch.ones_like(loss)
    torch.autograd.grad(loss, m.weight, up, retain_graph=True)
    rg.guard().check()
    up.view(-1)[-1] = math.nan
    torch.autograd.grad(loss, m.weight, up)
    assert rg.guard().first_offender() == "linear_cross_entropy gradient"
    rg.guard().reset()


@pytest.mark.parametrize("words", [1, 2, 90])
def test_a_frequent_word_over_several_batches_of_tokens(words):
    """Tokens are listed 8192 at a time: a word's in three batches, and in the middle one only."""
    n = 20011
    x, w, t = case(n, 5, 90, seed=words, words=words, ignored=range(3, n, 11))
    t[8192:16384:3] = 71
    want = results(x, w, t)
    assert_same(results(x.cuda(), w.cuda(), t.cuda()), want)
    assert_same(results(x.cuda(), w.cuda(), t.cuda()), want)
