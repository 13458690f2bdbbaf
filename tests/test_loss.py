"""The vocabulary projection's cross entropy and its gradients against the formula in 64 bits and against
differences, and its refusals, on the CPU."""
import ctypes
import math

import pytest
import torch

import bit_reproducible_training_amd as rg
from bit_reproducible_training_amd import _lib

EPS32 = 2.0 ** -24


def case(n, d, v, seed=0, lean=0.0, std=0.3, ignored=(), words=None, device="cpu"):
    """Hidden states that lean towards their targets by `lean`; words: how many the targets are among."""
    g = torch.Generator().manual_seed(seed)
    w = std * torch.randn(v, d, generator=g)
    t = torch.randint(0, words or v, (n,), generator=g)
    x = torch.randn(n, d, generator=g) + lean * w[t] / w[t].norm(dim=1, keepdim=True)
    for i in ignored:
        t[i] = -100
    return x.to(device), w.to(device), t.to(device)


def results(x, w, t, reduction="mean", up=None, **settings):
    """(loss, dx, dw)"""
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    loss = rg.linear_cross_entropy(x, w, t, reduction=reduction, **settings)
    return (loss.detach(), *torch.autograd.grad(loss, (x, w), torch.ones_like(loss) if up is None else up))


def step(top, S):
    """The fixed-point step of a row whose largest magnitude is top: the scale is at most 2 top / 127,
    and 7 (S - 1) bits are kept below it."""
    return 2 * top / 127 * 2.0 ** (-7 * (S - 1))


def bounds(x, w, t, reduction="mean", up=None, S=3):
    """The definition in 64 bits, (loss, dx, dw), and how far the float32 results may be from them.
    A product is off by half a step of one operand times the other, summed, and rounded once.
    Exponentials (one unit), their sums (2 + 4 + 6 levels and the strands' parts) and the quotient
    are roundings of positive numbers, 2^-24 of the result each, and the logits' errors multiply them by
    e^(2 off): `rho` relative to a probability. The target's own share is rounded by itself."""
    x, w, t = x.cpu().double(), w.cpu().double(), t.cpu()
    n, v = x.shape[0], w.shape[0]
    kept = t != -100
    safe = torch.where(kept, t, 0)
    z = x @ w.t()
    off_z = 0.5 * (step(x.abs().amax(1), S)[:, None] * w.abs().sum(1) + step(w.abs().amax(1), S) * x.abs().sum(1)[:, None]
                   + step(x.abs().amax(1), S)[:, None] * step(w.abs().amax(1), S) * x.shape[1]) + EPS32 * z.abs()
    off_z = off_z.amax(1)
    sums = (20 + v / 4096) * EPS32
    lse = torch.logsumexp(z, 1)
    rows = torch.where(kept, lse - z.gather(1, safe[:, None])[:, 0], 0.0)
    off_rows = torch.where(kept, 2 * off_z + sums + 2 * EPS32 * rows.abs(), 0.0)
    g = torch.ones(n, dtype=torch.float64)
    if reduction == "mean":
        loss, off_loss = rows.sum() / kept.sum(), off_rows.sum() / kept.sum()
        off_loss = off_loss + 2 * EPS32 * loss.abs()
        g = g / kept.sum() * (1.0 if up is None else float(up))
    elif reduction == "sum":
        loss, off_loss = rows.sum(), off_rows.sum() + EPS32 * rows.sum()
        g = g * (1.0 if up is None else float(up))
    else:
        loss, off_loss = rows, off_rows
        g = g if up is None else up.cpu().double()
    g = torch.where(kept, g, 0.0)
    rho = (torch.expm1(2 * off_z) + sums + 6 * EPS32)[:, None]
    p = torch.exp(z - lse[:, None])
    onehot = torch.zeros(n, v, dtype=torch.float64)
    onehot[torch.arange(n), safe] = 1.0
    dz = g[:, None] * (p - onehot)
    others = (g[:, None] * p).abs() * (1 - onehot)
    off_others = rho * others
    off_target = (g[:, None].abs() * onehot * (rho * p + 4 * EPS32))
    size_target = (dz * onehot).abs()
    dx, dw = dz @ w, dz.t() @ x
    off_dx = off_others @ w.abs() + 0.5 * (step(others.amax(1), S)[:, None] * w.abs().sum(0)
                                           + step(w.abs().amax(0), S) * others.sum(1, keepdim=True) * 1.01) \
        + off_target @ w.abs() + 3 * EPS32 * (dx.abs() + size_target @ w.abs() + others @ w.abs())
    groups = -(-n // _lib.lib.rg_loss_group_tokens(v))
    off_dw = off_others.t() @ x.abs() + 0.5 * (step(others.amax(0), S)[:, None] * x.abs().sum(0)
                                               + step(x.abs().amax(0), S) * others.sum(0)[:, None] * 1.01) \
        + off_target.t() @ x.abs() \
        + (4 + groups) * EPS32 * (others.t() @ x.abs()) + (8 + n / 16) * EPS32 * (size_target.t() @ x.abs())
    return (loss, dx, dw), (off_loss, off_dx, off_dw)


def check(got, x, w, t, **settings):
    want, off = bounds(x, w, t, **settings)
    for name, g, e, o in zip(("loss", "dx", "dw"), got, want, off):
        err = (g.cpu().double() - e).abs()
        assert torch.all(err <= o + 1e-37), (name, (err / (o + 1e-300)).max().item())


CASES = [(1, 1, 1), (1, 7, 3), (5, 16, 64), (17, 33, 65), (40, 24, 301), (130, 40, 1003), (9, 64, 5000)]


@pytest.mark.parametrize("n,d,v", CASES)
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_loss_and_gradients_are_the_formula(n, d, v, reduction):
    x, w, t = case(n, d, v, seed=n, lean=3.0, ignored=range(1, n, 7), words=max(1, v // 5))
    up = torch.randn(n, generator=torch.Generator().manual_seed(1)) if reduction == "none" else None
    check(results(x, w, t, reduction, up), x, w, t, reduction=reduction, up=up)


@pytest.mark.parametrize("S", [1, 2, 3])
def test_slices(S):
    x, w, t = case(20, 30, 90, seed=S)
    check(results(x, w, t, slices=S), x, w, t, S=S)
    rg.set_slices(S)
    try:
        assert all(torch.equal(a, b) for a, b in zip(results(x, w, t), results(x, w, t, slices=S)))
    finally:
        rg.set_slices(3)


def test_sure_and_hopeless_tokens():
    """Probabilities of the target from 1 - 1e-9 down to e^-80."""
    x, w, t = case(12, 20, 50, seed=5)
    x = x * torch.linspace(0.1, 12, 12)[:, None]
    for words in ((x @ w.t()).argmax(1), (x @ w.t()).argmin(1)):
        check(results(x, w, words, "sum"), x, w, words, reduction="sum")


def test_a_group_of_tokens_and_more(monkeypatch):
    """More tokens than a group holds: the groups' shares of dw are added."""
    v = 2 ** 20 + 3
    group = _lib.lib.rg_loss_group_tokens(v)
    assert group == 128
    x, w, t = case(group + 5, 2, v, seed=2, std=1.0, words=40)
    loss, dx, dw = results(x, w, t)
    first, second = slice(0, group), slice(group, None)
    count = group + 5
    halves = [results(x[s], w, t[s], "none", torch.full((len(t[s]),), 1.0 / count)) for s in (first, second)]
    assert torch.equal(dx, torch.cat([h[1] for h in halves]))
    untouched = torch.ones(v, dtype=torch.bool)
    untouched[t] = False
    assert torch.equal(dw[untouched], (halves[0][2] + halves[1][2])[untouched])
    for a in (1, 64, 1003, 4096, 4097, 50257, 2 ** 30):
        r = _lib.lib.rg_loss_group_tokens(a)
        assert r & (r - 1) == 0 and 128 <= r <= 2048 and (r * a <= 2 ** 27 or r == 128)
    assert _lib.lib.rg_loss_group_tokens(0) == 0


def test_gradients_are_the_differences():
    """Along random directions of both inputs, in the sum of 30 tokens' losses (near 4 each, off by 2e-5 of
    the products' rounding): 2 x 30^0.5 x 2e-5 / 2h = 0.011 with h = 0.01; truncation h^2 / 6 x a third
    derivative under 300: 0.005."""
    x, w, t = case(30, 20, 60, seed=8)
    _, dx, dw = results(x, w, t, "sum")
    g = torch.Generator().manual_seed(3)
    ex, ew, h = torch.randn(30, 20, generator=g) / 5, torch.randn(60, 20, generator=g) / 5, 1e-2
    value = lambda s: rg.linear_cross_entropy(x + s * ex, w + s * ew, t, reduction="none").double().sum().item()  # noqa: E731
    slope = (dx.double() * ex.double()).sum().item() + (dw.double() * ew.double()).sum().item()
    assert abs((value(h) - value(-h)) / (2 * h) - slope) < 0.016


def test_tokens_that_do_not_count():
    x, w, t = case(9, 8, 20, seed=1)
    t[2], t[5] = -100, 7
    loss, dx, dw = results(x, w, t)
    keep = torch.arange(9) != 2
    part = results(x[keep], w, t[keep])
    assert torch.equal(loss, part[0]) and torch.equal(dx[keep], part[1]) and torch.equal(dx[2], torch.zeros(8))
    same = results(x, w, torch.where(t == -100, 7, t), ignore_index=7)  # 7 itself left out
    assert torch.equal(same[1][5], torch.zeros(8)) and torch.equal(same[1][2], torch.zeros(8))
    everything = torch.full((9,), -100)
    loss, dx, dw = results(x, w, everything)
    assert loss.isnan() and not dx.any() and not dw.any()
    loss, dx, dw = results(x, w, everything, "sum")
    assert loss == 0 and not dx.any() and not dw.any()
    rows, dx, dw = results(x, w, everything, "none")
    assert not rows.any() and not dx.any() and not dw.any()


@pytest.mark.parametrize("word", [-1, 20, 2 ** 40])
def test_targets_that_are_no_words(word):
    x, w, t = case(6, 8, 20, seed=4)
    clean = results(x, w, t, "none")
    t[3] = word
    rows, dx, dw = results(x, w, t, "none")
    keep = torch.arange(6) != 3
    assert rows[3].isnan() and torch.equal(rows[keep], clean[0][keep])
    assert torch.equal(dx[3], torch.zeros(8)) and torch.equal(dx[keep], clean[1][keep])
    assert torch.isfinite(dw).all()


def test_no_tokens():
    x, w, t = torch.zeros(0, 4), torch.randn(6, 4), torch.zeros(0, dtype=torch.int64)
    loss, dx, dw = results(x, w, t)
    assert loss.isnan() and dx.shape == (0, 4) and torch.equal(dw, torch.zeros(6, 4))
    assert results(x, w, t, "sum")[0] == 0 and results(x, w, t, "none")[0].shape == (0,)


def test_scaled_losses_second_backwards_and_frozen_inputs():
    x, w, t = case(12, 10, 30, seed=6)
    _, dx, dw = results(x, w, t)
    _, sx, sw = results(x, w, t, up=torch.tensor(0.3))
    assert torch.equal(sx, dx * torch.tensor(0.3)) and torch.equal(sw, dw * torch.tensor(0.3))
    x, w = x.requires_grad_(), w.requires_grad_()
    loss = rg.linear_cross_entropy(x, w, t)
    for factor in (2.0, 1.0, 0.5):
        got = torch.autograd.grad(loss, (x, w), torch.tensor(factor), retain_graph=True)
        assert torch.equal(got[0], dx * factor) and torch.equal(got[1], dw * factor)
    (only,) = torch.autograd.grad(rg.linear_cross_entropy(x, w.detach(), t), [x])
    assert torch.equal(only, dx)
    (only,) = torch.autograd.grad(rg.linear_cross_entropy(x.detach(), w, t), [w])
    assert torch.equal(only, dw)
    with torch.no_grad():
        assert torch.equal(rg.linear_cross_entropy(x, w, t), loss) and not rg.linear_cross_entropy(x, w, t).requires_grad


def test_shapes_and_strides():
    x, w, t = case(24, 10, 30, seed=7)
    want = results(x, w, t, "none")
    wide = torch.randn(30, 20)
    wide[:, ::2] = w
    got = results(x.view(4, 6, 10), wide[:, ::2], t.view(6, 4).t().contiguous().t().reshape(4, 6), "none",
                  torch.ones(4, 6))
    assert got[0].shape == (4, 6) and torch.equal(got[0].view(-1), want[0])
    assert torch.equal(got[1].view(24, 10), want[1]) and torch.equal(got[2], want[2])
    expanded = torch.tensor(2.0).expand(24)
    doubled = results(x, w, t, "none", expanded)
    assert torch.allclose(doubled[1], 2 * want[1], rtol=1e-5, atol=1e-7)


def test_refusals():
    x, w, t = case(6, 8, 20)
    f = rg.linear_cross_entropy
    for k, bad in enumerate([
            lambda: f(x, w, t, reduction="max"), lambda: f(x, w, t[:-1]), lambda: f(x, w, t.view(2, 3)),
            lambda: f(x, w[:, :-1], t), lambda: f(x, w[0], t), lambda: f(x.double(), w, t), lambda: f(x, w.half(), t),
            lambda: f(x, w, t.int()), lambda: f(x, w, t, slices=0), lambda: f(x, w, t, slices=4),
            lambda: f(x[:, :0], w[:, :0], t), lambda: f(x, w[:0], t), lambda: f(x, w.to("meta"), t),
            lambda: f(torch.tensor(1.0), w, torch.tensor(1)), lambda: rg.LinearCrossEntropy(8, 20, reduction="max")]):
        with pytest.raises(ValueError):
            bad()
            pytest.fail("case %d" % k)


def test_c_entry_refuses_bad_arguments():
    lib, bad = _lib.lib, _lib.HIP_ERROR_INVALID_VALUE
    c = _lib.rg_loss_config()
    lib.rg_loss_config_init(ctypes.byref(c))
    assert (c.N, c.D, c.V, c.slices, c.reduction, c.ignore_index) == (0, 0, 0, 3, 0, -100)

    def config(**k):
        return _lib.rg_loss_config(**{**dict(N=4, D=8, V=9, slices=3, reduction=0, ignore_index=-100), **k})

    p, size = 4096, ctypes.c_size_t()
    for broken in (dict(N=-1), dict(N=2 ** 31), dict(D=0), dict(V=0), dict(slices=0), dict(slices=4), dict(reduction=3), dict(reduction=-1)):
        assert lib.rg_linear_cross_entropy_workspace(ctypes.byref(config(**broken)), 1, 1, ctypes.byref(size)) == bad
        assert lib.rg_linear_cross_entropy(ctypes.byref(config(**broken)), p, p, p, None, p, p, p, p, 1 << 40, None) == bad
    assert lib.rg_linear_cross_entropy_workspace(None, 1, 1, ctypes.byref(size)) == bad
    assert lib.rg_linear_cross_entropy_workspace(ctypes.byref(config()), 1, 1, None) == bad
    assert lib.rg_linear_cross_entropy(ctypes.byref(config(N=0)), None, None, None, None, None, None, None, None, 0, None) == 0
    for i in range(3):
        args = [p, p, p]
        args[i] = None
        assert lib.rg_linear_cross_entropy(ctypes.byref(config()), *args, None, p, p, p, p, 1 << 40, None) == bad
    for i in range(7):
        args = [p, p, p, p, p, p, p]
        args[i] = p + 2
        assert lib.rg_linear_cross_entropy(ctypes.byref(config()), *args, p, 1 << 40, None) == bad
    assert lib.rg_scale_fp32(None, 4, None, 0, p, None) == bad and lib.rg_scale_fp32(p, 4, p, 4, None, None) == bad
    assert lib.rg_scale_fp32(None, 0, None, 0, None, None) == 0


def test_module_reports_to_the_guard():
    rg.guard().reset()
    torch.manual_seed(0)
    m = rg.LinearCrossEntropy(8, 20)
    holder = torch.nn.ModuleDict({"head": m})
    rg.name_layers(holder)
    x, t = torch.randn(5, 8), torch.randint(0, 20, (5,))
    assert torch.equal(m(x, t), rg.linear_cross_entropy(x, m.weight, t)) and rg.guard().first_offender() is None
    x[2, 2] = math.nan
    m(x, t)
    assert rg.guard().first_offender() == "head input"
    rg.guard().reset()


def test_gradients_are_differentiable_no_further():
    x, w, t = case(6, 8, 20)
    x.requires_grad_()
    loss = rg.linear_cross_entropy(x, w, t)
    (dx,) = torch.autograd.grad(loss, [x], create_graph=True)
    assert torch.equal(dx, results(x, w, t)[1])
    with pytest.raises(RuntimeError, match="only once"):
        dx.sum().backward()


def test_backward_passes_of_several_threads():
    """The binding's backward passes run with and without the interpreter's lock."""
    import threading

    x, w, t = case(40, 16, 300, seed=3)
    want = results(x, w, t)
    got = [None] * 4

    def work(i):
        got[i] = results(x, w, t)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))


def words_past_the_range(n, below, above):
    """One value a row, so every finite logit is exact: `below` words whose logits are -infinity (products below
    float32's range), ten of -1 to 1.25, and `above` more of -infinity. (x, w, t, the first finite word)"""
    c = torch.arange(10) / 4.0 - 1.0
    lost = torch.tensor([-2.0 ** 70])
    w = torch.cat([lost.expand(below), c * 2.0 ** -70, lost.expand(above)])[:, None].contiguous()
    x = torch.full((n, 1), 2.0 ** 70)
    return x, w, below + torch.arange(n) % 10, below


@pytest.mark.parametrize("below,above", [(0, 64), (63, 0), (64, 0), (64, 64), (128, 5), (54, 300), (4096, 0)])
@pytest.mark.parametrize("n", [1, 3])
def test_parts_whose_logits_are_all_minus_infinity(n, below, above):
    """They have no share: the softmax is that of the ten words. Exponentials, sums and the quotient: 24 and 6
    roundings relative to a probability, as in bounds(); a word's row of dz is rounded at half a step of its largest value."""
    x, w, t, first = words_past_the_range(n, below, above)
    rows, _, dw = results(x, w, t, "none")
    z = torch.arange(10, dtype=torch.float64) / 4 - 1
    lse = torch.logsumexp(z, 0)
    want = lse - z[t - first]
    assert torch.all((rows.double() - want).abs() <= 24 * EPS32 + 2 * EPS32 * want)
    p = torch.exp(z - lse)
    counts = torch.bincount(t - first, minlength=10)
    want = (p * n - counts) * 2.0 ** 70
    got = dw[first:first + 10, 0].double()
    assert torch.all((got - want).abs() <= 2.0 ** 70 * (n * p * (40 * EPS32 + step(1.0, 3)) + 8 * EPS32 * counts))
    assert not dw[:first].any() and not dw[first + 10:].any()


def test_targets_and_rows_of_minus_infinity():
    x, w, t, first = words_past_the_range(2, 64, 3)
    rows, dx, dw = results(x, w, torch.tensor([0, first]), "none")  # a target of probability 0, and an ordinary one
    assert rows[0] == math.inf and torch.isfinite(rows[1]) and torch.isfinite(dw).all() and torch.isfinite(dx).all()
    rows, dx, dw = results(x, w[:64], torch.tensor([0, 1]), "none")  # no word has a probability
    assert rows.isnan().all() and dx.isnan().all() and dw[:2].isnan().all()
    rows, _, _ = results(x, -w, torch.tensor([first, 0]), "none")  # +infinity
    assert rows.isnan().all()


@pytest.mark.parametrize("large", [1e12, -3e38, math.inf, math.nan])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_hidden_states_of_tokens_that_do_not_count_reach_nothing(large, reduction):
    """Padding may hold anything: of tokens that are left out, whose target is no word, or whose finite loss has a factor
    of 0, nothing reaches the others' gradients. Without them the results are the same bits."""
    x, w, t = case(30, 12, 50, seed=11, lean=2.0)
    up = torch.randn(30, generator=torch.Generator().manual_seed(2))
    keep = torch.ones(30, dtype=torch.bool)
    keep[[0, 7, 8, 29]] = False
    part = results(x[keep], w, t[keep], reduction, up[keep] if reduction == "none" else None)
    t[~keep] = -100
    if reduction == "none":
        t[7] = 50
        if large == 1e12:
            t[8], up[8] = 3, 0.0
    x[~keep, ::2] = large
    got = results(x, w, t, reduction, up if reduction == "none" else None)
    assert torch.equal(got[2], part[2]) and torch.equal(got[1][keep], part[1])
    if math.isfinite(large):
        assert not got[1][~keep].any()
    assert torch.equal(got[0], part[0]) if reduction == "mean" else torch.equal(got[0][keep], part[0])


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_a_nan_or_infinity_in_x_reaches_its_token(bad, reduction):
    """Its loss, its row of dx and its target's row of dw are NaN; the other tokens' are those of a call without it."""
    x, w, t = case(17, 12, 40, seed=12, lean=2.0)
    t[5] = 39
    t[t == 39] = 38
    t[5] = 39  # no other token's target
    keep = torch.arange(17) != 5
    up = torch.ones(17)
    part = results(x[keep], w, t[keep], "none")
    x[5, 3] = bad
    loss, dx, dw = results(x, w, t, reduction, up if reduction == "none" else torch.tensor(17.0))
    assert loss.isnan() if reduction == "mean" else loss[5].isnan() and torch.equal(loss[keep], part[0])
    assert dx[5].isnan().all() and dw[39].isnan().all()
    if reduction == "none":
        assert torch.equal(dx[keep], part[1]) and torch.equal(dw[:39], part[2][:39])
    else:
        assert torch.isfinite(dx[keep]).all() and torch.isfinite(dw[:39]).all()


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_a_nan_or_infinity_in_the_weight_reaches_every_token(bad):
    x, w, t = case(9, 12, 40, seed=13)
    t[t == 30] = 3
    t[4] = -100
    w[30, 11] = bad  # a word that is no token's target
    keep = torch.arange(9) != 4
    rows, dx, dw = results(x, w, t, "none")
    assert rows[keep].isnan().all() and rows[4] == 0
    assert dx[keep].isnan().all() and not dx[4].any() and dw[t[keep]].isnan().all()
    assert results(x, w, t, "sum")[0].isnan()


@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_the_guard_hears_a_gradient_that_is_not_finite(reduction):
    rg.guard().reset()
    torch.manual_seed(0)
    m = rg.LinearCrossEntropy(8, 20, reduction=reduction)
    m.repro_name = "top"
    x, t = torch.randn(5, 8), torch.randint(0, 20, (5,))
    loss = m(x, t)
    up = torch.ones_like(loss)
    (clean,) = torch.autograd.grad(loss, m.weight, up, retain_graph=True)
    rg.guard().check()
    assert torch.equal(clean, results(x, m.weight, t, reduction)[2])
    up.view(-1)[-1] = math.inf
    torch.autograd.grad(loss, m.weight, up)
    assert rg.guard().first_offender() == "top gradient"
    rg.guard().reset()


def test_more_words_than_launches_take_are_refused():
    """A launch has fewer than 2^32 threads, and slicing takes 64 a word."""
    words = 2 ** 25
    assert 64 * words < 2 ** 32
    c, size = _lib.rg_loss_config(N=4, D=300, V=words + 1, slices=3, reduction=0, ignore_index=-100), ctypes.c_size_t()
    assert _lib.lib.rg_linear_cross_entropy_workspace(ctypes.byref(c), 0, 1, ctypes.byref(size)) == _lib.HIP_ERROR_INVALID_VALUE
    with pytest.raises(ValueError, match="too many"):
        rg.linear_cross_entropy(torch.zeros(2, 1), torch.zeros(1, 1).expand(words + 1, 1), torch.zeros(2, dtype=torch.int64))
