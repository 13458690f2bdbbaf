"""The AdamW step against the formula in 64 bits, its 8-bit moments against their definition, its
refusals, and the optimizer, on the CPU."""
import ctypes
import math

import pytest
import torch

import bit_reproducible_training_amd as rg
from bit_reproducible_training_amd import _lib

EPS32 = 2.0 ** -24
SETTINGS = dict(lr=2e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.05)


def tensors(sizes, seed, device="cpu"):
    g = torch.Generator().manual_seed(seed)
    p = [torch.randn(s, generator=g) for s in sizes]
    grad = [torch.randn(s, generator=g) * 10.0 ** torch.randint(-6, 2, (1,), generator=g).item() for s in sizes]
    m = [0.1 * torch.randn(s, generator=g) for s in sizes]
    v = [0.01 * torch.rand(s, generator=g) for s in sizes]
    return tuple([t.to(device) for t in ts] for ts in (p, grad, m, v))


def exact(p, g, m, v, step, lr, betas, eps, weight_decay):
    """The step in 64 bits: (p, m, v, the update's magnitude)."""
    p, g, m, v = (t.detach().cpu().double() for t in (p, g, m, v))
    b1, b2 = betas
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    update = lr * (m / (1 - b1 ** step)) / ((v / (1 - b2 ** step)).sqrt() + eps)
    return p * (1 - lr * weight_decay) - update, m, v, update.abs()


def check_step(before, after, step, settings):
    """Each rounding is 2^-24 of its result: m and v see two products, their constants' rounding and
    one addition (4 of them cover it); the update sees m's and half of v's, and the root, two products
    with constants, one addition, a division and a product: 16; p its own product and difference: 4.
    m's relative error is that of its two terms' magnitudes, which cancel at most to m."""
    for i in range(len(before[0])):
        p0, g, m0, v0 = (t[i] for t in before)
        p1, m1, v1 = (t[i].detach().cpu().double() for t in after)
        p, m, v, update = exact(p0, g, m0, v0, step, **settings)
        b1, b2 = settings["betas"]
        scale_m = b1 * m0.detach().cpu().double().abs() + (1 - b1) * g.detach().cpu().double().abs()
        assert torch.all((m1 - m).abs() <= 4 * EPS32 * scale_m + 2.0 ** -148)
        assert torch.all((v1 - v).abs() <= 4 * EPS32 * v + 2.0 ** -147)
        lost = scale_m / m.abs().clamp(min=1e-300)
        assert torch.all((p1 - p).abs() <= EPS32 * (4 * p0.detach().cpu().double().abs() + update * (16 + 4 * lost)) + 2.0 ** -148)


@pytest.mark.parametrize("step", [1, 2, 1000, 10 ** 9])
def test_step_is_the_formula(step):
    before = tensors([(1,), (3, 5), (255,), (256,), (4097,), (0,)], step % 97)
    p, g, m, v = ([t.clone() for t in ts] for ts in before)
    rg.adamw_step(p, g, m, v, step=step, **SETTINGS)
    check_step(before, (p, m, v), step, SETTINGS)
    assert all(torch.equal(a, b) for a, b in zip(g, before[1]))


def test_zero_gradient_from_the_start_only_decays():
    p = [torch.randn(300)]
    want = p[0] * torch.tensor(1 - 1e-2 * 0.5, dtype=torch.float32)
    zero = [torch.zeros(300)]
    rg.adamw_step(p, zero, [torch.zeros(300)], [torch.zeros(300)], step=1, lr=1e-2, weight_decay=0.5)
    assert torch.equal(p[0], want)


def test_nan_and_infinity_stay_with_their_value():
    p, g, m, v = tensors([(600,)], 3)
    g[0][7], g[0][301] = math.nan, math.inf
    want = exact(p[0], g[0], m[0], v[0], 1, **SETTINGS)[0]
    rg.adamw_step(p, g, m, v, step=1, **SETTINGS)
    bad = torch.zeros(600, dtype=torch.bool)
    bad[[7, 301]] = True
    assert torch.equal(p[0].isnan(), bad) and torch.isfinite(want[~bad]).all()


# ---- the 8-bit moments ----


def test_codes_of_every_exponent_decode_to_their_definition():
    codes = torch.arange(256, dtype=torch.uint8)
    for e in (34, 100, 127, 200, 254):
        exps = torch.tensor([e], dtype=torch.uint8)
        m, v = rg.adamw8_values(codes, exps, codes, exps)
        for c in range(256):
            a = c & 127
            want_m = a * 2.0 ** (e - 14 - 130) if a < 8 else (8 + a % 8) * 2.0 ** (e - 14 - 130 + a // 8 - 1)
            want_v = c * 2.0 ** (e - 30 - 130) if c < 8 else (8 + c % 8) * 2.0 ** (e - 30 - 130 + c // 8 - 1)
            assert m[c].item() == (-want_m if c >= 128 else want_m)
            assert v[c].item() == want_v


def quantum(a, e, span):
    """The spacing of the codes at magnitudes a in a block of exponent field e."""
    own = torch.floor(torch.log2(a.clamp(min=1e-300))) + 127
    return 2.0 ** (torch.maximum(own, torch.as_tensor(float(e - span))) - 130)


def test_moments_are_the_two_codes_next_to_their_value():
    p, g, m, v = tensors([(700,)], 11)
    p0, g0 = p[0].clone(), g[0].clone()
    state = rg.adamw8_state(p)
    step_m, step_v = (1 - 0.9) * g0.double(), (1 - 0.99) * g0.double() ** 2
    rg.adamw8_step(p, g, *state, step=1, **SETTINGS)
    got_m, got_v = rg.adamw8_values(*state)
    for b in range(3):
        at = slice(256 * b, min(700, 256 * (b + 1)))
        for got, want, e, span in ((got_m[at], step_m[at], state[1][b].item(), 14),
                                   (got_v[at], step_v[at], state[3][b].item(), 30)):
            assert e == int(math.floor(math.log2(want.abs().max().item() * 16 / 15))) + 127
            assert torch.all((got.double() - want).abs() <= quantum(want.abs(), e, span) * (1 + 1e-6))
            assert torch.all((got == 0) | (got.sign() == want.sign()))
    assert torch.all(got_v[:700][g0 != 0] > 0)
    assert torch.all(got_m[700:] == 0) and torch.all(got_v[700:] == 0) and torch.all(state[0][700:] == 0)
    want = exact(p0, g0, torch.zeros(700), torch.zeros(700), 1, **SETTINGS)
    assert torch.all((p[0].double() - want[0]).abs() <= EPS32 * (4 * p0.abs() + 20 * want[3]))


def test_rounding_of_the_moments_has_their_mean():
    """The second moment of a constant gradient from zero is g^2 (1 - b2^t). With rounding to nearest
    it would stop at the code where (1 - b2) g^2 is under half a code. Its steps' rounding errors are
    independent with zero mean, each at most one code (1/8 of the value), and decay with b2: the
    relative standard deviation is at most 1/8 / sqrt(1 - b2^2) = 0.89 per value, so 0.056 of the mean
    over 256 values; four of those are allowed."""
    n, b2 = 256, 0.99
    p, g = [torch.zeros(n)], [torch.full((n,), 0.5)]
    state = rg.adamw8_state(p)
    for step in range(1, 301):
        rg.adamw8_step(p, g, *state, step=step, lr=0.0, betas=(0.9, b2))
    m, v = rg.adamw8_values(*state)
    want = 0.25 * (1 - b2 ** 300)
    assert abs(v.double().mean().item() / want - 1) < 4 * 0.056
    assert abs(m.double().mean().item() / 0.5 - 1) < 4 * 0.125 / math.sqrt(1 - 0.81) / 16


def test_small_values_beside_large_ones_take_bounded_steps():
    """A value far below its block's largest keeps a positive second moment, so its step stays near lr."""
    n = 256
    p = [torch.zeros(n)]
    g = [torch.full((n,), 1e-7)]
    g[0][0] = 10.0
    state = rg.adamw8_state(p)
    for step in range(1, 20):
        before = p[0].clone()
        rg.adamw8_step(p, g, *state, step=step, lr=1e-3, weight_decay=0.0)
        # m's smallest code is 2^-17 of the largest's binade, v's 2^-33: a quotient of at most 2,
        # times the two corrections' sqrt(1 - b2^t) / (1 - b1^t), at most 1
        assert (p[0] - before).abs().max().item() <= 4e-3


def test_non_finite_moments_count_as_the_largest_finite_value():
    p, g = [torch.zeros(256)], [torch.zeros(256)]
    g[0][3] = math.nan
    state = rg.adamw8_state(p)
    rg.adamw8_step(p, g, *state, step=1)
    m, v = rg.adamw8_values(*state)
    assert p[0].isnan().sum() == 1 and torch.isfinite(m).all() and torch.isfinite(v).all()


def test_flat_and_listed_moments_are_the_same():
    sizes = [(5,), (256,), (3, 100), (1,)]
    p, g, _, _ = tensors(sizes, 4)
    q = [t.clone() for t in p]
    flat = rg.adamw8_state(p)
    listed = [rg.adamw8_state([t]) for t in p]
    for step in (1, 2, 3):
        rg.adamw8_step(p, g, *flat, step=step)
        rg.adamw8_step(q, g, *([s[k] for s in listed] for k in range(4)), step=step)
    assert all(torch.equal(a, b) for a, b in zip(p, q))
    for k in range(4):
        assert torch.equal(flat[k], torch.cat([s[k] for s in listed]))


# ---- refusals ----


def one(n=8):
    return [torch.zeros(n)]


@pytest.mark.parametrize("change", [
    dict(step=0), dict(lr=-1.0), dict(lr=math.nan), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)),
    dict(eps=-1.0), dict(weight_decay=-0.1)])
def test_settings_that_are_refused(change):
    settings = {"step": 1, **change}
    with pytest.raises(ValueError):
        rg.adamw_step(one(), one(), one(), one(), **settings)
    with pytest.raises(ValueError):
        rg.adamw8_step(one(), one(), *rg.adamw8_state(one()), **settings)


def test_tensors_that_are_refused():
    base = torch.zeros(4, 6)
    for p, g, m, v in [
        (one(), one(7), one(), one()), (one(), one(), one(9), one()), (one(), one(), one(), []),
        (one(), [], one(), one()), ([torch.zeros(8).double()], one(), one(), one()),
        (one(), [torch.zeros(8, dtype=torch.float16)], one(), one()),
        ([base[:, ::2]], [base[:, ::2]], [base[:, ::2]], [base[:, ::2]]),      # gaps
        ([torch.zeros(4, 6).t()], [torch.zeros(6, 4)], [torch.zeros(6, 4)], [torch.zeros(6, 4)]),  # other strides
        (one(), [torch._neg_view(torch.zeros(8))], one(), one()),
    ]:
        with pytest.raises(ValueError):
            rg.adamw_step(p, g, m, v, step=1)
    good = rg.adamw8_state(one(300))
    for k in range(4):
        for wrong in (good[k][:-1], good[k].to(torch.int8), torch.zeros(2 * good[k].numel(), dtype=torch.uint8)[::2]):
            state = list(good)
            state[k] = wrong
            with pytest.raises(ValueError):
                rg.adamw8_step(one(300), one(300), *state, step=1)
    with pytest.raises(ValueError):
        rg.adamw8_step(one(300), one(300), [good[0]], *good[1:], step=1)


def test_c_entry_refuses_bad_lists():
    lib = _lib.lib
    cfg = _lib.rg_adamw_config()
    lib.rg_adamw_config_init(ctypes.byref(cfg))
    assert (cfg.lr, cfg.beta1, cfg.beta2, cfg.eps, cfg.weight_decay, cfg.step) == (1e-3, 0.9, 0.999, 1e-8, 1e-2, 1)
    bad = _lib.HIP_ERROR_INVALID_VALUE
    t = (_lib.rg_adamw_tensor * 1)(_lib.rg_adamw_tensor(4096, 4096, 4096, 4096, -1))
    t8 = (_lib.rg_adamw8_tensor * 1)(_lib.rg_adamw8_tensor(4096, 4096, 4098, 4096, 4096, 4096, 5))
    null = (_lib.rg_adamw_tensor * 1)(_lib.rg_adamw_tensor(4096, 4096, None, 4096, 4))
    odd = (_lib.rg_adamw_tensor * 1)(_lib.rg_adamw_tensor(4097, 4096, 4096, 4096, 4))
    for tensors_, count in ((t, 1), (null, 1), (odd, 1), (t, -1), (None, 1)):
        assert lib.rg_adamw_fp32(tensors_, count, ctypes.byref(cfg), None) == bad
    assert lib.rg_adamw8_fp32(t8, 1, ctypes.byref(cfg), None) == bad
    assert lib.rg_adamw_fp32(None, 0, None, None) == bad
    assert lib.rg_adamw_fp32(None, 0, ctypes.byref(cfg), None) == 0  # nothing to do
    assert lib.rg_adamw8_values(None, None, None, None, None, None, 1, None) == bad
    assert lib.rg_adamw8_values(None, None, None, None, None, None, 0, None) == 0


# ---- the optimizer ----


@pytest.mark.parametrize("bits", [8, 32])
def test_optimizer_takes_the_steps(bits):
    torch.manual_seed(1)
    shapes = [(7, 9), (9,), (300,), (4, 6)]
    p = [torch.nn.Parameter(torch.randn(s)) for s in shapes]
    p[3] = torch.nn.Parameter(torch.randn(6, 4).t())  # dense, not contiguous
    q = [t.detach().clone() for t in p]
    opt = rg.AdamW([{"params": p[:2], "lr": 0.01}, {"params": p[2:], "weight_decay": 0.0}], lr=0.02, state_bits=bits)
    states = [rg.adamw8_state([t]) if bits == 8 else (torch.zeros_like(t), torch.zeros_like(t)) for t in q]
    counts = [0] * 4
    for it in range(4):
        for t in p:
            t.grad = torch.randn(t.shape)
        if it == 1:
            p[1].grad = None
        grads = [t.grad for t in p]
        opt.step()
        for group, lr, wd in (((0, 1), 0.01, 1e-2), ((2, 3), 0.02, 0.0)):
            batches = {}
            for i in group:
                if grads[i] is not None:
                    counts[i] += 1
                    batches.setdefault(counts[i], []).append(i)
            for step, held in batches.items():
                gs = [torch.empty_like(q[i]).copy_(grads[i]) for i in held]
                ps = [q[i] for i in held]
                settings = dict(step=step, lr=lr, weight_decay=wd)
                if bits == 8:
                    rg.adamw8_step(ps, gs, *([states[i][k] for i in held] for k in range(4)), **settings)
                else:
                    rg.adamw_step(ps, gs, [states[i][0] for i in held], [states[i][1] for i in held], **settings)
    assert all(torch.equal(a, b) for a, b in zip(p, q))


@pytest.mark.parametrize("bits", [8, 32])
def test_optimizer_resumes_from_its_state(bits, tmp_path):
    def model():
        torch.manual_seed(5)
        return [torch.nn.Parameter(torch.randn(500)), torch.nn.Parameter(torch.randn(3, 7))]

    def train(p, opt, steps):
        for s in steps:
            g = torch.Generator().manual_seed(s)
            for t in p:
                t.grad = torch.randn(t.shape, generator=g)
            opt.step()

    p = model()
    opt = rg.AdamW(p, state_bits=bits)
    train(p, opt, range(3))
    torch.save({"opt": opt.state_dict(), "p": [t.detach() for t in p]}, tmp_path / "s.pt")
    train(p, opt, range(3, 6))
    saved = torch.load(tmp_path / "s.pt", weights_only=True)
    q = [torch.nn.Parameter(t) for t in saved["p"]]
    again = rg.AdamW(q, state_bits=bits)
    again.load_state_dict(saved["opt"])
    train(q, again, range(3, 6))
    assert all(torch.equal(a, b) for a, b in zip(p, q))


def test_optimizer_refuses_bad_settings():
    p = [torch.nn.Parameter(torch.zeros(3))]
    for bad in (dict(lr=-1.0), dict(eps=-1.0), dict(weight_decay=-1.0), dict(betas=(0.9, 1.0)), dict(state_bits=16)):
        with pytest.raises(ValueError):
            rg.AdamW(p, **bad)


@pytest.mark.parametrize("bits", [8, 32])
def test_a_step_is_a_change_that_autograd_sees(bits):
    p = torch.nn.Parameter(torch.randn(5))
    opt = rg.AdamW([p], state_bits=bits)
    loss = (p * p).sum()
    loss.backward(retain_graph=True)
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.parametrize("bits", [8, 32])
def test_a_refused_step_is_not_counted(bits):
    import copy

    p = [torch.nn.Parameter(torch.randn(5)), torch.nn.Parameter(torch.randn(6))]
    opt = rg.AdamW(p, state_bits=bits)
    for t in p:
        t.grad = torch.randn(t.shape)
    opt.step()
    before = [t.detach().clone() for t in p]
    opt.param_groups[0]["lr"] = -1.0
    with pytest.raises(ValueError):
        opt.step()
    assert [opt.state[t]["step"] for t in p] == [1, 1] and all(torch.equal(a, b) for a, b in zip(before, p))
    opt.param_groups[0]["lr"] = 1e-3
    again = [torch.nn.Parameter(t) for t in before]
    other = rg.AdamW(again, state_bits=bits)
    other.load_state_dict(copy.deepcopy(opt.state_dict()))  # (float32 moments would be shared)
    for t, q in zip(p, again):
        q.grad = t.grad
    opt.step()
    other.step()
    assert all(torch.equal(a, b) for a, b in zip(p, again)) and opt.state[p[0]]["step"] == 2


@pytest.mark.filterwarnings("ignore:optimizer contains a parameter group with duplicate")
def test_a_parameter_that_is_listed_twice_takes_two_steps():
    p, q = torch.nn.Parameter(torch.randn(9)), None
    q = torch.nn.Parameter(p.detach().clone())
    p.grad = q.grad = torch.randn(9)
    twice, once = rg.AdamW([p, p]), rg.AdamW([q])
    twice.step()
    once.step()
    once.step()
    assert torch.equal(p, q) and twice.state[p]["step"] == 2


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_tensors_of_a_step_that_overlap_are_refused(device):
    """Values that two threads of a launch would read and write."""
    new = lambda n=600: torch.zeros(n, device=device)  # noqa: E731
    z, flat = new(), new(1000)
    for p, m, v in [([z, z], [new(), new()], [new(), new()]), ([new(), new()], [z, z], [new(), new()]),
                    ([new(), new()], [new(), new()], [z, z]), ([new()], [z], [z]), ([z], [z], [new()]), ([z], [new()], [z]),
                    ([flat[400:], flat[:600], new()], [new(), new(), new()], [new(), new(), new()][:3])]:
        p = [t[:600] for t in p]
        with pytest.raises(ValueError, match="overlap"):
            rg.adamw_step(p, [torch.ones_like(t) for t in p], m, v, step=1)
    apart = [flat[400:], new(0), flat[:400]]  # in no order, and an empty one
    rg.adamw_step(apart, *([torch.zeros_like(t) for t in apart] for _ in range(3)), step=1)
    with pytest.raises(ValueError, match="overlap"):
        rg.adamw8_step([z, z], [new(), new()], *rg.adamw8_state([z, z]), step=1)
    state = rg.adamw8_state([z])
    for k in range(4):
        states = [[s, s if i == k else s.clone()] for i, s in enumerate(state)]
        with pytest.raises(ValueError, match="overlap"):
            rg.adamw8_step([new(), new()], [new(), new()], *states, step=1)
    rg.adamw8_step([new(), new()], [z, z], *([s, s.clone()] for s in state), step=1)  # gradients are only read


def test_a_state_of_torchs_adamw_is_taken_up():
    """Its steps go on: against torch's own from the same state, within the roundings of two more steps of each (16 and 4
    as in check_step, twice, for both)."""
    import copy

    torch.manual_seed(2)
    p = [torch.nn.Parameter(torch.randn(40)), torch.nn.Parameter(torch.randn(3, 5))]
    theirs = torch.optim.AdamW(p, lr=1e-2, betas=(0.9, 0.98), weight_decay=0.1)
    grads = [[torch.randn(t.shape) for t in p] for _ in range(5)]
    for g in grads[:3]:
        for t, v in zip(p, g):
            t.grad = v
        theirs.step()
    q = [torch.nn.Parameter(t.detach().clone()) for t in p]
    ours = rg.AdamW(q, state_bits=8)
    ours.load_state_dict(copy.deepcopy(theirs.state_dict()))
    for g in grads[3:]:
        for a, b, v in zip(p, q, g):
            a.grad, b.grad = v, v.clone()
        theirs.step()
        ours.step()
    for a, b in zip(p, q):
        assert torch.all((a.double() - b.double()).abs() <= 2 * 2 * EPS32 * (4 * a.detach().double().abs() + 20 * 2 * 1e-2))
    assert all(int(ours.state[t]["step"]) == 5 and ours.state[t]["exp_avg"].dtype == torch.float32 for t in q)
    for unknown in (dict(amsgrad=True), dict(maximize=True)):
        state = torch.optim.AdamW([torch.nn.Parameter(torch.zeros(2))], **unknown).state_dict()
        with pytest.raises(ValueError):
            rg.AdamW([torch.nn.Parameter(torch.zeros(2))]).load_state_dict(state)
