"""The residual norm and its gradients against the formula in 64 bits and against differences, and its
refusals, on the CPU."""
import ctypes
import math

import pytest
import torch

import bit_reproducible_training_amd as rg
from bit_reproducible_training_amd import _lib

EPS32 = 2.0 ** -24
NAMES = ("x", "f", "gate", "weight", "bias", "post_weight", "post_bias")


def case(n, d, kind="layer", gate=None, post=False, seed=0, scale=0.5, offset=0.0, device="cpu"):
    """gate: None or its rows. A dict of the call's tensors (None where absent) and settings."""
    g = torch.Generator().manual_seed(seed)
    layer = kind == "layer"
    t = {"x": 2 * torch.randn(n, d, generator=g) + offset, "f": torch.randn(n, d, generator=g),
         "gate": None if gate is None else torch.randn(gate, d, generator=g),
         "weight": torch.randn(d, generator=g), "bias": torch.randn(d, generator=g) if layer else None,
         "post_weight": torch.randn(d, generator=g) if post else None,
         "post_bias": torch.randn(d, generator=g) if post and layer else None}
    t = {k: None if v is None else v.to(device) for k, v in t.items()}
    up = [torch.randn(n, d, generator=g).to(device) for _ in range(2)]
    return t, dict(kind=kind, scale=scale, post_norm=post), up


def call(t, settings):
    return rg.residual_norm(t["x"], t["f"], t["weight"], t["bias"], gate=t["gate"], post_weight=t["post_weight"],
                            post_bias=t["post_bias"], **settings)


def gradients(t, settings, up):
    """{r, y, d...} of the call."""
    t = {k: None if v is None else v.detach().requires_grad_() for k, v in t.items()}
    r, y = call(t, settings)
    held = [k for k in NAMES if t[k] is not None]
    grads = torch.autograd.grad((r, y), [t[k] for k in held], up)
    return {"r": r.detach(), "y": y.detach(), **{"d" + k: g for k, g in zip(held, grads)}}


def exact(t, settings, up, eps=1e-5):
    """The same in 64 bits on the CPU, and for each result the magnitude its roundings are relative to:
    the sum of the magnitudes that it is added up from, times how the norms amplify an error of their
    input (1 + largest value over deviation)."""
    t = {k: None if v is None else v.detach().cpu().double().requires_grad_() for k, v in t.items()}
    dr, dy = (u.cpu().double() for u in up)
    n, d = t["x"].shape
    layer = settings["kind"] == "layer"

    def parts(v):
        c = v - v.mean(1, keepdim=True) if layer else v
        rstd = 1.0 / (c.square().mean(1, keepdim=True) + eps).sqrt()
        return c * rstd, rstd, 1.0 + (v.abs().amax(1, keepdim=True) * rstd)

    u, k_f = t["f"], torch.ones(n, 1, dtype=torch.float64)
    f_hat = f_rstd = None
    if settings["post_norm"]:
        f_hat, f_rstd, k_f = parts(t["f"])
        u = f_hat * t["post_weight"] + (t["post_bias"] if layer else 0.0)
    gate = None if t["gate"] is None else t["gate"].repeat_interleave(n // t["gate"].shape[0], 0)
    gu = u if gate is None else u * gate
    r = t["x"] + settings["scale"] * gu
    hat, rstd, k_r = parts(r)
    y = hat * t["weight"] + (t["bias"] if layer else 0.0)
    held = [k for k in NAMES if t[k] is not None]
    grads = torch.autograd.grad((r, y), [t[k] for k in held], (dr, dy))
    out = {"r": r, "y": y, **{"d" + k: g for k, g in zip(held, grads)}}
    with torch.no_grad():
        k = k_r * k_f
        # the row's largest normalised value and branch, which errors of the statistics multiply
        top = lambda a: a.abs().amax(1, keepdim=True)  # noqa: E731
        branch = settings["scale"] * ((1 if gate is None else gate.abs()) * (u.abs() + (0 if not settings["post_norm"] else t["post_weight"].abs() * (1 + top(f_hat))) * k_f))
        size = {"r": t["x"].abs() + branch, "y": (hat.abs() + 1 + (t["x"].abs() + branch) * rstd) * t["weight"].abs() * k + (t["bias"].abs() if layer else 0.0)}
        a = (dy * t["weight"]).abs()
        dx = dr.abs() + rstd * (a + a.mean(1, keepdim=True) + (hat.abs() + 1) * (a * (hat.abs() + 1)).mean(1, keepdim=True)) * k
        size["dx"] = dx
        size["dweight"] = (dy.abs() * (hat.abs() + 1 + (t["x"].abs() + branch) * rstd) * k).sum(0)
        if layer:
            size["dbias"] = dy.abs().sum(0)
        db = settings["scale"] * dx
        if gate is not None:
            by_row = db * (u.abs() + 1) * k
            size["dgate"] = by_row.view(t["gate"].shape[0], -1, d).sum(1)
            db = db * gate.abs()
        if settings["post_norm"]:
            size["dpost_weight"] = (db * (f_hat.abs() + 1) * k).sum(0)
            if layer:
                size["dpost_bias"] = db.sum(0)
            b = db * t["post_weight"].abs()
            db = f_rstd * (b + b.mean(1, keepdim=True) + (f_hat.abs() + 1) * (b * (f_hat.abs() + 1)).mean(1, keepdim=True)) * k
        size["df"] = db
    return {k: v.detach() for k, v in out.items()}, size


def check(got, t, settings, up):
    """A value passes through at most about 20 roundings of its own and two nested row sums (each a tree
    of 4 + 10 levels); a column sum through its strand's rows and a tree of at most 50 more. 64 and 64 +
    rows a strand of 2^-24 of the magnitudes cover them."""
    want, size = exact(t, settings, up)
    rows = max(4, -(-t["x"].shape[0] // 512))
    for k, w in want.items():
        steps = 64 + (rows + 50 if k in ("dweight", "dbias", "dgate", "dpost_weight", "dpost_bias") else 0)
        off = (got[k].cpu().double() - w).abs()
        assert torch.all(off <= steps * EPS32 * size[k] + 1e-37), (k, (off / size[k]).max().item() / EPS32)


CASES = [(1, 1, "layer", None, False), (1, 5, "rms", 1, True), (3, 4, "layer", 3, True), (8, 33, "layer", 2, False),
         (6, 257, "rms", 6, True), (12, 768, "layer", 4, True), (10, 1001, "rms", None, False),
         (5, 1030, "layer", 1, True), (2, 4100, "rms", 2, True), (30, 64, "layer", 15, True), (2, 16384, "layer", 1, True)]


@pytest.mark.parametrize("n,d,kind,gate,post", CASES)
def test_values_and_gradients_are_the_formula(n, d, kind, gate, post):
    t, settings, up = case(n, d, kind, gate, post, seed=n + d)
    check(gradients(t, settings, up), t, settings, up)


@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_gradients_are_the_differences(kind):
    """Along a random direction of all inputs, (L(+h) - L(-h)) / 2h of L = <r, dr> + <y, dy>. The
    difference's rounding: outputs of 400 values near 3, errors 2^-24 x 16 each, over 2h: 400^0.5 x 3 x 1e-6 /
    0.02 = 3e-3; its truncation h^2 / 6 times a third derivative of some 1e3 along the direction: 0.02."""
    t, settings, up = case(10, 40, kind, 5, True, seed=3)
    got = gradients(t, settings, up)
    h = 1e-2
    g = torch.Generator().manual_seed(9)
    direction = {k: None if v is None else torch.randn(v.shape, generator=g) / 20 for k, v in t.items()}
    slope = sum((got["d" + k].double() * direction[k].double()).sum() for k in NAMES if t[k] is not None).item()

    def value(s):
        r, y = call({k: None if v is None else v + s * direction[k] for k, v in t.items()}, settings)
        return ((r.double() * up[0].double()).sum() + (y.double() * up[1].double()).sum()).item()

    assert abs((value(h) - value(-h)) / (2 * h) - slope) < 0.03


def test_norm_alone_is_the_norm_of_a_residual_of_nothing():
    t, settings, up = case(9, 50, "layer")
    y = rg.norm(t["x"], t["weight"], t["bias"])
    r, want = rg.residual_norm(t["x"], torch.zeros(9, 50), t["weight"], t["bias"])
    assert torch.equal(y, want) and torch.equal(r, t["x"])
    x = t["x"].requires_grad_()
    w, b = t["weight"].requires_grad_(), t["bias"].requires_grad_()
    got = torch.autograd.grad(rg.norm(x, w, b), (x, w, b), up[1])
    f = torch.zeros(9, 50, requires_grad=True)
    want = torch.autograd.grad(rg.residual_norm(x, f, w, b)[1], (x, w, b, f), up[1])
    assert all(torch.equal(p, q) for p, q in zip(got, want)) and torch.equal(want[0], want[3])


def test_unused_outputs_and_frozen_inputs():
    t, settings, up = case(7, 20, "layer", 7, True)
    zero = torch.zeros_like(up[0])
    full = gradients(t, settings, up)
    leaf = {k: v.detach().requires_grad_() for k, v in t.items()}
    r, y = call(leaf, settings)
    only_y = torch.autograd.grad(y, [leaf[k] for k in NAMES], up[1], retain_graph=True)
    want = gradients(t, settings, (zero, up[1]))
    for k, g in zip(NAMES, only_y):
        assert torch.equal(g, want["d" + k]), k
    only_r = torch.autograd.grad(r, [leaf[k] for k in NAMES], up[0], allow_unused=True)
    want = gradients(t, settings, (up[0], zero))
    for k, g in zip(NAMES, only_r):
        assert torch.equal(g, want["d" + k]), k
    for k in NAMES:  # one at a time
        leaf = {q: v.detach().requires_grad_(q == k) for q, v in t.items()}
        (g,) = torch.autograd.grad(call(leaf, settings), [leaf[k]], up)
        assert torch.equal(g, full["d" + k]), k


def test_absent_weights_are_ones_and_zeros():
    t, settings, up = case(6, 30, "layer", None, True)
    r, y = rg.residual_norm(t["x"], t["f"], post_norm=True)
    r1, y1 = rg.residual_norm(t["x"], t["f"], torch.ones(30), torch.zeros(30), post_norm=True,
                              post_weight=torch.ones(30), post_bias=torch.zeros(30))
    assert torch.equal(r, r1) and torch.equal(y, y1)
    x = t["x"].requires_grad_()
    f = t["f"].requires_grad_()
    got = torch.autograd.grad(rg.residual_norm(x, f, post_norm=True), (x, f), up)
    want = torch.autograd.grad(rg.residual_norm(x, f, torch.ones(30), post_norm=True, post_weight=torch.ones(30)),
                               (x, f), up)
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_shapes_strides_and_gate_forms():
    torch.manual_seed(2)
    x, f = torch.randn(4, 6, 24), torch.randn(24, 6, 4).permute(2, 1, 0)
    w = torch.randn(48)[::2]
    gate = torch.randn(4, 24)
    r, y = rg.residual_norm(x, f, w, gate=gate)
    want = rg.residual_norm(x.view(24, 24), f.reshape(24, 24), w.contiguous(), gate=gate[:, None].expand(4, 6, 24).reshape(24, 24))
    assert r.shape == x.shape and torch.equal(r.view(24, 24), want[0]) and torch.equal(y.view(24, 24), want[1])
    one = rg.residual_norm(x, f, w, gate=gate[0])[1]
    assert torch.equal(one, rg.residual_norm(x, f, w, gate=gate[0].expand(4, 6, 24))[1])
    assert torch.equal(rg.norm(torch._neg_view(x)), rg.norm(-x))


def test_rows_do_not_reach_each_other():
    t, settings, up = case(11, 37, "layer", None, True)
    clean = call(t, settings)
    t["x"][3, 5], t["f"][8, 0] = math.nan, math.inf
    r, y = call(t, settings)
    for n in range(11):
        if n in (3, 8):
            assert y[n].isnan().all()
        else:
            assert torch.equal(y[n], clean[1][n]) and torch.equal(r[n], clean[0][n])
    # rows equal everywhere: zero deviation, and all zero with eps 0
    assert torch.equal(rg.norm(torch.full((2, 8), 3.0)), torch.zeros(2, 8))
    assert rg.norm(torch.zeros(2, 8), kind="rms", eps=0.0).isnan().all()


@pytest.mark.parametrize("n", [0, 1])
def test_no_rows_and_one(n):
    t, settings, up = case(n, 12, "layer", None, True)
    got = gradients(t, settings, up)
    assert got["r"].shape == (n, 12)
    if n == 0:
        assert all(torch.equal(got[k], torch.zeros(12)) for k in ("dweight", "dbias", "dpost_weight", "dpost_bias"))


def test_refusals():
    x = torch.zeros(6, 8)
    bad = [
        lambda: rg.norm(x, kind="batch"), lambda: rg.norm(torch.zeros(2, 0)), lambda: rg.norm(torch.tensor(1.0)),
        lambda: rg.norm(torch.zeros(1, 16385)), lambda: rg.norm(x.double()), lambda: rg.norm(x, torch.ones(7)),
        lambda: rg.norm(x, torch.ones(8).double()), lambda: rg.norm(x, eps=-1.0), lambda: rg.norm(x, eps=math.nan),
        lambda: rg.residual_norm(x, torch.zeros(6, 7)), lambda: rg.residual_norm(x, x, gate=torch.ones(4, 8)),
        lambda: rg.residual_norm(x, x, gate=torch.ones(12, 8)), lambda: rg.residual_norm(x, x, gate=torch.ones(8, 6)),
        lambda: rg.residual_norm(x, x, gate=torch.ones(0, 8)), lambda: rg.residual_norm(x, x, post_weight=torch.ones(8)),
        lambda: rg.residual_norm(x, x, torch.ones(8, device="meta")), lambda: rg.Norm(8, kind="batch"),
    ]
    for k, b in enumerate(bad):
        with pytest.raises(ValueError):
            b()
            pytest.fail("case %d" % k)


def test_c_entry_refuses_bad_arguments():
    lib, bad = _lib.lib, _lib.HIP_ERROR_INVALID_VALUE
    c = _lib.rg_norm_config()
    lib.rg_norm_config_init(ctypes.byref(c))
    assert (c.N, c.D, c.rms, c.post, c.gate_rows, c.scale) == (0, 0, 0, 0, 0, 1.0) and abs(c.eps - 1e-5) < 1e-12
    p = 4096

    def forward(c, x=p, f=p, gate=None, pw=None, pb=None, w=None, b=None, r=p, y=p, stats=None):
        return lib.rg_residual_norm_fp32(ctypes.byref(c), x, f, gate, pw, pb, w, b, r, y, stats, None, 0, None)

    def config(**k):
        return _lib.rg_norm_config(**{**dict(N=4, D=8, rms=0, post=0, gate_rows=0, eps=1e-5, scale=1.0), **k})

    for broken in (dict(N=-1), dict(D=0), dict(D=16385), dict(eps=-1.0), dict(eps=math.nan), dict(gate_rows=3), dict(gate_rows=8)):
        assert forward(config(**broken)) == bad
    assert forward(config(N=0)) == 0
    for broken in (dict(x=None), dict(y=None), dict(r=None), dict(f=None), dict(gate=p), dict(pw=p)):
        assert forward(config(), **broken) == bad
    assert forward(config(gate_rows=2)) == bad and forward(config(post=1), f=None, r=None) == bad
    size = ctypes.c_size_t()
    assert lib.rg_residual_norm_grad_workspace(ctypes.byref(config()), 1, ctypes.byref(size)) == 0 and size.value > 0
    args = [p, p, p, p, None, None, None, None, p, p, p, None, None, None, p, p]

    def backward(c, args=args, ws=p, n=size.value):
        return lib.rg_residual_norm_grad_fp32(ctypes.byref(c), *args, ws, n, None, 0, None)

    for i, v in ((2, None), (8, None), (8, p + 4), (11, p), (12, p)):
        assert backward(config(), args[:i] + [v] + args[i + 1:]) == bad
    assert backward(config(), [None, None] + args[2:]) == bad
    assert backward(config(), ws=None) == bad and backward(config(), n=size.value - 1) == bad
    assert backward(config(), ws=p + 2) == bad


def test_modules_report_to_the_guard():
    rg.guard().reset()
    torch.manual_seed(0)
    m = rg.ResidualNorm(16, post_norm=True, scale=0.5)
    m.repro_name = "block.norm"
    x, f = torch.randn(3, 16), torch.randn(3, 16)
    r, y = m(x, f)
    want = rg.residual_norm(x, f, m.weight, m.bias, scale=0.5, post_norm=True, post_weight=m.post_weight, post_bias=m.post_bias)
    assert torch.equal(r, want[0]) and torch.equal(y, want[1])
    assert rg.guard().first_offender() is None
    f[1, 2] = math.inf
    m(x, f)
    assert rg.guard().first_offender() == "block.norm input"
    rg.guard().reset()
    n = rg.Norm(16, kind="rms")
    assert n.bias is None and torch.equal(n(x), rg.norm(x, n.weight, kind="rms"))


def test_gradients_are_differentiable_no_further():
    t, settings, up = case(5, 16, "layer", None)
    x = t["x"].requires_grad_()
    r, y = call(t, settings)
    (dx,) = torch.autograd.grad((r, y), [x], up, create_graph=True)
    with pytest.raises(RuntimeError, match="only once"):
        dx.sum().backward()


def test_gates_that_line_up_with_rows():
    """The gate's leading sizes, 1s at their end left out, are x's first ones (x's own 1s aside): the value of a row
    is that of its place among them."""
    x, f = torch.randn(2, 3, 4, 5), torch.randn(2, 3, 4, 5)
    for lead in ((), (1,), (1, 1, 1), (2,), (2, 1), (2, 1, 1), (2, 3), (2, 3, 1), (2, 3, 4)):
        gate = torch.randn(*lead, 5)
        full = gate.reshape(*lead, *(1,) * (3 - len(lead)), 5).expand(2, 3, 4, 5)
        assert torch.equal(rg.residual_norm(x, f, gate=gate)[0], x + full * f), lead
    one = torch.randn(4, 5)
    assert torch.equal(rg.residual_norm(x[:1, :1], f[:1, :1], gate=one)[0], x[:1, :1] + one * f[:1, :1])
    rows = torch.randn(2, 5)  # rows without further structure, in runs
    assert torch.equal(rg.residual_norm(x.view(24, 5), f.view(24, 5), gate=rows)[0],
                       x.view(24, 5) + rows.repeat_interleave(12, 0) * f.view(24, 5))


@pytest.mark.parametrize("lead", [(4,), (1, 4), (1, 3), (3,), (3, 4), (1, 3, 4), (2, 4), (2, 1, 4), (4, 3, 2), (6,), (24,),
                                  (2, 3, 4, 2), (12, 2)])
def test_gates_that_do_not_line_up_are_refused(lead):
    """Broadcasting or counts would read these in ways that differ."""
    x = torch.zeros(2, 3, 4, 5)
    with pytest.raises(ValueError, match="gate"):
        rg.residual_norm(x, x, gate=torch.ones(*lead, 5))
    with pytest.raises(ValueError, match="gate"):
        rg.ResidualNorm(5)(x, x, torch.ones(*lead, 5))
    with pytest.raises(ValueError, match="gate"):
        rg.residual_norm(x.view(24, 5), x.view(24, 5), gate=torch.ones(2, 4, 5))


@pytest.mark.parametrize("what", ["gradient", "input", "squares", "gate"])
@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_the_guard_hears_what_it_hears_on_a_gpu(what, kind):
    rg.guard().reset()
    m = rg.ResidualNorm(40, kind=kind)
    m.repro_name = "eight"
    x, f, gate = torch.randn(9, 40, requires_grad=True), torch.randn(9, 40), torch.ones(40)
    up = torch.zeros(9, 40)
    if what == "gradient":
        up[4, 39] = math.nan
    elif what == "input":
        f[8, 0] = -math.inf
    elif what == "gate":
        gate[3] = math.nan
    else:
        f[2] = 1e25 * torch.randn(40)  # finite, its squares are not
    r, y = m(x, f, gate)
    assert rg.guard().first_offender() == (None if what == "gradient" else "eight input")
    if what == "gradient":
        torch.autograd.grad(y, x, up)
        assert rg.guard().first_offender() == "eight gradient"
        rg.guard().reset()
        torch.autograd.grad(m(x, f, gate)[0], x, torch.full((9, 40), math.inf))
        assert rg.guard().first_offender() == "eight gradient"
    rg.guard().reset()
    n = rg.Norm(40, kind=kind)
    torch.autograd.grad(n(x), n.weight, up.fill_(1.0))
    rg.guard().check()


@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_the_guard_hears_a_block_whose_squares_pass_the_range(kind):
    """Normalised first, such an output becomes zeros, and r is an ordinary row."""
    rg.guard().reset()
    m = rg.ResidualNorm(40, kind=kind, post_norm=True)
    x, f = torch.randn(5, 40), torch.randn(5, 40)
    m(x, f)
    rg.guard().check()
    f[3] *= 1e25
    r, y = m(x, f)
    assert torch.isfinite(r).all() and torch.isfinite(y).all()
    assert rg.guard().first_offender() == "residual_norm input"
    rg.guard().reset()


def test_partial_sums_over_rows_are_few():
    """At most two for each strand that a GPU is given (2048 for rows of up to 1024 values, else 512): a launch of a block for
    each, and of a row of blocks for each sum, always fits. The workspace has five sums' partials."""
    g = torch.Generator().manual_seed(1)
    size = ctypes.c_size_t()
    for d, aim in ((8, 2048), (1024, 2048), (1025, 512), (16384, 512)):
        for k in range(400):
            n = int(2.0 ** (40 * torch.rand(1, generator=g, dtype=torch.float64).item()))
            rows = 2 ** int(torch.randint(0, 41, (1,), generator=g))  # groups of at least four rows, and shorter ones
            for total, gate in ((n, 0), (n, 1), (n, n), (n // rows * rows, n // rows)):
                if total == 0:
                    continue
                c = _lib.rg_norm_config(N=total, D=d, rms=0, post=0, gate_rows=gate, eps=1e-5, scale=1.0)
                assert _lib.lib.rg_residual_norm_grad_workspace(ctypes.byref(c), 1, ctypes.byref(size)) == 0
                assert 0 < size.value // (5 * 4 * d) <= 2 * aim, (total, d, gate)
