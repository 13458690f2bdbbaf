"""The residual norm and its gradients on the GPU against the CPU's: the same bits, for every width class,
gate form and alignment."""
import math

import pytest
import torch

import bit_reproducible_training_amd as rg
from test_norm import case, check, gradients

pytestmark = pytest.mark.gpu


def cuda(t):
    return {k: None if v is None else v.cuda() for k, v in t.items()}


def assert_same(got, want):
    assert got.keys() == want.keys()
    for k in want:
        a, b = got[k].cpu(), want[k]
        nan = b.isnan()
        assert torch.equal(a.isnan(), nan), k
        assert torch.equal(a[~nan].view(torch.int32), b[~nan].view(torch.int32)), k


# Each width class at its ends, by one row, a few, and enough for several rows a strand.
WIDTHS = [1, 2, 3, 4, 63, 255, 256, 257, 511, 513, 768, 769, 1001, 1024, 1025, 2047, 2049, 4096, 4097, 8192, 8195, 16384]


@pytest.mark.parametrize("d", WIDTHS)
@pytest.mark.parametrize("post", [False, True])
def test_gives_the_cpu_bits_at_every_width(d, post):
    for n, kind, gate in ((1, "layer", 1), (13, "rms", 13), (24, "layer", None), (24, "rms", 4)):
        print(n, d, kind, gate, flush=True)
        t, settings, up = case(n, d, kind, gate, post, seed=d)
        got = gradients(cuda(t), settings, [u.cuda() for u in up])
        assert_same(got, gradients(t, settings, up))
        check(got, t, settings, up)


@pytest.mark.parametrize("n,d,gate", [(9001, 20, None), (9000, 20, 1), (9000, 20, 3), (9000, 20, 4500), (9000, 20, 1800),
                                      (9000, 20, 9000), (2100, 1100, 7), (2100, 1100, 700), (3000, 4100, 5)])
@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_gives_the_cpu_bits_for_many_rows(n, d, gate, kind):
    """Sections of one group, strands of several groups, and of one."""
    t, settings, up = case(n, d, kind, gate, True, seed=n)
    assert_same(gradients(cuda(t), settings, [u.cuda() for u in up]), gradients(t, settings, up))


def test_norm_alone_and_partial_gradients():
    t, settings, up = case(700, 130, "layer", None)
    for device in ("cpu", "cuda"):
        x, w, b = (t[k].to(device).requires_grad_() for k in ("x", "weight", "bias"))
        got = torch.autograd.grad(rg.norm(x, w, b), (x, w, b), up[1].to(device))
        (only,) = torch.autograd.grad(rg.norm(x.detach(), w, b.detach()), [w], up[1].to(device))
        assert torch.equal(only, got[1])
        if device == "cpu":
            want = got
    assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want))


def test_extreme_rows_give_the_cpu_bits():
    t, settings, up = case(12, 300, "layer", 12, True)
    t["x"][1], t["x"][2], t["x"][3, 7], t["f"][4, 0] = 0.0, 1e-42, math.nan, -math.inf
    t["x"][5], t["f"][6], up[1][7, 3] = 3e38, 5.0, math.inf
    assert_same(gradients(cuda(t), settings, [u.cuda() for u in up]), gradients(t, settings, up))


@pytest.mark.parametrize("shift", [1, 2, 3])
def test_rows_off_16_bytes(shift):
    """Operands that start anywhere; what lies around the outputs is the allocator's, so only inputs."""
    t, settings, up = case(50, 516, "rms", None, True, seed=shift)

    def moved(v):
        if v is None:
            return None
        flat = torch.empty(v.numel() + 8, device="cuda")
        out = flat[shift:shift + v.numel()].view(v.shape)
        return out.copy_(v)

    got = gradients({k: moved(v) for k, v in t.items()}, settings, [moved(u) for u in up])
    assert_same(got, gradients(t, settings, up))


def test_another_stream_and_graph_replays():
    t, settings, up = case(333, 768, "layer", 3, True)
    want = gradients(t, settings, up)
    t, up = cuda(t), [u.cuda() for u in up]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert_same(gradients(t, settings, up), want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = gradients(t, settings, up)
    for _ in range(3):
        for v in got.values():
            v.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        assert_same(got, want)


def test_modules_report_to_the_guard_on_the_gpu():
    rg.guard().reset()
    m = rg.ResidualNorm(40, kind="rms").cuda()
    m.repro_name = "seven"
    x = torch.randn(9, 40, device="cuda", requires_grad=True)
    f = torch.randn(9, 40, device="cuda")
    r, y = m(x, f)
    rg.guard().check()
    up = torch.zeros_like(y)
    up[4, 39] = math.nan
    torch.autograd.grad(y, x, up)
    assert rg.guard().first_offender() == "seven gradient"
    rg.guard().reset()
    f[8, 0] = -math.inf
    m(x, f)
    assert rg.guard().first_offender() == "seven input"
    rg.guard().reset()


def test_refuses_tensors_on_two_devices():
    x = torch.zeros(4, 8, device="cuda")
    for bad in (lambda: rg.norm(x, torch.ones(8)), lambda: rg.residual_norm(x, x.cpu()),
                lambda: rg.residual_norm(x, x, gate=torch.ones(8))):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("d", [40, 1100])
def test_the_guard_hears_the_same_on_both_devices(kind, d):
    g = torch.Generator().manual_seed(d)
    for what in range(6):
        heard = []
        for device in ("cpu", "cuda"):
            rg.guard().reset()
            m = rg.ResidualNorm(d, kind=kind).to(device)
            m.repro_name = "nine"
            x, f = torch.randn(9, d, generator=g.manual_seed(what)), torch.randn(9, d, generator=g)
            up = [torch.randn(9, d, generator=g) for _ in range(2)]
            if what < 2:
                (x, f)[what][3, d - 1] = math.inf
            elif what == 2:
                x[5] *= 1e25
            elif what < 5:
                up[what - 3][8, d - 1] = math.nan
            x = x.to(device).requires_grad_()
            torch.autograd.grad(m(x, f.to(device)), x, [u.to(device) for u in up])
            heard.append(rg.guard().first_offender())
        rg.guard().reset()
        assert heard[0] == heard[1] == (None if what == 5 else "nine gradient" if what > 2 else "nine input")


@pytest.mark.parametrize("d", [40, 1100])
def test_the_guard_hears_a_block_whose_squares_pass_the_range(d):
    rg.guard().reset()
    m = rg.ResidualNorm(d, kind="rms", post_norm=True).cuda()
    x, f = torch.randn(5, d, device="cuda"), torch.randn(5, d, device="cuda")
    m(x, f)
    rg.guard().check()
    f[3] *= 1e25
    m(x, f)
    assert rg.guard().first_offender() == "residual_norm input"
    rg.guard().reset()
