"""Attention whose scores are large: far from one another or equal, so that a softmax is one key's or shared by equals, at every
magnitude of float32, on the CPU and on the GPU.

A row's scores are T times small numbers in eighths, T from 2^12 up, so two of them are equal (their keys are the same) or T / 8
apart: more than 300, and 2^17 times what a score is off by (size roundings of its products). What is not the largest has
less than 2^-400 of the softmax, and the formula in 64 bits is what is wanted."""
import math

import pytest
import torch

import bit_reproducible_training_amd as rg
from test_attention import EPS32, gradients

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def large_case(T, sign, tq, tk, d, h, bias, causal, seed):
    """Keys of three values (one that varies in eighths from 1/8 to 1, the others 0) under queries that see them as T sign times that."""
    g = torch.Generator().manual_seed(seed)
    k = torch.zeros(2, tk, 1, d)
    k[..., 0] = torch.randint(1, 9, (2, tk, 1), generator=g) / 8
    q = torch.randn(2, tq, h, d, generator=g)
    q[..., 0] = T * sign * (1 + torch.rand(2, tq, h, generator=g))
    t = {"q": q, "k": k, "v": torch.randn(2, tk, 1, d, generator=g),
         "relative_bias": torch.zeros(h, tq + tk - 1) if bias else None}
    return t, dict(causal=causal, query_start=max(tk - tq, 0), scale=1.0), torch.randn(2, tq, h, d, generator=g)


def check_shared_by_equals(got, t, s, dy):
    """Within the roundings' worst case, in units of 2^-24: p of a largest key is 2^x for the same x for each of them, so p is off by a
    rounding a key of the sum and eight for each of its rescalings (R); y, dp and delta and the sums of gradients as they are made."""
    q, k, v, dy = (x.double().cpu().transpose(1, 2) for x in (t["q"], t["k"], t["v"], dy))
    got = {n: x.double().cpu() for n, x in got.items()}
    tq, tk, h, d = q.shape[2], k.shape[2], q.shape[1], q.shape[3]
    z = (q @ k.transpose(2, 3)) * s["scale"]
    rows, keys = torch.arange(tq)[:, None], torch.arange(tk)[None, :]
    seen = (keys <= rows + s["query_start"]) | torch.tensor(not s["causal"])
    z = z.masked_fill(~seen, -math.inf)
    p = torch.softmax(z, -1)
    y = p @ v
    R = tk + 8 * (tk // 64 + tk // 256 + 2) + 16
    want, off = {"y": y}, {"y": R * (p @ v.abs())}
    dp, delta = dy @ v.transpose(2, 3), (dy * y).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    size = dy.abs() @ v.abs().transpose(2, 3) + (dy.abs() * (p @ v.abs())).sum(-1, keepdim=True)
    ds_off = p * (2 * R + 2 * d + 8) * size
    want["dq"], off["dq"] = ds @ k, (ds_off + (tk + 8) * p * size) @ k.abs()
    want["dk"] = (ds.transpose(2, 3) @ q).sum(1, keepdim=True)
    off["dk"] = ((ds_off + h * (tq + 8) * p * size).transpose(2, 3) @ q.abs()).sum(1, keepdim=True)
    want["dv"] = (p.transpose(2, 3) @ dy).sum(1, keepdim=True)
    off["dv"] = ((R + h * (tq + 8)) * p.transpose(2, 3) @ dy.abs()).sum(1, keepdim=True)
    for n, w in ((n, w) for n, w in want.items() if n in got):
        w, o = w.transpose(1, 2), off[n].transpose(1, 2)
        assert got[n].isfinite().all(), n
        far = (got[n] - w).abs()
        assert torch.all(far <= EPS32 * o + 1e-37), (n, (far / (EPS32 * o + 1e-37)).max().item())


def run(device, t, s, dy):
    on = {n: None if x is None else x.to(device) for n, x in t.items()}
    return gradients(on, {"key_lengths": None, "mask": None, **s}, dy.to(device))


SHAPES = [(1, 1, 1, 1), (1, 40, 3, 2), (3, 300, 16, 2), (40, 70, 8, 2), (150, 300, 64, 1), (70, 140, 100, 2)]  # tq, tk, d, h


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("tq,tk,d,h", SHAPES)
@pytest.mark.parametrize("sign", [1, -1])
def test_large_scores(device, tq, tk, d, h, sign):
    for n, T in enumerate((2.0 ** 12, 2.0 ** 20, 2.0 ** 23, 2.0 ** 24, 1e9, 3e10, 4e12, 1e20, 1e30, 2e36)):
        for bias, causal in ((False, False), (False, True), (True, True)):
            t, s, dy = large_case(T, sign, tq, tk, d, h, bias, causal, n)
            got = run(device, t, s, dy)
            check_shared_by_equals(got, t, s, dy)
            if device != "cpu":
                want = run("cpu", t, s, dy)
                assert all(torch.equal(got[m].cpu(), want[m]) for m in want), (T, bias, causal)


@pytest.mark.parametrize("device", DEVICES)
def test_one_key_is_its_value(device):
    """Whatever its score: three roundings, and none from 2^24 on."""
    g = torch.Generator().manual_seed(1)
    n = 2000
    size = 2.0 ** (torch.rand(n, generator=g) * 138 - 20)
    q = (size * (1 - 2 * torch.randint(0, 2, (n,), generator=g))).view(n, 1, 1, 1).float()
    v = torch.randn(n, 1, 1, 1, generator=g)
    for bias in (None, torch.zeros(1, 1)):
        y = rg.attention(q.to(device), torch.ones_like(q).to(device), v.to(device), scale=1.0,
                         relative_bias=None if bias is None else bias.to(device)).cpu()
        assert torch.all((y - v).abs() <= 3 * EPS32 * v.abs())
        assert torch.equal(y[size > 2.0 ** 24], v[size > 2.0 ** 24])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("d", [8, 100])
def test_large_scores_beside_masked_nans(device, d):
    """What the last query alone sees holds NaN: the others' bits stay."""
    t, s, dy = large_case(1e9, 1, 150, 150, d, 2, False, True, 3)
    want = run(device, t, s, dy)
    t["k"][:, -1], t["v"][:, -1], dy[:, -1] = math.nan, math.nan, math.nan
    got = run(device, t, s, dy)
    assert torch.equal(got["y"][:, :-1], want["y"][:, :-1]) and torch.equal(got["dq"][:, :-1], want["dq"][:, :-1])
    assert got["y"][:, -1].isnan().all() and got["dv"].isnan().all()


def same_bits(got, want):
    """NaN at the same places, and the same bits elsewhere."""
    return all(torch.equal(got[n].cpu().isnan(), want[n].isnan()) and torch.equal(got[n].cpu().nan_to_num(7.0), want[n].nan_to_num(7.0))
               for n in want)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("tq,tk,d,h", SHAPES)
def test_rows_whose_scores_are_all_far_below_zero(device, tq, tk, d, h):
    """Base 2 scores from -1.4e37 to float32's least. (Gradients of k would be T times a share of the gradient, past float32.)"""
    for T in (8e37, 1.17e38):
        for bias, causal in ((False, False), (False, True), (True, True)):
            t, s, dy = large_case(T, -1, tq, tk, d, h, bias, causal, 5)
            got = run(device, t, s, dy)
            check_shared_by_equals({n: got[n] for n in ("y", "dq", "dv")}, t, s, dy)
            assert same_bits(got, run("cpu", t, s, dy))


@pytest.mark.parametrize("device", DEVICES)
def test_scores_at_the_end_of_the_range(device):
    """Base 2 scores of +-1.6e38 beside each other; those of +-2e38 are further apart than float32 reaches and may give NaN but nothing else
    that is wrong, and one of 3.5e38 is past it and gives NaN. Other rows are as they are."""
    for T, bias, fine in ((1.1e38, False, True), (1.1e38, True, True), (1.4e38, False, False), (1.4e38, True, False), (2.4e38, True, False)):
        for tq in (1, 20):
            t = {"q": torch.ones(1, tq, 1, 1), "k": torch.zeros(1, 300, 1, 1), "v": torch.randn(1, 300, 1, 1),
                 "relative_bias": torch.zeros(1, tq + 299) if bias else None}
            t["q"][:, 0], t["k"][:, 9], t["k"][:, 270] = T, 1.0, -1.0
            s, dy = dict(scale=1.0, causal=False, query_start=0), torch.randn(1, tq, 1, 1)
            got, want = run(device, t, s, dy), run("cpu", t, s, dy)
            assert same_bits(got, want)
            y = got["y"][0, 0, 0].cpu()
            assert (torch.equal(y, t["v"][0, 9, 0]) and T < 2e38) or (y.isnan().all() and not fine)
            assert got["y"][0, 1:].isfinite().all() and got["dq"][0, 1:].isfinite().all()
