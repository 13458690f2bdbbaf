"""Attention and its gradients against the formula in 64 bits and against differences, what masks hide, and the refusals,
on the CPU."""
import math

import pytest
import torch

import bit_reproducible_training_amd as rg

EPS32 = 2.0 ** -24
NAMES = ("q", "k", "v", "relative_bias")


def case(b, h, kvh, tq, tk, d, causal=False, lengths=False, mask=None, bias=False, drop=0.0, seed=0):
    """The call's tensors (None where absent), its settings and a gradient of y. mask: "pairs", "keys" or None."""
    g = torch.Generator().manual_seed(seed + 7919 * tq + tk)
    t = {"q": torch.randn(b, tq, h, d, generator=g), "k": torch.randn(b, tk, kvh, d, generator=g),
         "v": torch.randn(b, tk, kvh, d, generator=g),
         "relative_bias": torch.randn(h, max(tq + tk - 1, 0), generator=g) if bias else None}
    s = dict(causal=causal, query_start=max(tk - tq, 0) if causal else 0, dropout=drop, seed=1234567 + seed, key_lengths=None, mask=None)
    if lengths:
        s["key_lengths"] = torch.randint(0, tk + 1, (b,), generator=g)
        s["key_lengths"][0] = tk
    if mask == "pairs":
        s["mask"] = torch.rand(b, 1, tq, tk, generator=g) < 0.6
        s["mask"][:, :, 3::7] = False
    elif mask == "keys":
        s["mask"] = torch.rand(h, 1, tk, generator=g) < 0.6
    return t, s, torch.randn(b, tq, h, d, generator=g)


def gradients(t, s, dy):
    """{y, d...} of the call."""
    t = {n: None if v is None else v.detach().requires_grad_() for n, v in t.items()}
    y = rg.attention(**t, **s)
    held = [n for n in NAMES if t[n] is not None]
    return {"y": y.detach(), **{"d" + n: g for n, g in zip(held, torch.autograd.grad(y, [t[n] for n in held], dy))}}


def keeps(b, h, tq, tk, p, seed):
    """The pairs that dropout keeps, in Python's whole numbers: [b, h, tq, tk]"""
    out = torch.ones(b * h, tq, tk, dtype=torch.bool)
    for n in range(b * h):
        for i in range(tq):
            for group in range((tk + 3) // 4):
                words = philox(group, i, n, 1, seed)
                for r in range(min(4, tk - 4 * group)):
                    out[n, i, 4 * group + r] = words[r] >= int(p * 2 ** 32)
    return out.view(b, h, tq, tk)


def philox(c0, c1, c2, c3, seed):
    k0, k1 = seed % 2 ** 32, seed >> 32
    for _ in range(10):
        a, b = 0xD2511F53 * c0, 0xCD9E8D57 * c2
        c0, c1, c2, c3 = (b >> 32) ^ c1 ^ k0, b % 2 ** 32, (a >> 32) ^ c3 ^ k1, a % 2 ** 32
        k0, k1 = (k0 + 0x9E3779B9) % 2 ** 32, (k1 + 0xBB67AE85) % 2 ** 32
    return c0, c1, c2, c3


def check(got, t, s, dy):
    """Against the formula in 64 bits, each value within the roundings' worst case.

    In units of 2^-24, relative to the magnitudes: a score's chain has size roundings and its factor and shift six more, in
    units of the sum of its products' magnitudes T (base 2); an exponential follows its exponent's error times ln 2 and has four of its
    own; each tile and chunk rescales with eight at most and exponents of at most 2 T; a sum over keys has a rounding a key. p is off by
    R = 1.4 (size + 8) T + keys + 16 (tiles + chunks) + 16, twice for the quotient. dp and delta have size roundings and carry y's error;
    a gradient's sum has a rounding for each of its terms and a handful for its parts."""
    t = {n: None if v is None else v.detach().cpu().double() for n, v in t.items()}
    got = {n: v.cpu().double() for n, v in got.items()}
    dy = dy.cpu().double()
    q, k, v = t["q"], t["k"], t["v"]
    b, tq, h, d = q.shape
    tk, kvh = k.shape[1], k.shape[2]
    group = h // kvh
    q, dy = q.transpose(1, 2), dy.transpose(1, 2)
    k, v = (x.transpose(1, 2).repeat_interleave(group, 1) for x in (k, v))
    scale = s.get("scale") or d ** -0.5
    z, size = q @ k.transpose(2, 3) * scale, q.abs() @ k.abs().transpose(2, 3) * abs(scale)
    rows, keys = torch.arange(tq)[:, None], torch.arange(tk)[None, :]
    place = keys - rows + tq - 1
    if t["relative_bias"] is not None:
        z, size = z + t["relative_bias"][:, place], size + t["relative_bias"].abs()[:, place]
    seen = torch.ones(b, h, tq, tk, dtype=torch.bool)
    if s["causal"]:
        seen &= keys <= rows + s["query_start"]
    if s["key_lengths"] is not None:
        seen &= (keys < s["key_lengths"].cpu()[:, None])[:, None, None, :]
    if s["mask"] is not None:
        seen &= s["mask"].cpu()
    z = z.masked_fill(~seen, -math.inf)
    top = z.amax(-1, keepdim=True) if tk else z.new_zeros(b, h, tq, 1)
    e = torch.exp(z - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total == 0, 1.0, total)
    factor = torch.ones(b, h, tq, tk, dtype=torch.float64)
    if s["dropout"]:
        factor = keeps(b, h, tq, tk, s["dropout"], s["seed"]) / (1 - s["dropout"])
    u = p * factor
    y = u @ v
    big = size.masked_fill(~seen, 0.0).amax() * 1.4427 if tk else 0.0
    R = 2 * (1.4 * (d + 8) * big + tk + 16 * (tk // 64 + tk // 256 + 2) + 16)
    off = {"y": R * (u @ v.abs())}
    want = {"y": y}
    if len(got) > 1:
        dp = dy @ v.transpose(2, 3) * factor
        delta = (dy * y).sum(-1, keepdim=True)
        ds = p * (dp - delta)
        dp_size = dy.abs() @ v.abs().transpose(2, 3) * factor
        delta_size = (dy.abs() * y.abs()).sum(-1, keepdim=True)
        ds_off = p * (R * (dp_size + delta_size) + (d + 4) * (dp_size + delta_size) + (dy.abs() * off["y"]).sum(-1, keepdim=True))
        ds_size = p * (dp_size + delta_size)
        want["dq"], off["dq"] = ds @ k * scale, (ds_off + (tk + tk // 128 + 4) * ds_size) @ k.abs() * abs(scale)
        many = group * (tq + tq // 256 + 4)

        def shared(x):
            return x.view(b, kvh, group, tk, d).sum(2)

        want["dk"] = shared(ds.transpose(2, 3) @ q) * scale
        off["dk"] = shared((ds_off + many * ds_size).transpose(2, 3) @ q.abs()) * abs(scale)
        want["dv"] = shared(u.transpose(2, 3) @ dy)
        off["dv"] = shared(((R + many) * u).transpose(2, 3) @ dy.abs())
        if t["relative_bias"] is not None:
            def by_distance(x):
                out = torch.zeros(h, tq + tk - 1, dtype=torch.float64)
                for head in range(h):
                    out[head].index_add_(0, place.flatten(), x[:, head].sum(0).flatten())
                return out
            want["drelative_bias"] = by_distance(ds)
            off["drelative_bias"] = by_distance(ds_off + b * (min(tq, tk) + 8) * ds_size)
    for n, w in want.items():
        w, o = (x if n == "drelative_bias" else x.transpose(1, 2) for x in (w, off[n]))
        assert got[n].shape == w.shape, n
        far = (got[n] - w).abs()
        assert torch.all(far <= EPS32 * o + 1e-37), (n, (far / (EPS32 * o + 1e-37)).max().item())


CASES = [  # b, h, kvh, tq, tk, d, causal, lengths, mask, bias, drop
    (1, 1, 1, 1, 1, 1, False, False, None, False, 0.0), (2, 2, 1, 1, 77, 64, False, True, None, False, 0.0),
    (2, 4, 2, 70, 70, 33, True, False, None, True, 0.25), (1, 2, 2, 5, 300, 16, False, True, "pairs", True, 0.0),
    (2, 3, 1, 129, 65, 8, False, False, "keys", False, 0.5), (1, 2, 1, 300, 17, 128, True, False, None, False, 0.0),
    (3, 1, 1, 9, 513, 7, True, True, "pairs", True, 0.1), (1, 6, 2, 40, 40, 96, False, False, "pairs", False, 0.0)]


@pytest.mark.parametrize("c", CASES)
def test_values_and_gradients_are_the_formula(c):
    t, s, dy = case(*c, seed=sum(c[:6]))
    check(gradients(t, s, dy), t, s, dy)


def test_a_scale_and_a_late_start():
    t, s, dy = case(2, 2, 2, 20, 50, 12)
    s.update(scale=-0.7, causal=True, query_start=-5)
    check(gradients(t, s, dy), t, s, dy)
    assert torch.all(rg.attention(**t, **s)[:, :5] == 0)


def test_gradients_are_the_differences():
    """Central differences of a weighted sum of y over steps of 2^-6, in 64 bits of differences: float32's noise in a sum of n values of
    about 1 is below n 2^-20, over the step's 2^-5; the third derivative's share is below the step squared times 40."""
    t, s, dy = case(1, 2, 1, 6, 9, 5, causal=True, bias=True, drop=0.2)
    got, step = gradients(t, s, dy), 2.0 ** -6
    n = dy.numel()

    def value(moved):
        return (rg.attention(**moved, **s).double() * dy.double()).sum().item()

    for name in NAMES:
        for at in range(0, t[name].numel(), 3):
            ends = []
            for sign in (1, -1):
                moved = {m: x.clone() for m, x in t.items()}
                moved[name].view(-1)[at] += sign * step
                ends.append(value(moved))
            slope = (ends[0] - ends[1]) / (2 * step)
            assert abs(slope - got["d" + name].reshape(-1)[at].item()) <= n * 2.0 ** -20 / (2 * step) + 40 * step ** 2


def test_rows_that_see_nothing_are_zero():
    t, s, dy = case(2, 2, 2, 7, 20, 8, mask="pairs", bias=True)
    s["mask"][:] = False
    got = gradients(t, s, dy)
    assert all(torch.all(x == 0) for x in got.values())
    s["mask"][:, :, 2, 5] = True
    got = gradients(t, s, dy)
    assert torch.equal(got["y"][:, 2], t["v"][:, 5]) and torch.all(got["y"][:, :2] == 0)


@pytest.mark.parametrize("hidden", [math.nan, math.inf, -math.inf, torch.finfo(torch.float32).min])
def test_what_is_masked_reaches_nothing(hidden):
    """Keys past the length, keys after the query, pairs of a mask: with anything in them the visible results keep their bits."""
    t, s, dy = case(2, 2, 1, 80, 80, 8, causal=True, bias=True, drop=0.1)
    s["key_lengths"] = torch.tensor([70, 80])
    s["mask"] = torch.ones(80, 80, dtype=torch.bool)
    s["mask"][:, 33] = False
    want = gradients(t, s, dy)
    for name in ("k", "v"):
        t[name][0, 70:] = hidden
        t[name][:, 33] = hidden
    got = gradients(t, s, dy)
    for n in want:
        assert torch.equal(got[n], want[n]), n
    # a key that only the last queries see
    t["v"][:, 60] = hidden
    got = gradients(t, s, dy)
    assert torch.equal(got["y"][:, :60], want["y"][:, :60]) and torch.equal(got["dq"][:, :60], want["dq"][:, :60])
    # a query and its gradient reach no key that it does not see
    t, s, dy = case(2, 2, 1, 80, 80, 8, causal=True, drop=0.1)
    want = gradients(t, s, dy)
    t["q"][:, 40], dy[:, 40] = hidden, hidden
    got = gradients(t, s, dy)
    for n in ("dk", "dv"):
        assert torch.equal(got[n][:, 41:], want[n][:, 41:]), n


def test_a_visible_nan_is_its_rows():
    t, s, dy = case(1, 1, 1, 6, 6, 4, causal=True)
    t["v"][0, 3, 0, 1] = math.nan
    got = gradients(t, s, dy)
    assert torch.all(got["y"][0, 3:, 0, 1].isnan()) and not got["y"][0, :, 0, 0].isnan().any()
    t, s, dy = case(1, 1, 1, 6, 6, 4)
    t["q"][0, 2] = math.inf
    got = gradients(t, s, dy)
    assert got["y"][0, 2].isnan().all() and not got["y"][0, [0, 1, 3, 4, 5]].isnan().any()


def test_a_row_has_its_bits_alone_and_among_others():
    t, s, dy = case(3, 4, 2, 200, 200, 16, causal=True, bias=True)
    whole = rg.attention(**t, **s)
    for i in (0, 63, 64, 130, 199):
        one = rg.attention(t["q"][1:2, i:i + 1], t["k"][1:2, :i + 1], t["v"][1:2, :i + 1],
                           relative_bias=t["relative_bias"][:, 199 - i:200].contiguous())
        assert torch.equal(one[0, 0], whole[1, i])
    padded = torch.nn.functional.pad(t["k"], (0, 0, 0, 0, 0, 300)), torch.nn.functional.pad(t["v"], (0, 0, 0, 0, 0, 300))
    bias = torch.nn.functional.pad(t["relative_bias"], (0, 300))
    assert torch.equal(rg.attention(t["q"], *padded, key_lengths=torch.tensor([200] * 3), causal=True, relative_bias=bias), whole)


def test_any_strides_and_no_values():
    t, s, dy = case(2, 4, 2, 9, 30, 12)
    want = gradients(t, s, dy)
    kv = torch.stack((t["k"], t["v"]), 2)
    odd = torch.zeros(2, 9, 4, 13)[..., 1:]
    odd.copy_(t["q"])
    for q, k, v in ((odd, kv[:, :, 0], kv[:, :, 1]),
                    (t["q"].permute(3, 2, 1, 0).contiguous().permute(3, 2, 1, 0), t["k"].transpose(1, 2).contiguous().transpose(1, 2), t["v"])):
        got = gradients({"q": q, "k": k, "v": v, "relative_bias": None}, s, dy)
        assert all(torch.equal(got[n], want[n]) for n in want)
    for b, tq, tk in ((0, 4, 5), (2, 0, 5), (2, 4, 0), (0, 0, 0)):
        t, s, dy = case(b, 2, 1, tq, tk, 8, bias=True, causal=True)
        got = gradients(t, s, dy)
        assert all(torch.all(x == 0) for x in got.values()) and got["dk"].shape == t["k"].shape


def test_one_key_for_every_query():
    """Expanded operands: strides of 0."""
    t, s, dy = case(1, 2, 2, 5, 40, 8)
    t["k"], t["v"] = (x.expand(3, 40, 2, 8) for x in (t["k"], t["v"]))
    t["q"], dy = t["q"].expand(3, 5, 2, 8).contiguous(), dy.expand(3, 5, 2, 8).contiguous()
    y = rg.attention(**t, **s)
    assert torch.equal(y[0], y[2])
    check(gradients(t, s, dy), t, s, dy)


def test_a_second_gradient_is_refused():
    t, s, dy = case(1, 1, 1, 3, 3, 4)
    q = t["q"].requires_grad_()
    (g,) = torch.autograd.grad(rg.attention(q, t["k"], t["v"]), q, dy, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable"):
        g.sum().backward()


def refused(match, **change):
    t = {n: torch.zeros(2, 4, 2, 8) for n in ("q", "k", "v")}
    t.update(change)
    with pytest.raises(ValueError, match=match):
        rg.attention(**t)


def test_refusals():
    z = torch.zeros
    refused("float32", q=z(2, 4, 2, 8, dtype=torch.float64))
    refused("float32", v=z(2, 4, 2, 8, dtype=torch.bfloat16))
    refused("batch, positions", k=z(4, 2, 8))
    refused("one shape", v=z(2, 5, 2, 8))
    refused("one shape", k=z(3, 4, 2, 8), v=z(3, 4, 2, 8))
    refused("1 to 128", **{n: z(2, 4, 2, 129) for n in "qkv"})
    refused("1 to 128", **{n: z(2, 4, 2, 0) for n in "qkv"})
    refused("divide", k=z(2, 4, 3, 8), v=z(2, 4, 3, 8))
    refused("divide", k=z(2, 4, 0, 8), v=z(2, 4, 0, 8))
    refused("finite", scale=math.nan)
    refused("finite", scale=1e300)
    refused(r"\[0, 1\)", dropout=1.0)
    refused(r"\[0, 1\)", dropout=-0.1)
    refused(r"\[0, 1\)", dropout=math.nan)
    refused("key_lengths", key_lengths=torch.tensor([4]))
    refused("key_lengths", key_lengths=torch.tensor([4.0, 4.0]))
    refused("bool", mask=z(4, 4))
    refused("broadcast", mask=z(3, 4, dtype=torch.bool))
    refused("4 dimensions", mask=z(1, 1, 1, 4, 4, dtype=torch.bool))
    refused("relative_bias must be", relative_bias=z(2, 8))
    refused("relative_bias must be", relative_bias=z(1, 7))
    refused("seed", dropout=0.1, seed=torch.tensor([1, 2]))
    refused("same device", k=z(2, 4, 2, 8, device="meta"))


def test_the_layer_is_its_parts():
    torch.manual_seed(3)
    layer = rg.Attention(24, 4, num_kv_heads=2, states_width=10, dropout=0.3)
    bias = rg.RelativePositionBias(4, num_buckets=8, max_distance=20)
    x, states = torch.randn(2, 6, 24), torch.randn(2, 9, 10)
    lengths = torch.tensor([9, 4])
    y = layer(x, states, key_lengths=lengths, relative_bias=bias(6, 9), seed=5)
    q = layer.query(x).view(2, 6, 4, 6)
    k, v = layer.key_value(states).view(2, 9, 2, 2, 6).unbind(2)
    want = layer.out(rg.attention(q, k, v, key_lengths=lengths, relative_bias=bias(6, 9), dropout=0.3, seed=5).reshape(2, 6, 24))
    assert torch.equal(y, want)
    y.sum().backward()
    assert all(p.grad is not None and p.grad.isfinite().all() for m in (layer, bias) for p in m.parameters())
    torch.manual_seed(4)
    a = layer(x, states)
    torch.manual_seed(4)
    assert torch.equal(a, layer(x, states)) and not torch.equal(a, layer(x, states))
    layer.eval()
    assert torch.equal(layer(x, states), layer(x, states))
    for bad in (dict(width=10, num_heads=3), dict(width=12, num_heads=4, num_kv_heads=3), dict(width=256, num_heads=1),
                dict(width=12, num_heads=4, dropout=1.0)):
        with pytest.raises(ValueError):
            rg.Attention(**bad)


def test_transforms_raise_an_error():
    q = torch.randn(2, 3, 1, 4)
    table = torch.randn(8, 2)
    for f, x in ((lambda x: rg.attention(x, x, x), q), (lambda x: rg.dropout(x, 0.5, seed=1), q),
                 (lambda x: rg.relative_position_bias(x, 3, 3, max_distance=9), table)):
        with pytest.raises(Exception):
            torch.func.grad(lambda x: f(x).sum())(x)
        with pytest.raises(Exception):
            torch.func.jvp(f, (x,), (x,))
        with pytest.raises(Exception):
            torch.func.vmap(f)(x[None])


def test_modules_on_the_meta_device():
    with torch.device("meta"):
        rg.Attention(8, 2), rg.RelativePositionBias(2), rg.Dropout(0.1)
