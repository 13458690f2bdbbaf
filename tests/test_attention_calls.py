"""Calls of attention that its documents allow: starts, sizes, operands and surroundings at their ends, on the CPU and on the GPU."""
import pytest
import torch

import bit_reproducible_training_amd as rg
from test_attention import case, gradients

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def to(device, t):
    return {n: v.to(device) if isinstance(v, torch.Tensor) else v for n, v in t.items()}


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("tq,tk", [(1, 40), (3, 300), (70, 90)])
def test_a_start_past_every_key_sees_all_and_one_before_sees_none(device, tq, tk):
    t, s, dy = case(2, 2, 1, tq, tk, 8, bias=True)
    want = gradients(t, s, dy)
    for start in (tk, 2 ** 32 + 1, 2 ** 62, 2 ** 63 - 1):
        got = gradients(to(device, t), {**s, "causal": True, "query_start": start}, dy.to(device))
        assert all(torch.equal(got[n].cpu(), want[n]) for n in want), start
    for start in (-tq, -2 ** 32 - 1, -2 ** 63):
        got = gradients(to(device, t), {**s, "causal": True, "query_start": start}, dy.to(device))
        assert all(torch.all(x == 0) for x in got.values()), start


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["x", "states", "relative_bias"])
def test_the_layer_refuses_a_capture_beside_an_eager_graph_of_an_operand(which):
    """(The layer's own parameters have none.)"""
    layer = rg.Attention(16, 2).cuda()
    t = {"x": torch.randn(1, 5, 16, device="cuda"), "states": torch.randn(1, 7, 16, device="cuda"),
         "relative_bias": torch.randn(2, 11, device="cuda")}
    t[which].requires_grad_()
    alive = t[which] * 2
    torch.cuda.synchronize()
    refused = None
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        torch.zeros(4, device="cuda").add_(1)
        try:
            layer(**t)
        except ValueError as e:
            refused = str(e)
        with torch.no_grad():
            layer(**t)
    assert "still alive" in refused
    del alive
    want = torch.autograd.grad(layer(**t).sum(), t[which])[0]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(layer(**t).sum(), t[which])[0]
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_a_capture_is_asked_for_where_there_can_be_one():
    from bit_reproducible_training_amd._lib import _backend

    assert not _backend.capturing(torch.zeros(1))


def each_alone(t, s, dy, of, index):
    """{y, d...} of the slices of dimension `of` (0: items, 2: heads of queries) that `index` names, by themselves."""
    cut = lambda x: None if x is None else x[index:index + 1] if of == 0 else x[:, :, index:index + 1]
    own = {n: cut(x) if of == 0 or n == "q" else x for n, x in t.items()}
    if of == 2 and t["relative_bias"] is not None:
        own["relative_bias"] = t["relative_bias"][index:index + 1]
    return gradients(own, s, cut(dy))


@pytest.mark.gpu
def test_a_gradient_of_many_items_over_many_key_blocks():
    """2^18 heads over 32 blocks of keys: 2^23 in all, which takes two turns."""
    g = torch.Generator(device="cuda").manual_seed(1)
    t = {"q": torch.randn(2048, 1, 128, 1, device="cuda", generator=g), "relative_bias": None,
         **{n: torch.randn(2048, 4096, 1, 1, device="cuda", generator=g) for n in "kv"}}
    dy = torch.randn(2048, 1, 128, 1, device="cuda", generator=g)
    got = gradients(t, {}, dy)
    for b in (0, 1000, 2047):
        alone = each_alone(t, {}, dy, 0, b)
        assert all(torch.equal(got[n][b], alone[n][0]) for n in alone), b


@pytest.mark.gpu
def test_a_bias_gradient_of_many_heads_and_distances():
    """2^15 heads of 257 x 64 distances."""
    g = torch.Generator(device="cuda").manual_seed(2)
    t = {"q": torch.randn(1, 1, 2 ** 15, 1, device="cuda", generator=g), "relative_bias": torch.randn(2 ** 15, 16385, device="cuda", generator=g),
         **{n: torch.randn(1, 16385, 1, 1, device="cuda", generator=g) for n in "kv"}}
    dy = torch.randn(1, 1, 2 ** 15, 1, device="cuda", generator=g)
    got = gradients(t, {}, dy)
    for h in (0, 20000, 2 ** 15 - 1):
        alone = each_alone(t, {}, dy, 2, h)
        assert torch.equal(got["drelative_bias"][h], alone["drelative_bias"][0]) and torch.equal(got["dq"][:, :, h], alone["dq"][:, :, 0])


@pytest.mark.gpu
def test_many_single_queries_over_many_chunks_of_keys():
    """2^15 items by 258 chunks of the same keys: more than 2^23 blocks, which takes two launches."""
    g = torch.Generator(device="cuda").manual_seed(3)
    q = torch.randn(2 ** 15, 1, 1, 1, device="cuda", generator=g)
    k, v = (torch.randn(1, 65793, 1, 1, device="cuda", generator=g) for _ in range(2))
    y = rg.attention(q, k.expand(2 ** 15, -1, -1, -1), v.expand(2 ** 15, -1, -1, -1))
    for b in (0, 20000, 2 ** 15 - 1):
        assert torch.equal(y[b], rg.attention(q[b:b + 1], k, v)[0])


@pytest.mark.gpu
def test_many_items_of_many_queries():
    """2^20 items of 9 blocks of queries, and a NaN that the last queries of the last items alone see."""
    g = torch.Generator(device="cuda").manual_seed(4)
    n = 2 ** 20
    q, k = torch.randn(1, 1025, 1, 1, device="cuda", generator=g), torch.randn(1, 3, 1, 1, device="cuda", generator=g)
    v = torch.randn(1, 3, 1, 1, device="cuda", generator=g).repeat(n, 1, 1, 1)
    s = dict(causal=True, query_start=-1000)
    want = rg.attention(q, k, v[:1], **s)
    v[-5:, 2] = float("nan")
    y = rg.attention(q.expand(n, -1, -1, -1), k.expand(n, -1, -1, -1), v, **s)
    assert (y[:-5] == want).all()
    assert (y[-5:, :1002] == want[:, :1002]).all() and y[-5:, 1002:].isnan().all()


@pytest.mark.gpu
def test_a_table_of_many_heads_and_buckets():
    """1026 buckets of 2^14 heads: more sums than a launch has blocks. (Only the C entry takes so many heads.)"""
    import ctypes

    from bit_reproducible_training_amd import _lib

    h, count = 2 ** 14, 512
    borders = (ctypes.c_int * count)(*range(1, count + 1))
    c = _lib.rg_relative_bias_config(3, 700, 0, h, count, 1, 0, borders)
    dout = torch.randn(h, 702, device="cuda")
    out = torch.full((1026, h), 7.0, device="cuda")
    torch.cuda.synchronize()
    assert _lib.lib.rg_relative_bias_grad_fp32(ctypes.byref(c), dout.data_ptr(), out.data_ptr(), None, 0, None) == 0
    torch.cuda.synchronize()
    want = torch.zeros(1026, h, device="cuda")
    want[:3] = dout[:, [2, 1, 0]].t()  # distances 0, -1 and -2
    want[514:514 + 511] = dout[:, 3:3 + 511].t()  # 1 to 511
    assert torch.equal(out[:1025], want[:1025])
    size = dout[:, 514:].double()
    assert torch.all((out[1025].double() - size.sum(1)).abs() <= 20 * 2.0 ** -24 * size.abs().sum(1))  # 188 in 256 strands and a tree


@pytest.mark.parametrize("device", DEVICES)
def test_gradients_of_some_operands(device):
    """Each alone, and each pair, as with all of them."""
    t, s, dy = case(2, 4, 2, 40, 70, 16, causal=True, lengths=True, bias=True, drop=0.1)
    t, s, dy = to(device, t), to(device, s), dy.to(device)
    want = gradients(t, s, dy)
    names = list(t)
    for some in [{a} for a in names] + [{a, b} for a in names for b in names if a < b]:
        own = {n: x.detach().requires_grad_(n in some) for n, x in t.items()}
        leaves = [own[n] for n in names if n in some]
        got = torch.autograd.grad(rg.attention(**own, **s), leaves, dy)
        assert all(torch.equal(g, want["d" + n]) for g, n in zip(got, [n for n in names if n in some])), some


def windows(x, tk, d):
    """Keys that overlap: key j is values j .. j + d - 1 of x."""
    return x.as_strided((1, tk, 1, d), (0, 1, 0, 1))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("tq", [1, 6, 40])
def test_a_value_that_is_not_finite_stays_in_its_place(device, value, tq):
    """One key, keys at one address and keys that overlap, where rows past the last lie in the same memory: a visible value that is not finite
    reaches the outputs that it belongs to, as it is, and no others."""
    g = torch.Generator().manual_seed(tq)
    q, x = torch.randn(1, tq, 1, 8, generator=g), torch.randn(200, generator=g)
    x[20] = value
    dy = torch.randn(1, tq, 1, 8, generator=g)
    one = torch.randn(1, 1, 1, 8, generator=g)
    one[..., 3] = value
    for name, v in (("one key", one), ("one address", one.expand(1, 70, 1, 8)), ("overlapping", windows(x, 21, 8)),
                    ("past the length", windows(x, 90, 8))):
        k = torch.randn(v.shape, generator=g)
        lengths = torch.tensor([15]) if name == "past the length" else None
        seen = v.shape[1] if lengths is None else 15
        t = {"q": q, "k": k, "v": v, "relative_bias": None}
        want = gradients({**t, "v": v.contiguous()}, {"key_lengths": lengths}, dy)
        on = {n: None if a is None else a.to(device) for n, a in t.items()}
        if name != "one key":  # (to() lays them out anew)
            on["v"] = one.to(device).expand(1, 70, 1, 8) if name == "one address" else windows(x.to(device), v.shape[1], 8)
        y = rg.attention(on["q"], on["k"], on["v"], key_lengths=None if lengths is None else lengths.to(device)).cpu()
        for d in range(8):
            column = v[0, :seen, 0, d]
            if column.isfinite().all():
                assert y[..., d].isfinite().all(), (name, d)
            else:
                assert torch.all(y[..., d].isnan() if value != value else y[..., d] == value), (name, d)
        got = gradients(on, {"key_lengths": None if lengths is None else lengths.to(device)}, dy.to(device))
        for n in ("y", "dq", "dk", "dv"):
            a, b = got[n].cpu(), want[n]
            if n in ("dk", "dv") and a.shape != b.shape:
                continue
            assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)), (name, n)
