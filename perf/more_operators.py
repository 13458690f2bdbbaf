"""The operators of a training step that let positions of a sequence look at others, as they are
measured: attention to states of the same or another length, the learned bias of relative positions
by buckets, and dropout from a counter-based generator.

A case is a dict of plain values; its "op" says which operator it is:
  attend   q [b, tq, h, d], k and v [b, tk, kvh, d] -> y [b, tq, h, d]; with "train", the gradients of q, k, v
           (and of the bias's table) for a given gradient of y too
  bias     table [buckets, h] -> [h, tq, tk]; with "train", the table's gradient for a given gradient of that
  dropout  x [n, d] -> y; with "train", x's gradient for a given gradient of y

Where `own` is false, run() computes them with elementary torch operations in float32.

The dropout's bits are Philox 4x32-10's (Salmon et al., 2011): four 32-bit words from a counter of four words and the
seed's two as the key. A value is kept where its word is at least p 2^32. Value e of a tensor has word e mod 4 of the counter
(e / 4, e / 2^34, 0, 0); the pair of query i and key j of head t (counted through the batch) has word j mod 4 of (j / 4, i, t, 1).
"""
import math

import torch

own = False


def _attend(name, b, h, kvh, tq, tk, d, causal=False, mask="none", bias=0, drop=0.0, train=True):
    """mask: "none", "lengths" (each sequence's number of keys) or "pairs" (truth values [b, 1, tq, tk] that leave some
    queries nothing). bias: buckets of a learned bias, or 0. Causal queries stand at the last tq of the tk positions."""
    return {"name": name, "op": "attend", "b": b, "h": h, "kvh": kvh, "tq": tq, "tk": tk, "d": d, "causal": causal,
            "mask": mask, "bias": bias, "drop": drop, "train": train}


def _bias(name, h, tq, tk, buckets, both, train):
    return {"name": name, "op": "bias", "h": h, "tq": tq, "tk": tk, "buckets": buckets, "both": both, "train": train}


def _dropout(name, n, d, drop, train):
    return {"name": name, "op": "dropout", "n": n, "d": d, "drop": drop, "train": train}


def listed():
    return [
        # A decoder's token looks at a short encoded sentence: the smallest call, where latency counts.
        _attend("one query of 77 keys", 1, 12, 12, 1, 77, 64, mask="lengths", train=False),
        # A batch's next tokens look at long encoded documents, of differing lengths.
        _attend("next tokens, long states", 16, 12, 12, 1, 4096, 64, mask="lengths", train=False),
        # The self attention of a small decoder in training: 8 sequences of 1024 tokens, 12 heads.
        _attend("decoder, 1024 tokens", 8, 12, 12, 1024, 1024, 64, causal=True, bias=32, drop=0.1),
        # Its cross attention to an encoder's padded states of another length.
        _attend("cross, 512 to 1500", 8, 12, 12, 512, 1500, 64, mask="lengths", drop=0.1),
        # Wide heads that share keys and values, long sequences.
        _attend("shared keys, 2048 tokens", 4, 16, 4, 2048, 2048, 128, causal=True),
        # An encoder over long sequences without a mask: the largest products.
        _attend("encoder, 4096 tokens", 2, 16, 16, 4096, 4096, 64, bias=32),
        # Odd sizes and a mask of pairs with empty rows, as packed or structured inputs have.
        _attend("odd sizes, pairs masked", 3, 5, 5, 333, 1001, 80, mask="pairs"),
        # The bias for an attention that takes it dense, with its gradient; and one new token's row of it.
        _bias("bias 1024 x 1024", 12, 1024, 1024, 32, True, True),
        _bias("bias of one row", 12, 1, 513, 32, False, False),
        # Dropout of a block's output in a small model's step, of a few rows, and of a wide hidden layer.
        _dropout("dropout 8192 x 768", 8192, 768, 0.1, True),
        _dropout("dropout 63 x 127", 63, 127, 0.5, False),
        _dropout("dropout 32768 x 2048", 32768, 2048, 0.1, True),
    ]


def draw(rng):
    def log_int(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    op = rng.choice(("attend", "attend", "attend", "bias", "dropout"))
    if op == "bias":
        h, tq, tk = rng.choice((1, 5, 12, 16)), log_int(1, 1500), log_int(1, 1500)
        return _bias(None, h, tq, tk, 2 * rng.randint(4, 32), rng.random() < 0.5, rng.random() < 0.6)
    if op == "dropout":
        return _dropout(None, log_int(1, 16384), log_int(16, 4096), rng.choice((0.1, 0.25, 0.5)), rng.random() < 0.6)
    kvh, group = rng.choice((1, 2, 4, 8)), rng.choice((1, 1, 2, 4))
    d = rng.choice((16, 32, 40, 64, 64, 80, 96, 128))
    tk = log_int(1, 4096)
    causal = rng.random() < 0.4
    tq = rng.choice((1, log_int(1, 2048)))
    if causal:
        tq = min(tq, tk)
    mask = rng.choice(("none", "none", "lengths", "pairs"))
    b = rng.randint(1, 8)
    while b > 1 and b * kvh * group * tq * tk > 1 << 26:
        b -= 1
    while kvh > 1 and b * kvh * group * tq * tk > 1 << 26:
        kvh //= 2
    train = rng.random() < 0.6
    return _attend(None, b, kvh * group, kvh, tq, tk, d, causal, mask, rng.choice((0, 0, 32)), rng.choice((0.0, 0.1)) if train else 0.0,
                   train)


# ---- inputs ----

def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed * 1000003 + 17)

    def normal(*size, std=1.0):
        return torch.randn(*size, generator=gen, device="cuda") * std

    s = {"case": case, "seed": (seed * 0x9E3779B97F4A7C15 + 0x1234567) % (1 << 63)}
    if case["op"] == "dropout":
        s["x"] = normal(case["n"], case["d"])
        s["dy"] = normal(case["n"], case["d"]) if case["train"] else None
        s["leaves"] = [s["x"]]
    elif case["op"] == "bias":
        s["table"] = normal(case["buckets"], case["h"])
        s["dy"] = normal(case["h"], case["tq"], case["tk"], std=0.01) if case["train"] else None
        s["leaves"] = [s["table"]]
    else:
        b, tq, tk, h, kvh, d = (case[n] for n in ("b", "tq", "tk", "h", "kvh", "d"))
        # keys and values come out of one projection of the states, as a layer makes them
        kv = normal(b, tk, 2, kvh, d)
        s["q"], s["k"], s["v"] = normal(b, tq, h, d), kv[:, :, 0], kv[:, :, 1]
        s["table"] = normal(case["bias"], h) if case["bias"] else None
        s["lengths"] = s["mask"] = None
        if case["mask"] == "lengths":
            s["lengths"] = torch.randint((tk + 1) // 2, tk + 1, (b,), generator=gen, device="cuda")
        elif case["mask"] == "pairs":
            s["mask"] = torch.rand(b, 1, tq, tk, generator=gen, device="cuda") < 0.7
            s["mask"][:, :, 8::17] = False
            s["mask"][:, :, 0, 0] = True
        s["dy"] = normal(b, tq, h, d) if case["train"] else None
        s["leaves"] = [t for t in (s["q"], s["k"], s["v"], s["table"]) if t is not None]
    if case["train"]:
        s["leaves"] = [t.requires_grad_() for t in s["leaves"]]
    return s


# ---- plain forms ----

def _philox(c0, c1, c2, c3, seed):
    """The four words (in int64) of counters that broadcast against each other."""
    low = 0xFFFFFFFF
    k0, k1 = seed & low, seed >> 32
    c0, c1, c2, c3 = torch.broadcast_tensors(c0, c1, c2, c3)
    for _ in range(10):
        # the products pass 2^63: int64 wraps, and its two halves are those of the unsigned product
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & low) ^ c1 ^ k0, b & low, ((a >> 32) & low) ^ c3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return c0, c1, c2, c3


def _words(*args):
    return torch.stack(_philox(*args), dim=-1).flatten(-2)


def _number(value, device):
    return torch.tensor(value, dtype=torch.int64, device=device)


def _kept_values(shape, drop, seed, device):
    n = math.prod(shape)
    group = torch.arange((n + 3) // 4, device=device)
    zero = _number(0, device)
    return (_words(group & 0xFFFFFFFF, group >> 32, zero, zero, seed)[:n] >= int(drop * 2.0 ** 32)).view(shape)


def _kept_pairs(heads, tq, tk, drop, seed, device):
    """[heads, tq, tk]"""
    def count(n):
        return torch.arange(n, device=device)
    words = _words(count((tk + 3) // 4)[None, None, :], count(tq)[None, :, None], count(heads)[:, None, None], _number(1, device), seed)
    return words[..., :tk] >= int(drop * 2.0 ** 32)


def _borders(buckets, max_distance):
    """The distances at which the next of `buckets` begins: one each up to buckets / 2, then evenly in the logarithm up
    to max_distance. (n / exact)^steps >= (max_distance / exact)^t, in whole numbers."""
    exact = buckets // 2
    steps, found = buckets - exact, list(range(1, exact + 1))
    n = exact
    for t in range(1, steps):
        while n ** steps * exact ** t < max_distance ** t * exact ** steps:
            n += 1
        found.append(n)
    return found


def _buckets(tq, tk, start, buckets, both, device):
    """[tq, tk]: the bucket of key j seen from the query at position start + i."""
    relative = torch.arange(tk, device=device)[None, :] - (torch.arange(tq, device=device) + start)[:, None]
    side = buckets // 2 if both else buckets
    distance = relative.abs() if both else (-relative).clamp(min=0)
    borders = torch.tensor(_borders(side, 128), device=device)
    at = torch.searchsorted(borders, distance.contiguous(), right=True)
    return at + side * (relative > 0) if both else at


def _visible(s):
    """What a pair of query and key needs to be seen, broadcast to [b, 1, tq, tk], or None."""
    case, seen = s["case"], None
    tq, tk, device = case["tq"], case["tk"], s["q"].device
    if case["causal"]:
        ahead = torch.arange(tk, device=device)[None, :] - torch.arange(tq, device=device)[:, None]
        seen = (ahead <= tk - tq)[None, None]
    if s["lengths"] is not None:
        within = (torch.arange(tk, device=device) < s["lengths"][:, None])[:, None, None, :]
        seen = within if seen is None else seen & within
    if s["mask"] is not None:
        seen = s["mask"] if seen is None else seen & s["mask"]
    return seen


def _start(case):
    return case["tk"] - case["tq"] if case["causal"] else 0


def _plain_attend(s):
    case = s["case"]
    b, tq, tk, h, kvh, d = (case[n] for n in ("b", "tq", "tk", "h", "kvh", "d"))
    with torch.no_grad():
        group, scale = h // kvh, 1.0 / math.sqrt(d)
        q = s["q"].transpose(1, 2).reshape(b * h, tq, d)
        k, v = (t.transpose(1, 2).repeat_interleave(group, 1).reshape(b * h, tk, d) for t in (s["k"], s["v"]))
        z = torch.matmul(q, k.transpose(1, 2).contiguous()).view(b, h, tq, tk) * scale
        if case["bias"]:
            bucket = _buckets(tq, tk, _start(case), case["bias"], not case["causal"], z.device)
            z = z + s["table"].t()[:, bucket]
        seen = _visible(s)
        if seen is not None:
            z = torch.where(seen, z, -math.inf)
        top = z.amax(-1, keepdim=True)
        e = torch.exp(z - torch.where(top == -math.inf, 0.0, top))
        total = e.sum(-1, keepdim=True)
        p = e / torch.where(total == 0, 1.0, total)
        del z, e
        factor, used = 1.0 / (1.0 - case["drop"]), p
        if case["drop"]:
            kept = _kept_pairs(b * h, tq, tk, case["drop"], s["seed"], p.device).view(b, h, tq, tk)
            used = torch.where(kept, p * factor, 0.0)
        y = torch.matmul(used.view(b * h, tq, tk), v)
        out = y.view(b, h, tq, d).transpose(1, 2).contiguous()
        if not case["train"]:
            return (out,)
        dy = s["dy"].transpose(1, 2).reshape(b * h, tq, d)
        dv = torch.matmul(used.view(b * h, tq, tk).transpose(1, 2), dy)
        dp = torch.matmul(dy, v.transpose(1, 2).contiguous()).view(b, h, tq, tk)
        if case["drop"]:
            dp = torch.where(kept, dp * factor, 0.0)
        ds = p * (dp - (p * dp).sum(-1, keepdim=True))
        del dp, used
        flat = ds.view(b * h, tq, tk)
        dq = torch.matmul(flat, k) * scale
        dk = torch.matmul(flat.transpose(1, 2), q) * scale
        grads = [dq.view(b, h, tq, d).transpose(1, 2).contiguous()]
        grads += [t.view(b, kvh, group, tk, d).sum(2).transpose(1, 2).contiguous() for t in (dk, dv)]
        if case["bias"]:
            grads.append(_table_gradient(ds.sum(0), bucket, case["bias"]))
        return (out, *grads)


def _table_gradient(dy, bucket, buckets):
    """dy [h, tq, tk], bucket [tq, tk] -> [buckets, h]. A pair's distance is its column once each row is moved one place
    further than the row below it."""
    h, tq, tk = dy.shape
    moved = torch.nn.functional.pad(dy.flip(1), (0, tq)).flatten(1)[:, :tq * (tq + tk - 1)]
    by_distance = moved.view(h, tq, tq + tk - 1).sum(1)
    of_distance = torch.cat((bucket[:, 0].flip(0), bucket[0, 1:]))
    return torch.stack([torch.where(of_distance == n, by_distance, 0.0).sum(1) for n in range(buckets)])


def _plain(s):
    case = s["case"]
    if case["op"] == "attend":
        return _plain_attend(s)
    with torch.no_grad():
        if case["op"] == "bias":
            bucket = _buckets(case["tq"], case["tk"], case["tk"] - case["tq"], case["buckets"], case["both"], s["table"].device)
            y = s["table"].t()[:, bucket].contiguous()
            return (y, _table_gradient(s["dy"], bucket, case["buckets"])) if case["train"] else (y,)
        kept = _kept_values(s["x"].shape, case["drop"], s["seed"], s["x"].device)
        factor = 1.0 / (1.0 - case["drop"])
        y = torch.where(kept, s["x"] * factor, 0.0)
        return (y, torch.where(kept, s["dy"] * factor, 0.0)) if case["train"] else (y,)


# ---- the framework's operators ----

def _own(s):
    import bit_reproducible_training_amd as rg

    case = s["case"]
    if case["op"] == "attend":
        bias = None
        if case["bias"]:
            bias = rg.relative_position_bias(s["table"], case["tq"], case["tk"], max_distance=128, bidirectional=not case["causal"],
                                             query_start=_start(case), dense=False)
        y = rg.attention(s["q"], s["k"], s["v"], causal=case["causal"], query_start=_start(case), key_lengths=s["lengths"],
                         mask=s["mask"], relative_bias=bias, dropout=case["drop"], seed=s["seed"])
    elif case["op"] == "bias":
        y = rg.relative_position_bias(s["table"], case["tq"], case["tk"], max_distance=128, bidirectional=case["both"],
                                      query_start=case["tk"] - case["tq"])
    else:
        y = rg.dropout(s["x"], case["drop"], seed=s["seed"])
    if not case["train"]:
        return (y,)
    return (y.detach(), *torch.autograd.grad(y, s["leaves"], s["dy"]))


def run(state):
    return _own(state) if own else _plain(state)


# ---- what a pass cannot do without ----

def work(case):
    if case["op"] == "dropout":
        return {"bytes": 8 * case["n"] * case["d"] * (2 if case["train"] else 1), "flops": 0}
    if case["op"] == "bias":
        return {"bytes": 4 * case["h"] * case["tq"] * case["tk"] * (2 if case["train"] else 1), "flops": 0}
    b, tq, tk, h, kvh, d = (case[n] for n in ("b", "tq", "tk", "h", "kvh", "d"))
    pairs = tq * (tk - tq) + tq * (tq + 1) // 2 if case["causal"] else tq * tk
    if case["mask"] != "none":  # three quarters of the keys, or 0.7 of the pairs, on average
        pairs = pairs * 3 // 4
    values = 2 * b * tq * h * d + 2 * b * tk * kvh * d
    if case["train"]:  # reads y and its gradient too, writes three more
        values += 2 * b * tq * h * d + 2 * b * tk * kvh * d
    return {"bytes": 4 * values, "flops": (14 if case["train"] else 4) * b * h * pairs * d}


# ---- in 64 bits, from the definitions ----

def _exact_kept(counters, seed, drop):
    """counters: four int64 tensors -> which of the four words are at least drop 2^32, stacked last. The 64-bit products are
    taken from halves of 16 bits."""
    x = [t.clone() for t in torch.broadcast_tensors(*counters)]
    key = [seed % 2 ** 32, seed // 2 ** 32]

    def product(t, m):
        high_m, low_m = divmod(m, 65536)
        first = t * low_m
        second = t * high_m + (first >> 16)
        return second >> 16, ((second & 65535) << 16) | (first & 65535)

    for turn in range(10):
        k0, k1 = (key[0] + turn * 0x9E3779B9) % 2 ** 32, (key[1] + turn * 0xBB67AE85) % 2 ** 32
        high0, low0 = product(x[0], 0xD2511F53)
        high1, low1 = product(x[2], 0xCD9E8D57)
        x = [high1 ^ x[1] ^ k0, low1, high0 ^ x[3] ^ k1, low0]
    return torch.stack([t.double() >= math.floor(drop * 4294967296.0) for t in x], -1)


def _exact_bucket(relative, buckets, both):
    """The bucket of a relative position (key less query), from its definition; a distance that ends a step exactly belongs to the next."""
    side, at = (buckets // 2, buckets // 2 if relative > 0 else 0) if both else (buckets, 0)
    n = abs(relative) if both else max(0, -relative)
    exact = side // 2
    if n < exact:
        return at + n
    steps = side - exact
    t = min(steps - 1, int(steps * math.log(n / exact) / math.log(128 / exact)) + 2)
    while t > 0 and n ** steps * exact ** t < 128 ** t * exact ** steps:
        t -= 1
    return at + exact + t


def _exact_bias(table, tq, tk, start, both):
    """(bias [h, tq, tk] in 64 bits, the buckets of the distances tk - 1 - start .. -(tq - 1) - start, where each pair's is)"""
    by_distance = torch.tensor([_exact_bucket(r, table.shape[0], both) for r in range(-(tq - 1) - start, tk - start)], device=table.device)
    place = torch.arange(tk, device=table.device)[None, :] + (tq - 1 - torch.arange(tq, device=table.device))[:, None]
    return table.detach().double()[by_distance[place]].permute(2, 0, 1), by_distance, place


def _exact_sums(dy, by_distance, place, buckets):
    """The sums of dy [tq, tk] over each bucket"""
    diagonal = torch.zeros(len(by_distance), dtype=torch.float64, device=dy.device).index_add_(0, place.flatten(), dy.flatten())
    return torch.zeros(buckets, dtype=torch.float64, device=dy.device).index_add_(0, by_distance, diagonal)


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return _exact(case, s)


def _exact(case, s):
    if case["op"] == "dropout":
        n = case["n"] * case["d"]
        e = torch.arange(-(-n // 4), device="cuda")
        zero = torch.zeros((), dtype=torch.int64, device="cuda")
        kept = _exact_kept((e % 2 ** 32, e // 2 ** 32, zero, zero), s["seed"], case["drop"]).flatten()[:n].view(case["n"], case["d"])
        outs = [s["x"]] + ([s["dy"]] if case["train"] else [])
        return tuple(kept * (t.double() / (1.0 - case["drop"])) for t in outs)
    if case["op"] == "bias":
        y, by_distance, place = _exact_bias(s["table"], case["tq"], case["tk"], case["tk"] - case["tq"], case["both"])
        if not case["train"]:
            return (y,)
        return y, torch.stack([_exact_sums(s["dy"][t].double(), by_distance, place, case["buckets"]) for t in range(case["h"])], 1)
    b, tq, tk, h, kvh, d = (case[n] for n in ("b", "tq", "tk", "h", "kvh", "d"))
    q, k, v = (s[n].double() for n in "qkv")
    y, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros(b, tk, kvh, d, dtype=q.dtype, device=q.device), None
    dv = torch.zeros_like(dk)
    offset = tk - tq if case["causal"] else 0
    if case["bias"]:
        bias, by_distance, place = _exact_bias(s["table"], tq, tk, offset, not case["causal"])
        dtable = torch.zeros(case["bias"], h, dtype=q.dtype, device=q.device)
    rows, keys = torch.arange(tq, device=q.device)[:, None], torch.arange(tk, device=q.device)[None, :]
    for item in range(b):
        for head in range(h):
            shared = head * kvh // h
            z = q[item, :, head] @ k[item, :, shared].t() / math.sqrt(d)
            if case["bias"]:
                z = z + bias[head]
            hidden = torch.zeros(tq, tk, dtype=torch.bool, device=q.device)
            if case["causal"]:
                hidden |= keys > rows + offset
            if s["lengths"] is not None:
                hidden |= keys >= s["lengths"][item]
            if s["mask"] is not None:
                hidden |= ~s["mask"][item, 0]
            z[hidden] = -1e300  # against a row's largest this is e^-infinity; rows without any are cleared below
            p = torch.softmax(z, -1)
            p[hidden] = 0
            share = torch.ones((), dtype=q.dtype, device=q.device)
            if case["drop"]:
                counters = (torch.arange(-(-tk // 4), device=q.device)[None, :], rows, torch.full_like(rows, item * h + head),
                            torch.ones_like(rows))
                share = _exact_kept(counters, s["seed"], case["drop"]).flatten(-2)[:, :tk] / (1.0 - case["drop"])
            y[item, :, head] = (p * share) @ v[item, :, shared]
            if not case["train"]:
                continue
            g = s["dy"][item, :, head].double()
            dv[item, :, shared] += (p * share).t() @ g
            dz = p * (share * (g @ v[item, :, shared].t()) - (g * y[item, :, head]).sum(-1, keepdim=True))
            dq[item, :, head] = dz @ k[item, :, shared] / math.sqrt(d)
            dk[item, :, shared] += dz.t() @ q[item, :, head] / math.sqrt(d)
            if case["bias"]:
                dtable[:, head] += _exact_sums(dz, by_distance, place, case["bias"])
    if not case["train"]:
        return (y,)
    return (y, dq, dk, dv, dtable) if case["bias"] else (y, dq, dk, dv)
