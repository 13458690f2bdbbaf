"""The operators of a language model's training step around its matrix products, as they are
measured: the loss of a vocabulary projection with its gradients, the residual addition with the
norms before and after a block, and the optimizer's step.

A case is a dict of plain values; its "op" says which operator it is:
  loss    x [n, d], weight [v, d], target [n] -> the mean loss and the gradients of x and weight
          ("train"), or every token's loss ("eval")
  norm    r = x + scale * gate * f (f normalised first where "post"), y = norm(r) * weight (+ bias);
          with "train", the gradients of everything for given gradients of r and y too
  adamw   one step over many tensors; "bits" says how the two moments are held

Where `own` is false, run() computes them with elementary torch operations in float32.
"""
import math

import torch

own = False

_IGNORE = -100
_STEP = 10  # the optimizer step that a case is at
_LR, _B1, _B2, _EPS, _DECAY = 6e-4, 0.9, 0.95, 1e-8, 0.1
_BLOCK = 256  # values that share an exponent where moments are held in 8 bits


def _loss(name, n, d, v, mode, ignored):
    return {"name": name, "op": "loss", "n": n, "d": d, "v": v, "mode": mode, "ignored": ignored}


def _norm(name, n, d, kind, gate, post, train):
    """gate: "none", "channel" ([d]), "sequence" (8 sequences, or one a row where 8 does not divide
    n) or "element" ([n, d])."""
    return {"name": name, "op": "norm", "n": n, "d": d, "kind": kind, "gate": gate, "post": post, "train": train}


def _adamw(name, model, width, depth, vocab, bits):
    """model "gpt": the tensors of a GPT of this width, depth and vocabulary; "lenet": LeNet-5's;
    "mixed": `depth` tensors of 1 to `width` values."""
    return {"name": name, "op": "adamw", "model": model, "width": width, "depth": depth, "vocab": vocab, "bits": bits}


def listed():
    return [
        # A small model's head on a short batch: the calls of a first script, where launches count.
        _loss("loss_small", 96, 128, 1003, "train", False),
        # GPT-2 small's head on one 1024-token sequence.
        _loss("loss_gpt2_1024", 1024, 768, 50257, "train", False),
        # The same on a batch of eight sequences, some of the tokens padding: the largest.
        _loss("loss_gpt2_8192", 8192, 768, 50257, "train", True),
        # Scoring a document of an odd length with it: every token's loss, no gradients.
        _loss("loss_eval_2047", 2047, 768, 50257, "eval", True),
        # One token at generation: the smallest call.
        _norm("norm_token", 1, 768, "layer", "none", False, False),
        # GPT-2 small's residual addition and layer norm over 8192 tokens, forward and backward.
        _norm("norm_gpt2_8192", 8192, 768, "layer", "none", False, True),
        # A wide block with RMS norms on both sides and a gate for each channel.
        _norm("norm_sandwich_4096", 4096, 4096, "rms", "channel", True, True),
        # A block conditioned for each sequence, sizes that are multiples of nothing.
        _norm("norm_sequence_odd", 8 * 1031, 1001, "layer", "sequence", False, True),
        # LeNet-5's ten tensors, and a list of many small tensors of odd sizes: launches count.
        _adamw("adamw_lenet", "lenet", 0, 0, 0, 32),
        _adamw("adamw8_mixed", "mixed", 20000, 300, 0, 8),
        # GPT-2 small's 148 tensors with moments in 32 and in 8 bits.
        _adamw("adamw_gpt2", "gpt", 768, 12, 50257, 32),
        _adamw("adamw8_gpt2", "gpt", 768, 12, 50257, 8),
    ]


def _log(rng, lo, hi):
    """A whole number spread over [lo, hi] by its logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["loss", "loss", "norm", "norm", "adamw"])
    while True:
        if op == "loss":
            case = _loss(None, _log(rng, 1, 8192), rng.choice([_log(rng, 33, 1600), 64 * _log(rng, 1, 25)]),
                         _log(rng, 100, 130000), rng.choice(["train", "train", "eval"]), rng.random() < 0.5)
            if case["n"] * case["v"] > 4.2e8 or case["d"] * case["v"] > 1e8 or case["n"] * case["d"] * case["v"] > 3.1e11:
                continue
        elif op == "norm":
            case = _norm(None, _log(rng, 1, 16384), rng.choice([_log(rng, 3, 8192), 64 * _log(rng, 1, 128)]),
                         rng.choice(["layer", "rms"]), rng.choice(["none", "channel", "sequence", "element"]),
                         rng.random() < 0.4, rng.random() < 0.7)
            if case["n"] * case["d"] > 3e7:
                continue
        elif rng.random() < 0.5:
            case = _adamw(None, "gpt", 64 * rng.randint(2, 12), rng.randint(1, 12), _log(rng, 256, 50257), rng.choice([8, 32]))
        else:
            case = _adamw(None, "mixed", _log(rng, 100, 200000), _log(rng, 1, 400), 0, rng.choice([8, 32]))
        del case["name"]
        return case


def _sizes(case):
    """How many values each tensor of an adamw case has."""
    d, n = case["width"], case["depth"]
    if case["model"] == "lenet":
        return [150, 6, 2400, 16, 48000, 120, 10080, 84, 840, 10]
    if case["model"] == "gpt":
        block = [d, d, 3 * d * d, 3 * d, d * d, d, d, d, 4 * d * d, 4 * d, 4 * d * d, d]
        return [case["vocab"] * d, 1024 * d] + block * n + [d, d]
    # spread by the logarithm over 1..d, in an order of no pattern
    return [max(1, int(round(d ** (((i * 0.6180339887) % 1.0))))) for i in range(n)]


def _groups(case):
    """How many rows a norm case's gate has."""
    return {"none": 0, "channel": 1, "sequence": 8 if case["n"] % 8 == 0 else case["n"], "element": case["n"]}[case["gate"]]


def work(case):
    """Bytes (each input read once, each output written once) and operations of one pass."""
    if case["op"] == "loss":
        n, d, v = case["n"], case["d"], case["v"]
        if case["mode"] == "eval":
            return {"bytes": 4.0 * (n * d + v * d + n) + 8.0 * n, "flops": 2.0 * n * d * v}
        return {"bytes": 8.0 * (n * d + v * d) + 8.0 * n + 4.0, "flops": 6.0 * n * d * v}
    if case["op"] == "norm":
        n, d = case["n"], case["d"]
        per_column = d * (2 if case["kind"] == "layer" else 1) * (2 if case["post"] else 1) + _groups(case) * d
        b = 4.0 * (4 * n * d + per_column)
        if case["train"]:  # two gradients in, two out (x, f and r are read once for both directions)
            b += 4.0 * (4 * n * d + per_column)
        return {"bytes": b, "flops": (10.0 if not case["train"] else 40.0) * n * d}
    n = float(sum(_sizes(case)))
    if case["bits"] == 32:
        return {"bytes": 28.0 * n, "flops": 14.0 * n}
    return {"bytes": (12.0 + 4.0 + 8.0) * n, "flops": 60.0 * n}  # the moments' values come back too


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device="cuda") * std


def prepare(case, seed):
    g = _generator(seed)
    state = {"case": case}
    if case["op"] == "loss":
        n, d, v = case["n"], case["d"], case["v"]
        # A head at GPT-2's scale of weights. Words have their usual skewed frequencies, and the
        # hidden states lean towards their targets by different amounts, so the model is sure of
        # some tokens and has no idea of others.
        weight = _normal(g, v, d, std=0.02)
        target = (v * torch.rand(n, generator=g, device="cuda") ** 3).long().clamp_(max=v - 1)
        lean = 24.0 * torch.rand(n, 1, generator=g, device="cuda")
        w = weight[target]
        x = _normal(g, n, d) + lean * w / w.norm(dim=1, keepdim=True)
        if case["ignored"]:
            target = torch.where(torch.rand(n, generator=g, device="cuda") < 0.05, _IGNORE, target)
            target[0] = 1  # not every token is padding
        state.update(x=x, weight=weight, target=target)
    elif case["op"] == "norm":
        n, d, groups = case["n"], case["d"], _groups(case)
        layer = case["kind"] == "layer"
        # A residual stream that has grown past its blocks' outputs, with a few large channels.
        x = _normal(g, n, d, std=3.0)
        x[:, :: max(1, d // 5)] *= 10.0
        state["x"], state["f"] = x, _normal(g, n, d) + 0.1
        state["weight"] = 1.0 + _normal(g, d, std=0.2)
        state["bias"] = _normal(g, d, std=0.1) if layer else None
        state["post_weight"] = 1.0 + _normal(g, d, std=0.2) if case["post"] else None
        state["post_bias"] = _normal(g, d, std=0.1) if case["post"] and layer else None
        state["gate"] = None if groups == 0 else _normal(g, d) if case["gate"] == "channel" else _normal(g, groups, d)
        state["scale"] = 0.5 if case["gate"] != "none" else 1.0
        if case["train"]:
            state["dr"], state["dy"] = _normal(g, n, d, std=1e-3), _normal(g, n, d, std=1e-3)
            names = ("x", "f", "gate", "weight", "bias", "post_weight", "post_bias")
            state["inputs"] = [state[k].requires_grad_() for k in names if state[k] is not None]
    else:
        # The tensors as a trainer has them, cut from flat buffers (each at a whole block of 256).
        sizes = _sizes(case)
        starts, total = [], 0
        for s in sizes:
            starts.append(total)
            total += (s + _BLOCK - 1) // _BLOCK * _BLOCK
        held = torch.zeros(total, dtype=torch.bool, device="cuda")
        for a, s in zip(starts, sizes):
            held[a:a + s] = True
        p = _normal(g, total, std=0.02) * held
        # Gradients of very different sizes, from tensor to tensor and value to value.
        grad = _normal(g, total) * torch.exp(_normal(g, total, std=1.5) - 9.0) * held
        m = 0.3 * grad + _normal(g, total, std=1e-5) * held
        v = (grad * grad) * torch.rand(total, generator=g, device="cuda") + 1e-12 * held
        state.update(p=p, grad=grad)
        state["params"] = [p[a:a + s] for a, s in zip(starts, sizes)]
        state["grads"] = [grad[a:a + s] for a, s in zip(starts, sizes)]
        if case["bits"] == 32:
            state.update(m=m, v=v)
            state["exp_avgs"] = [m[a:a + s] for a, s in zip(starts, sizes)]
            state["exp_avg_sqs"] = [v[a:a + s] for a, s in zip(starts, sizes)]
        else:
            half = torch.full_like(p, 0.5)
            state["m"], state["m_exp"] = _to_codes(m, 14, half, True)
            state["v"], state["v_exp"] = _to_codes(v, 30, half, False)
            state["block"] = torch.arange(total // _BLOCK, device="cuda")
    return state


# ---- moments in 8 bits, in plain form ----
#
# A block of 256 values shares the exponent e of its largest magnitude, one more where that could
# round up to the next power of two. A magnitude a, with
# k = max(exponent of a, e - range), is a whole number q of 2^(k - 3), and its code is
# 8 (k - (e - range)) + q, at most 8 range + 15. a / 2^(k - 3) is rounded to a whole number up where
# its fraction exceeds a number u in [0, 1), else down.


def _exponent(a):
    """The exponent field of a float32's magnitude (0 for zero and subnormal numbers)."""
    return (a.view(torch.int32) >> 23) & 255


def _pow2(e):
    """2^(e - 127) for exponent fields e; 0 below the normal range."""
    return (e.clamp(min=0).to(torch.int32) << 23).view(torch.float32)


def _to_codes(x, span, u, signed):
    a = x.abs().view(-1, _BLOCK)
    top = a.amax(dim=1, keepdim=True).contiguous()
    e = ((top.view(torch.int32) + (1 << 20)) >> 23).clamp(min=span + 4, max=254)
    k = torch.maximum(_exponent(a), e - span)
    t = a * _pow2(257 - k)  # a / 2^(k - 127 - 3), exact
    low = torch.floor(t)
    q = low.to(torch.int32) + (t - low > u.view(-1, _BLOCK)).to(torch.int32)
    if not signed:  # a positive value never becomes zero
        q = torch.where(a > 0, q.clamp(min=1), q)
    code = (8 * (k - (e - span)) + q).clamp(max=8 * span + 15)
    if signed:
        code = torch.where(x.view(-1, _BLOCK) < 0, code + 128, code)
    return code.to(torch.uint8).view(-1), e.to(torch.uint8).view(-1)


def _from_codes(code, e, span, signed):
    c = code.to(torch.int32).view(-1, _BLOCK)
    negative = c >= 128 if signed else None
    c = c & 127 if signed else c
    e = e.to(torch.int32).view(-1, 1)
    up = ((c >> 3) - 1).clamp(min=0)
    q = torch.where(c < 8, c, 8 + (c & 7)).to(torch.float32)
    x = q * _pow2(e - span + up - 3)
    return (torch.where(negative, -x, x) if signed else x).view(-1)


def _mix(h):
    """32 well-mixed bits of a 32-bit number (held in 64)."""
    mask = 0xFFFFFFFF
    h = ((h ^ (h >> 16)) * 0x6A09E667) & mask
    h = ((h ^ (h >> 15)) * 0xBB67AE85) & mask
    return h ^ (h >> 16)


def _uniform(state):
    """The two rounding numbers of every value: the mixed position, step and moment, 16 bits each."""
    block = state["block"]
    at = block[:, None] * _BLOCK + torch.arange(_BLOCK, device=block.device)
    h = _mix((at ^ ((_STEP * 0x9E3779B9) & 0xFFFFFFFF)) & 0xFFFFFFFF).view(-1)
    return (h & 0xFFFF).to(torch.float32) * 2.0 ** -16, (h >> 16).to(torch.float32) * 2.0 ** -16


# ---- plain forms ----


def _plain_loss(state):
    x, weight, target = state["x"], state["weight"], state["target"]
    z = x @ weight.t()
    kept = target != _IGNORE
    safe = torch.where(kept, target, 0)[:, None]
    top = z.amax(dim=1, keepdim=True)
    zt = z.gather(1, safe)
    p = torch.exp(z - top)
    total = p.sum(dim=1, keepdim=True)
    rows = torch.where(kept, (torch.log(total) + (top - zt))[:, 0], 0.0)
    if state["case"]["mode"] == "eval":
        return {"loss": rows}
    count = kept.sum()
    dz = p / total
    dz.scatter_add_(1, safe, torch.full_like(zt, -1.0))
    dz = dz * (kept / count)[:, None]
    return {"loss": rows.sum() / count, "dx": dz @ weight, "dweight": dz.t() @ x}


def _plain_statistics(t, kind):
    """(t normalised, 1 / deviation)"""
    centred = t - t.mean(dim=1, keepdim=True) if kind == "layer" else t
    rstd = 1.0 / torch.sqrt((centred * centred).mean(dim=1, keepdim=True) + 1e-5)
    return centred * rstd, rstd


def _plain_norm_backward(d, hat, rstd, kind):
    inner = d - hat * (d * hat).mean(dim=1, keepdim=True)
    if kind == "layer":
        inner = inner - d.mean(dim=1, keepdim=True)
    return inner * rstd


def _plain_norm(state):
    case, kind = state["case"], state["case"]["kind"]
    with torch.no_grad():
        x, f, weight, bias, gate = (state[k] for k in ("x", "f", "weight", "bias", "gate"))
        n, d = x.shape
        if gate is not None and case["gate"] == "sequence":
            gate = gate.repeat_interleave(n // gate.shape[0], dim=0)
        scale = state["scale"]
        inner = f
        if case["post"]:
            f_hat, f_rstd = _plain_statistics(f, kind)
            inner = f_hat * state["post_weight"]
            inner = inner + state["post_bias"] if kind == "layer" else inner
        r = x + scale * (inner * gate if gate is not None else inner)
        r_hat, r_rstd = _plain_statistics(r, kind)
        y = r_hat * weight
        y = y + bias if kind == "layer" else y
        if not case["train"]:
            return {"r": r, "y": y}
        dy = state["dy"]
        dr = state["dr"] + _plain_norm_backward(dy * weight, r_hat, r_rstd, kind)
        grads = {"dx": dr, "dweight": (dy * r_hat).sum(dim=0)}
        if kind == "layer":
            grads["dbias"] = dy.sum(dim=0)
        d_inner = scale * dr
        if gate is not None:
            d_gate = d_inner * inner
            d_inner = d_inner * gate
            grads["dgate"] = {"channel": lambda: d_gate.sum(dim=0), "element": lambda: d_gate,
                              "sequence": lambda: d_gate.view(_groups(case), -1, d).sum(dim=1)}[case["gate"]]()
        if case["post"]:
            grads["dpost_weight"] = (d_inner * f_hat).sum(dim=0)
            if kind == "layer":
                grads["dpost_bias"] = d_inner.sum(dim=0)
            d_inner = _plain_norm_backward(d_inner * state["post_weight"], f_hat, f_rstd, kind)
        grads["df"] = d_inner
        return {"r": r, "y": y, **grads}


def _plain_adamw(state):
    p, grad = state["p"], state["grad"]
    small = state["case"]["bits"] == 8
    m, v = state["m"], state["v"]
    if small:
        m, v = _from_codes(m, state["m_exp"], 14, True), _from_codes(v, state["v_exp"], 30, False)
    m = m * _B1 + grad * (1.0 - _B1)
    v = v * _B2 + grad * grad * (1.0 - _B2)
    inverse = 1.0 / math.sqrt(1.0 - _B2 ** _STEP)
    step = _LR / (1.0 - _B1 ** _STEP)
    p.copy_(p * (1.0 - _LR * _DECAY) - m / (torch.sqrt(v) * inverse + _EPS) * step)
    if not small:
        state["m"].copy_(m)
        state["v"].copy_(v)
        return {"p": p, "m": state["m"], "v": state["v"]}
    um, uv = _uniform(state)
    state["m"], state["m_exp"] = _to_codes(m, 14, um, True)
    state["v"], state["v_exp"] = _to_codes(v, 30, uv, False)
    return {"p": p, "m": _from_codes(state["m"], state["m_exp"], 14, True),
            "v": _from_codes(state["v"], state["v_exp"], 30, False)}


# ---- the framework's operators ----


def _own_loss(state):
    import bit_reproducible_training_amd as rg

    x, weight, target = state["x"], state["weight"], state["target"]
    if state["case"]["mode"] == "eval":
        with torch.no_grad():
            return {"loss": rg.linear_cross_entropy(x, weight, target, reduction="none")}
    x, weight = x.detach().requires_grad_(), weight.detach().requires_grad_()
    loss = rg.linear_cross_entropy(x, weight, target)
    dx, dweight = torch.autograd.grad(loss, (x, weight))
    return {"loss": loss, "dx": dx, "dweight": dweight}


def _own_norm(state):
    import bit_reproducible_training_amd as rg

    case = state["case"]

    def forward():
        return rg.residual_norm(state["x"], state["f"], state["weight"], state["bias"], kind=case["kind"], eps=1e-5,
                                gate=state["gate"], scale=state["scale"], post_norm=case["post"],
                                post_weight=state["post_weight"], post_bias=state["post_bias"])

    if not case["train"]:
        with torch.no_grad():
            r, y = forward()
        return {"r": r, "y": y}
    r, y = forward()
    grads = iter(torch.autograd.grad((r, y), state["inputs"], (state["dr"], state["dy"])))
    names = ("x", "f", "gate", "weight", "bias", "post_weight", "post_bias")
    return {"r": r, "y": y, **{"d" + k: next(grads) for k in names if state[k] is not None}}


def _own_adamw(state):
    import bit_reproducible_training_amd as rg

    settings = dict(step=_STEP, lr=_LR, betas=(_B1, _B2), eps=_EPS, weight_decay=_DECAY)
    if state["case"]["bits"] == 32:
        rg.adamw_step(state["params"], state["grads"], state["exp_avgs"], state["exp_avg_sqs"], **settings)
        return {"p": state["p"], "m": state["m"], "v": state["v"]}
    rg.adamw8_step(state["params"], state["grads"], state["m"], state["m_exp"], state["v"], state["v_exp"], **settings)
    m, v = rg.adamw8_values(state["m"], state["m_exp"], state["v"], state["v_exp"])
    return {"p": state["p"], "m": m, "v": v}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"loss": _own_loss, "norm": _own_norm, "adamw": _own_adamw}[op](state)
    return {"loss": _plain_loss, "norm": _plain_norm, "adamw": _plain_adamw}[op](state)


# ---- the definitions in 64 bits ----


def _exact_loss(case, s):
    x, weight, target = s["x"].double().requires_grad_(), s["weight"].double().requires_grad_(), s["target"]
    if case["mode"] == "eval":
        with torch.no_grad():
            return {"loss": torch.nn.functional.cross_entropy(x @ weight.t(), target, ignore_index=_IGNORE, reduction="none")}
    loss = torch.nn.functional.cross_entropy(x @ weight.t(), target, ignore_index=_IGNORE)
    dx, dweight = torch.autograd.grad(loss, (x, weight))
    return {"loss": loss, "dx": dx, "dweight": dweight}


def _exact_norm(case, s):
    names = [k for k in ("x", "f", "gate", "weight", "bias", "post_weight", "post_bias") if s[k] is not None]
    t = {k: s[k].detach().double().requires_grad_() for k in names}

    def normalise(a):
        if case["kind"] == "layer":
            return torch.nn.functional.layer_norm(a, a.shape[-1:], eps=1e-5)
        return a * (a.pow(2).mean(-1, keepdim=True) + 1e-5).rsqrt()

    f = t["f"]
    if case["post"]:
        f = normalise(f) * t["post_weight"] + t.get("post_bias", 0.0)
    if "gate" in t:
        gate = t["gate"]
        if case["gate"] == "sequence":
            f = (f.view(gate.shape[0], -1, f.shape[1]) * gate[:, None]).view_as(f)
        else:
            f = f * gate
    r = t["x"] + s["scale"] * f
    y = normalise(r) * t["weight"] + t.get("bias", 0.0)
    if not case["train"]:
        return {"r": r, "y": y}
    grads = torch.autograd.grad((r, y), [t[k] for k in names], (s["dr"].double(), s["dy"].double()))
    return {"r": r, "y": y, **{"d" + k: d for k, d in zip(names, grads)}}


def _exact_adamw(case, s):
    p, g = s["p"].double(), s["grad"].double()
    if case["bits"] == 8:
        m = _from_codes(s["m"], s["m_exp"], 14, True).double()
        v = _from_codes(s["v"], s["v_exp"], 30, False).double()
    else:
        m, v = s["m"].double(), s["v"].double()
    m.lerp_(g, 1.0 - _B1)
    v.lerp_(g.square(), 1.0 - _B2)
    m_hat, v_hat = m / (1.0 - _B1 ** _STEP), v / (1.0 - _B2 ** _STEP)
    p = p - _LR * (_DECAY * p + m_hat / (v_hat.sqrt() + _EPS))
    if case["bits"] == 8:  # the moments' rounding goes by the random numbers: no value of its own
        return {"p": p, "m": None, "v": None}
    return {"p": p, "m": m, "v": v}


def exact(case, seed):
    state = prepare(case, seed)
    value = {"loss": _exact_loss, "norm": _exact_norm, "adamw": _exact_adamw}[case["op"]](case, state)
    return {k: v.detach() if v is not None else None for k, v in value.items()}
