"""AdamW over many tensors at once, with the moments in float32 or in 8 bits.

  adamw_step     one step over lists of float32 tensors, moments in float32
  adamw8_step    the same with the moments in 8 bits (one byte a value and one exponent for every
                 256 values, each moment): 16 instead of 28 bytes a value are moved
  AdamW          a torch.optim.Optimizer over them

Every operation is rounded once in a fixed order (include/repro_adamw_math.h), and the 8-bit moments
are rounded by numbers that mix a value's position with the step, so a step gives the same bits on
every run, on the GPU and on the CPU. On a GPU a step is a few launches on the current stream, whatever
the number of tensors, and does not synchronise; its constants are launch arguments, so a captured
graph repeats the captured step. Tensors are updated in place.
"""
import torch

from ._lib import _backend

__all__ = ["AdamW", "adamw8_state", "adamw8_step", "adamw8_values", "adamw_step"]

BLOCK = 256  # values that share an exponent


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, *, step, lr=1e-3, betas=(0.9, 0.999), eps=1e-8,
               weight_decay=1e-2):
    """One AdamW step, in place: for each value
        m <- m b1 + g (1 - b1),  v <- v b2 + g^2 (1 - b2),
        p <- p (1 - lr weight_decay) - m / (sqrt(v) / sqrt(1 - b2^step) + eps) lr / (1 - b1^step).
    params, grads, exp_avgs and exp_avg_sqs are lists of float32 tensors on one GPU or on the CPU; a
    parameter's four tensors are dense and laid out alike, and none that is updated overlaps another of the call (neighbours
    in a list and a parameter's own are checked). step is 1 for the first."""
    _backend.adamw_step(params, grads, exp_avgs, exp_avg_sqs, float(lr), float(betas[0]), float(betas[1]), float(eps),
                        float(weight_decay), int(step))


def adamw8_step(params, grads, exp_avgs, exp_avg_exponents, exp_avg_sqs, exp_avg_sq_exponents, *, step, lr=1e-3,
                betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2):
    """adamw_step with the moments in 8 bits: uint8 codes, 256 for each started block of 256 values
    of a parameter, and one uint8 exponent for each block. Each of the four is a list with a tensor
    for each parameter, or one tensor that holds all parameters' blocks in their order
    (adamw8_state makes such). All zero is the state before the first step."""
    flat = isinstance(exp_avgs, torch.Tensor)
    states = (exp_avgs, exp_avg_exponents, exp_avg_sqs, exp_avg_sq_exponents)
    if any(isinstance(s, torch.Tensor) != flat for s in states):
        raise ValueError("adamw: the moments are four tensors or four lists")
    if flat:
        states = [[s] for s in states]
    _backend.adamw8_step(params, grads, *states, flat, float(lr), float(betas[0]), float(betas[1]), float(eps),
                         float(weight_decay), int(step))


def adamw8_state(params):
    """(exp_avgs, exp_avg_exponents, exp_avg_sqs, exp_avg_sq_exponents) before the first step, one
    tensor each for all of params (an iterable of tensors on one device)."""
    params = list(params)
    blocks = sum(-(-p.numel() // BLOCK) for p in params)
    device = params[0].device if params else None
    return tuple(torch.zeros(n, dtype=torch.uint8, device=device) for n in (blocks * BLOCK, blocks) * 2)


def adamw8_values(exp_avg, exp_avg_exponent, exp_avg_sq, exp_avg_sq_exponent):
    """(m, v): the float32 values that 8-bit moments stand for, 256 for each block."""
    m, v = _backend.adamw8_values(exp_avg, exp_avg_exponent, exp_avg_sq, exp_avg_sq_exponent)
    return m, v


class AdamW(torch.optim.Optimizer):
    """torch.optim.AdamW's lr, betas, eps and weight_decay and its update (amsgrad, maximize, capturable and the
    choice of an implementation are not there), reproducible bit for bit; state_bits=8 keeps the
    moments in 8 bits. Parameters are float32, each group's on one device. A parameter without a
    gradient is left out of a step; each counts its own steps."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32):
        if not lr >= 0.0 or not eps >= 0.0 or not weight_decay >= 0.0:
            raise ValueError("lr, eps and weight_decay must not be negative")
        if not all(0.0 <= b < 1.0 for b in betas):
            raise ValueError("betas must be in [0, 1)")
        if state_bits not in (8, 32):
            raise ValueError("state_bits must be 8 or 32")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits))

    def _state_of(self, p, bits):
        state = self.state[p]
        if not state:
            state["step"] = 0
            if bits == 8:
                blocks = -(-p.numel() // BLOCK)
                for name in ("exp_avg", "exp_avg_sq"):
                    state[name] = torch.zeros(blocks * BLOCK, dtype=torch.uint8, device=p.device)
                    state[name + "_exponent"] = torch.zeros(blocks, dtype=torch.uint8, device=p.device)
            else:
                state["exp_avg"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                state["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.preserve_format)
        return state

    def __setstate__(self, state):
        super().__setstate__(state)
        for group in self.param_groups:
            group.setdefault("state_bits", 32)

    def load_state_dict(self, state_dict):
        """As torch's, except that 8-bit moments stay what they are (torch converts a state to its
        parameter's type). A state of torch.optim.AdamW is taken up, with moments in float32."""
        for group in state_dict["param_groups"]:
            if group.get("amsgrad") or group.get("maximize"):
                raise ValueError("AdamW has no amsgrad and no maximize")
        saved = {k: {n: t for n, t in s.items() if isinstance(t, torch.Tensor) and t.dtype == torch.uint8}
                 for k, s in state_dict["state"].items()}
        super().load_state_dict(state_dict)
        for state in self.state.values():
            if "step" in state:
                state["step"] = int(state["step"])  # torch's is a tensor
        numbers = [n for g in state_dict["param_groups"] for n in g["params"]]
        params = [p for g in self.param_groups for p in g["params"]]
        for number, p in zip(numbers, params):
            for name, t in saved.get(number, {}).items():
                self.state[p][name] = t.detach().clone().to(p.device)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            bits = group["state_bits"]
            by_step = {}
            try:
                for p in group["params"]:
                    if p.grad is None:
                        continue
                    if p.grad.is_sparse:
                        raise RuntimeError("AdamW takes dense gradients")
                    state = self._state_of(p, bits)
                    state["step"] += 1
                    by_step.setdefault((int(state["step"]), p.device), []).append((p, state))
                while by_step:
                    key = next(iter(by_step))
                    self._take(group, bits, key[0], by_step[key])
                    del by_step[key]
            except BaseException:  # steps that were not taken do not count
                for held in by_step.values():
                    for _, state in held:
                        state["step"] -= 1
                raise
        return loss

    def _take(self, group, bits, step, held):
        params = [p for p, _ in held]
        grads = [_laid_out_as(p.grad, p) for p in params]
        settings = dict(step=step, lr=group["lr"], betas=group["betas"], eps=group["eps"], weight_decay=group["weight_decay"])
        if bits == 8:
            names = ("exp_avg", "exp_avg_exponent", "exp_avg_sq", "exp_avg_sq_exponent")
            adamw8_step(params, grads, *([s[n] for _, s in held] for n in names), **settings)
        else:
            adamw_step(params, grads, [s["exp_avg"] for _, s in held], [s["exp_avg_sq"] for _, s in held], **settings)


def _laid_out_as(grad, p):
    """The gradient with its parameter's strides (itself where it has them)."""
    if grad.is_neg():
        grad = grad.resolve_neg()
    if p.is_contiguous():
        return grad.contiguous()
    return grad if grad.stride() == p.stride() else torch.empty_like(p).copy_(grad)
