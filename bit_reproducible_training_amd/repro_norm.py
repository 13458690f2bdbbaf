"""The residual addition of a transformer block with the norms before and after it, and its gradients.

  norm            y = Norm(x) * weight + bias
  residual_norm   r = x + scale * gate * u, y = Norm(r) * weight + bias, where u is f, or with post_norm
                  Norm(f) * post_weight + post_bias: what lies between one block's output f and the
                  next block's input y, in one pass over the rows
  Norm, ResidualNorm   modules over them that report to the layers' guard

Norm is a layer norm ("layer") or an RMS norm ("rms"). float32 tensors on a GPU (on the current
stream) or on the CPU, the same bits either way: every operation is rounded once and every sum has an
order that the sizes fix (include/repro_norm_math.h).
"""
import torch

from ._lib import _backend
from .layers import guard

__all__ = ["Norm", "ResidualNorm", "norm", "residual_norm"]

_KINDS = {"layer": False, "rms": True}


class _NormOp(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, f, gate, post_weight, post_bias, weight, bias, settings, watch, wanted):
        operands = (x, f, gate, post_weight, post_bias, weight, bias)
        flag, number = watch.cell(x) if watch else (None, 0)
        r, y, stats = _backend.residual_norm(*operands, *settings, wanted, flag, number)
        if wanted:
            ctx.save_for_backward(x if f is None else r, f, gate, post_weight, post_bias, weight, stats)
            ctx.settings, ctx.watch = settings, watch
        ctx.set_materialize_grads(False)
        return (y,) if f is None else (r, y)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *grads):
        dr, dy = (None, grads[0]) if len(grads) == 1 else grads
        if dr is None and dy is None:
            return (None,) * 10
        r, f, gate, post_weight, post_bias, weight, stats = ctx.saved_tensors
        flag, number = ctx.watch.gradient_cell(r) if ctx.watch else (None, 0)
        out = _backend.residual_norm_grad(dr, dy, r.contiguous(), f, gate, post_weight, post_bias, weight, stats,
                                          *ctx.settings, list(ctx.needs_input_grad[:7]), flag, number)
        if out[2] is not None:
            out[2] = out[2].view(gate.shape)
        return (*out, None, None, None)


class _Watch:
    """Where a module reports a NaN or infinity: the guard's cells, on a GPU in the norm's own launch."""

    def __init__(self, name):
        self.name, self.guard = name, guard()

    def cell(self, x):
        return self._cell(x, self.name + " input")

    def gradient_cell(self, x):
        return self._cell(x, self.name + " gradient")

    def _cell(self, x, label):
        if not x.is_cuda:
            return None, 0
        return self.guard._cell(x.device), self.guard._number(label)


def _rows(t, d):
    return None if t is None else t.reshape(-1, d)


def _apply(x, f, weight, bias, kind, eps, gate, scale, post_norm, post_weight, post_bias, watch):
    if kind not in _KINDS:
        raise ValueError('kind must be "layer" or "rms"')
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("norm: x must be [..., values]")
    if f is not None and f.shape != x.shape:
        raise ValueError("norm: f must have x's shape")
    d = x.shape[-1]
    for name, t in (("weight", weight), ("bias", bias), ("post_weight", post_weight), ("post_bias", post_bias)):
        if t is not None and tuple(t.shape) != (d,):
            raise ValueError("norm: %s must be [%d]" % (name, d))
    if gate is not None and (gate.dim() < 1 or gate.shape[-1] != d):
        raise ValueError("norm: the gate's last dimension must be x's")
    if watch is not None and not x.is_cuda:
        watch.guard.scan(x, watch.name + " input")
        if f is not None:
            watch.guard.scan(f, watch.name + " input")
    settings = (_KINDS[kind], bool(post_norm), float(eps), float(scale))
    operands = (_rows(x, d), _rows(f, d), gate, post_weight, post_bias, weight, bias)
    wanted = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in operands)
    out = _NormOp.apply(*operands, settings, watch, wanted)
    return tuple(t.view(x.shape) for t in out)


def norm(x, weight=None, bias=None, *, kind="layer", eps=1e-5):
    """Norm(x) * weight + bias over the last dimension (1 to 16384 values) of a float32 tensor."""
    return _apply(x, None, weight, bias, kind, eps, None, 1.0, False, None, None, None)[0]


def residual_norm(x, f, weight=None, bias=None, *, kind="layer", eps=1e-5, gate=None, scale=1.0, post_norm=False,
                  post_weight=None, post_bias=None):
    """(r, y): r = x + scale * gate * u and y = Norm(r) * weight + bias, where u is f, or with
    post_norm Norm(f) * post_weight + post_bias. x and f are float32 [..., D] of one shape; weights
    and biases [D], or None. gate is None or [..., D] with G leading elements, G a divisor of x's
    rows (its leading elements): each run of rows / G rows takes one of its rows. So [D] gates channels,
    [batch, D] gates each sequence of an x of [batch, tokens, D], and x's shape each value. Gradients
    reach every tensor; r and y may be used or not."""
    return _apply(x, f, weight, bias, kind, eps, gate, scale, post_norm, post_weight, post_bias, None)


class Norm(torch.nn.Module):
    """Reproducible torch.nn.LayerNorm(size) or torch.nn.RMSNorm(size)."""

    repro_name = "norm"

    def __init__(self, size, kind="layer", eps=1e-5, bias=None):
        super().__init__()
        if kind not in _KINDS:
            raise ValueError('kind must be "layer" or "rms"')
        self.kind, self.eps = kind, eps
        self.weight = torch.nn.Parameter(torch.ones(size))
        biased = kind == "layer" if bias is None else bias
        self.bias = torch.nn.Parameter(torch.zeros(size)) if biased else None

    def forward(self, x):
        return _apply(x, None, self.weight, self.bias, self.kind, self.eps, None, 1.0, False, None, None,
                      _Watch(self.repro_name))[0]


class ResidualNorm(Norm):
    """residual_norm with the weights of its norms: forward(x, f, gate=None) returns (r, y). With
    post_norm the block's output f is normalised too."""

    repro_name = "residual_norm"

    def __init__(self, size, kind="layer", eps=1e-5, bias=None, scale=1.0, post_norm=False):
        super().__init__(size, kind, eps, bias)
        self.scale, self.post_norm = scale, post_norm
        self.post_weight = torch.nn.Parameter(torch.ones(size)) if post_norm else None
        self.post_bias = torch.nn.Parameter(torch.zeros(size)) if post_norm and self.bias is not None else None

    def forward(self, x, f, gate=None):
        return _apply(x, f, self.weight, self.bias, self.kind, self.eps, gate, self.scale, self.post_norm,
                      self.post_weight, self.post_bias, _Watch(self.repro_name))
