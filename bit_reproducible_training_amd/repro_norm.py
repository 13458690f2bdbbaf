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


def _apply(x, f, weight, bias, kind, eps, gate, scale, post_norm, post_weight, post_bias, name=None):
    if kind not in _KINDS:
        raise ValueError('kind must be "layer" or "rms"')
    cell, input_label, gradient_label = None, 0, 0
    if name is not None and (x.is_cuda or x.is_cpu):
        # a module's: the guard hears of rows whose norm is not finite and of gradients, in the norm's own passes
        watcher = guard()
        cell = watcher._cell(x.device)
        input_label, gradient_label = watcher._number(name + " input"), watcher._number(name + " gradient")
    return _backend.norm_apply(x, f, gate, post_weight, post_bias, weight, bias, _KINDS[kind], bool(post_norm),
                               float(eps), float(scale), cell, input_label, gradient_label)


def norm(x, weight=None, bias=None, *, kind="layer", eps=1e-5):
    """Norm(x) * weight + bias over the last dimension (1 to 16384 values) of a float32 tensor."""
    return _apply(x, None, weight, bias, kind, eps, None, 1.0, False, None, None)[0]


def residual_norm(x, f, weight=None, bias=None, *, kind="layer", eps=1e-5, gate=None, scale=1.0, post_norm=False,
                  post_weight=None, post_bias=None):
    """(r, y): r = x + scale * gate * u and y = Norm(r) * weight + bias, where u is f, or with
    post_norm Norm(f) * post_weight + post_bias. x and f are float32 [..., D] of one shape; weights
    and biases [D], or None. gate is None or [..., D] whose leading sizes are the first of x's leading sizes (1s at
    their end do not count): [D] gates channels, [batch, D] or [batch, 1, D] each sequence of an x of
    [batch, tokens, D], and x's shape each value. For an x of [rows, D] it may be [G, D], G a divisor of
    rows, and each run of rows / G rows takes one of its rows. Other gates are refused. Gradients
    reach every tensor; r and y may be used or not."""
    r, y = _apply(x, f, weight, bias, kind, eps, gate, scale, post_norm, post_weight, post_bias)
    return r, y


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
                      self.repro_name)[0]


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
        r, y = _apply(x, f, self.weight, self.bias, self.kind, self.eps, gate, self.scale, self.post_norm,
                      self.post_weight, self.post_bias, self.repro_name)
        return r, y
