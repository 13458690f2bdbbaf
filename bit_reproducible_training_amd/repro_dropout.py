"""Dropout whose mask is never stored: its random bits are a function of a seed and a value's place.

  dropout   zeroes values at random and scales the others, differentiable
  Dropout   a module over it

The bits come from a counter-based generator (include/repro_dropout_math.h), so the backward pass makes them again, and
the same seed gives the same mask on every run, on the GPU and on the CPU.
"""
import torch

from ._lib import _backend

__all__ = ["Dropout", "dropout"]


def _seed_of(seed):
    """(number, tensor or None)"""
    if isinstance(seed, torch.Tensor):
        return 0, seed
    return int(seed) & (2 ** 64 - 1), None


def fresh_seed():
    """A seed from torch's default CPU generator: torch.manual_seed fixes it, and checkpointing, which puts that generator
    back, gets it again."""
    return int(torch.randint(2 ** 63 - 1, (), dtype=torch.int64))


def dropout(x, p=0.5, *, seed):
    """x / (1 - p) where a value is kept and 0 where it is dropped, each with probability p (0 <= p < 1). x is float32 of any
    shape; values are told apart by their place in it, not in memory. seed is a number of 64 bits, or an int64
    tensor of one element on x's device, read when the kernel runs (so that each replay of a captured graph can have its own).
    One seed gives one mask to every tensor of a size: calls that are to differ need seeds that do."""
    return _backend.dropout_apply(x, float(p), *_seed_of(seed))


class Dropout(torch.nn.Module):
    """torch.nn.Dropout, reproducible: in training, forward(x) takes its seed from torch's CPU generator (torch.manual_seed), the
    same for x on a GPU and on the CPU, or the given one (a captured graph repeats a number, and reads a tensor at each replay); in
    evaluation it returns x."""

    def __init__(self, p=0.5):
        super().__init__()
        if not 0.0 <= p < 1.0:
            raise ValueError("the probability to drop must be in [0, 1)")
        self.p = float(p)

    def forward(self, x, seed=None):
        if not self.training or self.p == 0.0:
            return x
        return dropout(x, self.p, seed=fresh_seed() if seed is None else seed)

    def extra_repr(self):
        return "p=%g" % self.p
