"""The softmax cross entropy of a language model's head: x W^T, the loss and its gradients, without
keeping the logits.

  linear_cross_entropy   the loss of hidden states against target words, differentiable
  LinearCrossEntropy     a module with the head's weight, which reports to the layers' guard

The three products (logits, the gradients of x and of the weight) are the reproducible GEMM's; the
softmax's exponentials, logarithms and sums have their own definition (include/repro_loss_math.h). So loss
and gradients have the same bits on every run, on the GPU and on the CPU. Tokens are taken in groups (of
up to 2048, whose logits fill at most 512 MB, or of 128), and a group's logits are used for its gradients at once,
so training takes three products. With the sum or the mean of the losses, the forward pass leaves the
gradients for the backward pass to hand out. Without a reduction, whose gradients need what arrives there, the
backward pass computes the logits again.

Memory on a GPU while a call runs: for one group 4 bytes a logit, and with both gradients 2 slices bytes more
(the digits of the logits' gradient in both orientations: at 3 slices 2.5 times the logits in all); 2 slices bytes
for each value of the weight and about as much for each of x; the products' partial sums.
"""
import torch

from ._lib import _backend
from .layers import _CallInfo, _watch_operands, get_slices, guard

__all__ = ["LinearCrossEntropy", "linear_cross_entropy"]

_REDUCTIONS = {"mean": 0, "sum": 1, "none": 2}


def linear_cross_entropy(x, weight, target, *, ignore_index=-100, reduction="mean", slices=None):
    """The cross entropy of softmax(x weight^T) against target, for float32 x [..., size], weight
    [words, size] and int64 target [...]; reduction "mean" (over the tokens that count), "sum", or
    "none" (a loss for each token). Tokens whose target is ignore_index are left out; one whose target
    is no word has a NaN loss and no gradients. A token whose row of x holds a NaN or an infinity, or whose largest
    logit is infinite, has a NaN loss, a NaN row in x's gradient and makes its target's row of the weight's NaN; where the
    weight holds one, every token that counts is such. slices: the products' S (the layers' by default)."""
    return _apply(x, weight, target, ignore_index, reduction, get_slices() if slices is None else int(slices), None, 0)


def _apply(x, weight, target, ignore_index, reduction, slices, cell, gradient_label):
    if reduction not in _REDUCTIONS:
        raise ValueError('reduction must be "mean", "sum" or "none"')
    return _backend.loss_apply(x, weight, target, slices, _REDUCTIONS[reduction], int(ignore_index), cell, gradient_label)


class LinearCrossEntropy(torch.nn.Module):
    """A head of num_words words over hidden states of in_features values with its loss:
    forward(x, target) is linear_cross_entropy of them. The weight [num_words, in_features] may be
    shared with an embedding."""

    repro_name = "linear_cross_entropy"

    def __init__(self, in_features, num_words, ignore_index=-100, reduction="mean"):
        super().__init__()
        if reduction not in _REDUCTIONS:
            raise ValueError('reduction must be "mean", "sum" or "none"')
        self.ignore_index, self.reduction = ignore_index, reduction
        self.weight = torch.nn.Parameter(torch.empty(num_words, in_features))
        torch.nn.init.normal_(self.weight, std=0.02)

    def forward(self, x, target):
        info = _CallInfo(self.repro_name, get_slices(), guard())
        _watch_operands(info, x, self.weight)
        return _apply(x, self.weight, target, self.ignore_index, self.reduction, info.slices, info.guard._cell(x.device),
                      info.guard._number(info.name + " gradient"))
