"""Attention to the states of the same or another sequence, the learned bias of relative positions, and a layer of
several heads.

  attention                softmax(scale q k^T + bias) v with masks and dropout, differentiable, nothing of size
                           queries x keys ever stored
  relative_position_bias   a table's row for each bucket of distances, by distance or dense, differentiable
  RelativePositionBias     a module with the table
  Attention                projections, attention and the output projection (self or cross attention)

float32 tensors on a GPU (on the current stream) or on the CPU, the same bits either way: every operation is rounded once and
every sum's order is fixed (include/repro_attention_math.h). A query's result depends on the query and the keys it sees
alone: the same bits in a batch, in a padded batch, or one token at a time. (With dropout also on its places in the call, by
which pairs are dropped: the item's and head's number, the query's and the keys'.)
"""
import functools

import torch

from ._lib import _backend
from .layers import Linear
from .repro_dropout import _seed_of, fresh_seed

__all__ = ["Attention", "RelativePositionBias", "attention", "relative_position_bias"]


def attention(q, k, v, *, scale=None, causal=False, query_start=0, key_lengths=None, mask=None, relative_bias=None, dropout=0.0,
              seed=0):
    """softmax over the keys of (scale q_i . k_j + bias) times v, for q [batch, queries, heads, size] and k, v [batch, keys,
    key heads, size] (key heads divide heads: neighbouring query heads share one; size 1 to 128; any strides), as
    [batch, queries, heads, size].

    scale: 1 / sqrt(size) by default. Query i sees key j where j < key_lengths[batch] (int64 or int32), with causal j <= i +
    query_start (query_start: the keys' position at which the first query stands), and where mask (bool, broadcast to [batch,
    heads, queries, keys]) is true. A query that sees none has 0 and no gradients; what keys hold that it does not see, NaN or not,
    does not reach it. relative_bias [heads, queries + keys - 1] is added at column j - i + queries - 1
    (relative_position_bias(..., dense=False) makes one). dropout: the probability that a pair's share of v is dropped, by seed
    (as of rg.dropout). Gradients reach q, k, v and relative_bias; those of q, k and v are made together, whichever are wanted."""
    size = q.shape[-1] if q.dim() else 0
    if scale is None:
        scale = size ** -0.5 if size else 1.0
    number, at = _seed_of(seed)
    return _backend.attention_apply(q, k, v, float(scale), bool(causal), int(query_start), key_lengths, mask, relative_bias,
                                    float(dropout), number, at)


@functools.lru_cache(maxsize=64)
def _borders(buckets, max_distance):
    """The distances at which the next of a side's buckets begin: one bucket a distance for the first half, the others evenly in
    the logarithm up to max_distance, found in whole numbers: the least n of (n / exact)^steps >= (max_distance / exact)^t."""
    exact = buckets // 2
    steps = buckets - exact
    found = list(range(1, exact + 1))
    for t in range(1, steps):
        low, high = exact, max_distance
        target = max_distance ** t * exact ** (steps - t)
        while low < high:
            n = (low + high) // 2
            if n ** steps >= target:
                high = n
            else:
                low = n + 1
        found.append(low)
    return found


def _side(buckets, max_distance, bidirectional):
    """The buckets of a side of a table."""
    side = buckets // 2 if bidirectional else buckets
    if side < 2 or side > 513 or (bidirectional and buckets % 2):
        raise ValueError("relative_position_bias: 2 to 513 buckets a side, evenly divided")
    if not side // 2 < max_distance < 2 ** 31:
        raise ValueError("relative_position_bias: max_distance must be more than half a side's buckets and less than 2^31")
    return side


def relative_position_bias(table, q_len, k_len, *, max_distance=128, bidirectional=True, query_start=0, dense=True):
    """A learned bias for each pair of a query and a key by the bucket of their distance: table [buckets, heads] -> [heads, q_len, k_len],
    or with dense=False [heads, q_len + k_len - 1] by distance (key minus query, ascending), as attention takes it.

    Key j is j - i - query_start away from query i. bidirectional: half the buckets for the keys up to the query, half for those
    after it; else keys after it share bucket 0. Of a side's buckets the first half are a distance each, the others
    even steps of the logarithm up to max_distance, and the last takes all beyond. Gradients reach the table."""
    if table.dim() != 2:
        raise ValueError("relative_position_bias: the table must be [buckets, heads]")
    side = _side(table.shape[0], max_distance, bidirectional)
    return _backend.relative_bias_apply(table, int(q_len), int(k_len), int(query_start), _borders(side, int(max_distance)),
                                        bool(bidirectional), bool(dense))


class RelativePositionBias(torch.nn.Module):
    """A learned table for relative_position_bias: forward(q_len, k_len, query_start=0) gives the bias by distance, which
    attention and Attention take (one may serve every layer); dense() every pair's."""

    def __init__(self, num_heads, num_buckets=32, max_distance=128, bidirectional=True):
        super().__init__()
        _side(num_buckets, max_distance, bidirectional)
        self.max_distance, self.bidirectional = max_distance, bidirectional
        self.weight = torch.nn.Parameter(torch.empty(num_buckets, num_heads))
        torch.nn.init.normal_(self.weight, std=0.02)

    def forward(self, q_len, k_len, query_start=0):
        return self._of(q_len, k_len, query_start, False)

    def dense(self, q_len, k_len, query_start=0):
        return self._of(q_len, k_len, query_start, True)

    def _of(self, q_len, k_len, query_start, dense):
        return relative_position_bias(self.weight, q_len, k_len, max_distance=self.max_distance, bidirectional=self.bidirectional,
                                      query_start=query_start, dense=dense)


class Attention(torch.nn.Module):
    """A layer of attention with num_heads heads over num_kv_heads (as many by default) heads of keys and values, each of
    head_size (width / num_heads by default): forward(x, states=None, ...) lets the positions of x [batch, queries, width] look at
    those of states [batch, keys, states_width], or of x itself. The products are the reproducible Linear's. In training, dropout
    drops shares of v by seeds from torch's CPU generator, as Dropout's; a captured graph repeats the seed that it was captured with, unless
    seed is a tensor."""

    def __init__(self, width, num_heads, num_kv_heads=None, head_size=None, states_width=None, bias=False, dropout=0.0):
        super().__init__()
        num_kv_heads = num_heads if num_kv_heads is None else num_kv_heads
        if num_heads < 1 or num_kv_heads < 1 or num_heads % num_kv_heads:
            raise ValueError("num_kv_heads must divide num_heads")
        if head_size is None and width % num_heads:
            raise ValueError("num_heads must divide width where head_size is not given")
        if not 0.0 <= dropout < 1.0:
            raise ValueError("the probability to drop must be in [0, 1)")
        self.num_heads, self.num_kv_heads = num_heads, num_kv_heads
        self.head_size = width // num_heads if head_size is None else head_size
        if not 1 <= self.head_size <= 128:
            raise ValueError("a head's size must be 1 to 128")
        self.dropout = float(dropout)
        self.query = Linear(width, num_heads * self.head_size, bias=bias)
        self.key_value = Linear(width if states_width is None else states_width, 2 * num_kv_heads * self.head_size, bias=bias)
        self.out = Linear(num_heads * self.head_size, width, bias=bias)

    def forward(self, x, states=None, *, causal=False, query_start=0, key_lengths=None, mask=None, relative_bias=None, seed=None):
        if _backend.capturing(x):
            operands = [t for t in (x, states, relative_bias) if t is not None]
            _backend.need_capturable(operands + list(self.parameters()), "Attention")
        states = x if states is None else states
        q = self.query(x).unflatten(-1, (self.num_heads, self.head_size))
        k, v = self.key_value(states).unflatten(-1, (2, self.num_kv_heads, self.head_size)).unbind(-3)
        p = self.dropout if self.training else 0.0
        if seed is None:
            seed = fresh_seed() if p else 0
        y = attention(q, k, v, causal=causal, query_start=query_start, key_lengths=key_lengths, mask=mask,
                      relative_bias=relative_bias, dropout=p, seed=seed)
        return self.out(y.flatten(-2))
