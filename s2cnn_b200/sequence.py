"""Operators for sequences of spherical signals: what stands between the feature vectors that a spherical
network gives for signals in order (the frames of a recording, the shells of a volume, the rings of a
sphere) and an answer about all of them.

* ``attention`` with a learned bias by buckets of the relative position (``relative_buckets``), its output
  and its gradients computed without storing a score;
* ``layer_norm`` over the last axis;
* ``dropout`` with a counter-based mask that is never stored, optionally added to a residual;

and the modules built on them, ``RelativeBias``, ``LayerNorm``, ``Dropout`` and ``SequenceBlock``.  The
reference has no counterpart.  Tensors are float32 or bfloat16 (one type per call).  Sums, the statistics of
softmax and norm and what is computed element by element are float32; bfloat16 attention takes its weights (of more
than 16 query rows per key head), and in the backward pass weights and score gradients, into the products rounded
to bfloat16 (results are off by 2.4e-3 in the 2-norm, of which their own rounding is 1.7e-3).  Results and
gradients are the same to the last bit in every call on the same inputs, recorded for gradients or not (but for
the output of bfloat16 attention where the gradient of a bias is wanted: its weights are kept more exactly then).
"""
import math

import torch
from torch import nn
from torch.nn.parameter import Parameter

from .ops import cuda_ops


def relative_buckets(num_buckets, reach, device=None):
    """The bucket of each relative position ``-reach ... reach`` (key minus query), int32 [2 reach + 1].

    Half of the buckets are for keys at or before the query, half for those behind it.  Of a half, the first
    half are single steps; the others grow as powers, the last one holding everything from about ``reach`` on.
    """
    assert num_buckets >= 4 and num_buckets % 2 == 0 and reach >= num_buckets // 4
    side = num_buckets // 2
    exact = max(1, side // 2)
    edges = [exact * (reach / exact) ** (k / (side - exact)) for k in range(1, side - exact)]
    steps = [d if d < exact else exact + sum(d >= e for e in edges) for d in range(reach + 1)]
    return torch.tensor([steps[-d] if d <= 0 else side + steps[d] for d in range(-reach, reach + 1)],
                        dtype=torch.int32, device=device)


def attention(q, k, v, bias=None, buckets=None, causal=False, scale=None, q_start=0, q_lengths=None, kv_lengths=None):
    """Softmax attention.

    :param q: [batch, queries, heads, dim], dim <= 128; any strides with a contiguous last axis (slices of
        one projection of all three are read where they lie)
    :param k, v: [batch, keys, kv_heads, dim]; heads is a multiple of kv_heads, and heads / kv_heads
        neighbouring query heads share a key head
    :param bias: [num_buckets, heads], added to the scaled scores by the bucket of the relative position
    :param buckets: int32 [2 reach + 1], the bucket of each relative position -reach ... reach (farther ones
        count as +-reach; an entry outside the buckets adds nothing), see ``relative_buckets``; reach <= 2048
    :param causal: a query sees the keys up to its own position only
    :param scale: of q . k, 1 / sqrt(dim) by default
    :param q_start: position of the first query among the keys, a number or int32 [batch]
    :param q_lengths, kv_lengths: int32 [batch], the queries and keys that are filled; what is beyond them
        is not looked at.  A query that sees no key gives 0 and no gradient
    :return: [batch, queries, heads, dim]

    An infinity or NaN that a query sees makes its column (in v) or the query's whole row (in q, k) infinite or NaN;
    which of the two depends on the size of the call.
    """
    starts = None
    if isinstance(q_start, torch.Tensor):
        q_start, starts = 0, q_start
    if scale is None:
        scale = 1.0 / math.sqrt(q.size(-1))
    return cuda_ops().ag_attention(q, k, v, bias, buckets, starts, q_lengths, kv_lengths, bool(causal), float(scale), int(q_start))


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last axis (at most 16384 values)."""
    return cuda_ops().ag_layer_norm(x, weight, bias, float(eps))


def dropout(x, p, seed, step=0, residual=None):
    """``residual + x * mask / (1 - p)``, an element kept with probability 1 - p.

    The mask is a function of (seed, step, index of the element): the same for the same numbers, never
    stored, computed again for the gradient.  Give every place in a model a ``seed`` and every call a ``step``
    of its own (both below 2^63).  Numbers are part of a captured or recorded call; ``seed`` may instead be an
    int64 tensor of the two on the device of x, which the kernel reads when it runs.
    """
    if isinstance(seed, torch.Tensor):
        assert step == 0, "dropout: the tensor holds the step, too"
        return cuda_ops().ag_dropout(x, residual, float(p), 0, 0, seed)
    assert 0 <= seed < 1 << 63 and 0 <= step < 1 << 63
    return cuda_ops().ag_dropout(x, residual, float(p), int(seed), int(step), None)


class RelativeBias(nn.Module):
    """A learned bias per head and bucket of the relative position: ``weight`` [num_buckets, heads] and the
    ``buckets`` that ``attention`` looks it up by."""

    def __init__(self, heads, num_buckets=32, reach=128):
        super().__init__()
        self.weight = Parameter(torch.zeros(num_buckets, heads))
        self.register_buffer("buckets", relative_buckets(num_buckets, reach), persistent=False)


class LayerNorm(nn.Module):
    """``layer_norm`` with a learned weight and bias (parameter names as in torch), in the type of these."""

    def __init__(self, features, eps=1e-5):
        super().__init__()
        self.eps = eps
        self.weight = Parameter(torch.ones(features))
        self.bias = Parameter(torch.zeros(features))

    def forward(self, x):
        if x.dtype in (torch.float32, torch.bfloat16):          # (others are refused)
            x = x.to(self.weight.dtype)
        return layer_norm(x, self.weight, self.bias, self.eps)


class Dropout(nn.Module):
    """``dropout`` with a seed and a step that every call in training mode draws from torch's generator of the device of
    x; in evaluation ``residual + x``.  So a call that activation checkpointing repeats has the mask of the first one (it
    restores the generator), a saved state of the generator brings the masks back, and a captured call has a new mask
    in every replay."""

    def __init__(self, p):
        super().__init__()
        assert 0 <= p < 1
        self.p = p

    def forward(self, x, residual=None):
        if not self.training or self.p == 0:
            return x if residual is None else residual + x
        return dropout(x, self.p, torch.randint(1 << 62, (2,), device=x.device), residual=residual)


class SequenceBlock(nn.Module):
    """One layer of a model over a sequence, x [batch, length, features]:
    x + dropout(attention(norm(x))), then x + dropout(two linear layers of norm(x)).

    ``forward(x, lengths)`` takes whole sequences, padded to the longest (``lengths`` int32 [batch]).
    ``step(x, keys, values, filled)`` takes new positions [batch, new, features] of sequences whose first
    ``filled`` (int32 [batch]) keys and values are kept in ``keys``, ``values`` [batch, room, kv_heads, dim]:
    it writes the new ones behind them and answers for the new positions.  A sequence whose room they exceed gives NaN (the
    numbers stay on the device), and the last of its keys and values are lost.

    With its parameters in bfloat16, or under ``torch.autocast`` to bfloat16 (``keys`` and ``values`` bfloat16 then), the products and
    attention run in that type; what goes around them keeps the type of x.
    """

    def __init__(self, features, heads, kv_heads=None, causal=False, p=0.1, num_buckets=32, reach=128, hidden=None):
        super().__init__()
        kv_heads = heads if kv_heads is None else kv_heads
        assert features % heads == 0 and heads % kv_heads == 0
        self.heads, self.kv_heads, self.dim, self.causal = heads, kv_heads, features // heads, causal
        self.norm1, self.norm2 = LayerNorm(features), LayerNorm(features)
        self.project = nn.Linear(features, (heads + 2 * kv_heads) * self.dim)
        self.bias = RelativeBias(heads, num_buckets, reach)
        self.out = nn.Linear(features, features)
        hidden = 4 * features if hidden is None else hidden
        self.mlp = nn.Sequential(nn.Linear(features, hidden), nn.GELU(), nn.Linear(hidden, features))
        self.drop1, self.drop2 = Dropout(p), Dropout(p)

    def _projected(self, x):
        return self.project(self.norm1(x)).unflatten(-1, (-1, self.dim)).split((self.heads, self.kv_heads, self.kv_heads), dim=2)

    def _rest(self, x, a):
        x = self.drop1(self.out(a.flatten(2)).to(x.dtype), residual=x)
        return self.drop2(self.mlp(self.norm2(x)).to(x.dtype), residual=x)

    def forward(self, x, lengths=None):
        q, k, v = self._projected(x)
        a = attention(q, k, v, self.bias.weight.to(q.dtype), self.bias.buckets, causal=self.causal, q_lengths=lengths, kv_lengths=lengths)
        return self._rest(x, a)

    def step(self, x, keys, values, filled):
        q, k, v = self._projected(x)
        assert x.size(1) <= keys.size(1), "step: more new positions than there is room"
        first = filled.clamp(0, keys.size(1) - x.size(1))
        at = first.long()[:, None] + torch.arange(x.size(1), device=x.device)
        which = torch.arange(x.size(0), device=x.device)[:, None]
        keys[which, at], values[which, at] = k, v
        a = attention(q, keys, values, self.bias.weight.to(q.dtype), self.bias.buckets, causal=self.causal, q_start=filled,
                      kv_lengths=filled + x.size(1))
        return self._rest(x, a.masked_fill((first != filled)[:, None, None, None], math.nan))
