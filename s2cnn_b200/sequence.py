"""Operators for sequences of spherical signals: what stands between the feature vectors that a spherical
network gives for signals in order (the frames of a recording, the shells of a volume, the rings of a
sphere) and an answer about all of them.

* ``attention`` with a learned bias by buckets of the relative position (``relative_buckets``), its output
  and its gradients computed without storing a score;
* ``norm_rotate``: heads of queries and keys normed, and turned by their position (``rotary_frequencies``), for attention without a bias;
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
from .pages import norm_rotate_store, paged_attention


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


def rotary_frequencies(dim, base=10000.0, factor=1.0, length=None, slow=1.0, fast=32.0, device=None):
    """The frequencies of ``norm_rotate``, float64 [dim / 2], radians per position: base^(-2 i / dim) for pair i.

    For recordings ``factor`` times as long as those a model was trained on they are slowed: all by the factor, or, with the
    trained ``length`` given, those that turn less than ``slow`` times over it by the factor, those that turn more than
    ``fast`` times not at all, and the ones between gradually.
    """
    assert dim >= 2 and dim % 2 == 0 and base > 0 and factor > 0 and slow < fast
    f = torch.tensor([base ** (-2 * i / dim) for i in range(dim // 2)], dtype=torch.float64)
    kept = 0.0 if length is None else ((f * length / (2 * math.pi) - slow) / (fast - slow)).clamp(0, 1)
    return (f * (kept + (1 - kept) / factor)).to(device)


def norm_rotate(q, k=None, frequencies=None, q_weight=None, k_weight=None, eps=None, positions=0, interleaved=False, magnitude=1.0):
    """Queries and keys as attention takes them: each head normed, and turned by its position, in one pass.

    :param q, k: [batch, length, heads, dim] and [batch, length, kv_heads, dim] (None: only the other), dim <= 128; any strides with a
        contiguous last axis
    :param frequencies: float64 [pairs], radians per position, see ``rotary_frequencies``; the first 2 pairs values of a head are turned,
        the others not (None: no value is).  They have no gradient; one that is infinite or NaN makes its pair NaN
    :param q_weight, k_weight: [dim], of the norm
    :param eps: x / sqrt(mean(x^2) + eps) * weight over the values of a head comes first (zeros where the sum of squares is beyond float32: values
        from some 1e19 on); None: no norm
    :param positions: of the first row, a number or int32 [batch], or of each row, int32 [batch, length]
    :param interleaved: pairs are neighbours (2 i, 2 i + 1) instead of halves (i, i + pairs)
    :param magnitude: a factor of what is turned
    :return: (q, k), contiguous

    Angles are exact modulo whole turns however far the position, sums and what is computed value by value float32.
    """
    assert eps is None or eps >= 0, "eps is negative"
    start, positions = (0, positions) if isinstance(positions, torch.Tensor) else (positions, None)
    out = list(cuda_ops().ag_norm_rotate(q, k, frequencies, q_weight, k_weight, positions, -1.0 if eps is None else float(eps), int(start), bool(interleaved),
                                         float(magnitude)))
    return out.pop(0) if q is not None else None, out.pop(0) if k is not None else None


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

    ``step_pages(x, keys, values, pages, filled)`` is ``step`` with the kept keys and values in pages (one layer of a
    ``PagedCache``): ``pages`` int32 [batch, columns].

    With ``rotary`` (an even number, at most the values of a head) positions enter by rotation instead of the bias: that many
    values of each head of queries and keys are turned (``norm_rotate``), by ``frequencies`` (those of base 10000 unless given, see
    ``rotary_frequencies``), after a norm of every head with learned weights where ``head_norm`` is set.

    With its parameters in bfloat16, or under ``torch.autocast`` to bfloat16 (``keys`` and ``values`` bfloat16 then), the products and
    attention run in that type; what goes around them keeps the type of x.
    """

    rotary, head_norm = None, False                        # (blocks saved whole before these were there)

    def __init__(self, features, heads, kv_heads=None, causal=False, p=0.1, num_buckets=32, reach=128, hidden=None, rotary=None, frequencies=None,
                 head_norm=False):
        super().__init__()
        kv_heads = heads if kv_heads is None else kv_heads
        assert features % heads == 0 and heads % kv_heads == 0
        self.heads, self.kv_heads, self.dim, self.causal = heads, kv_heads, features // heads, causal
        self.norm1, self.norm2 = LayerNorm(features), LayerNorm(features)
        self.project = nn.Linear(features, (heads + 2 * kv_heads) * self.dim)
        self.rotary, self.head_norm = rotary, head_norm
        assert rotary is not None or (frequencies is None and not head_norm), "SequenceBlock: frequencies and norms of heads come with rotary"
        self.bias = RelativeBias(heads, num_buckets, reach) if rotary is None else None
        if rotary is not None:
            frequencies = rotary_frequencies(rotary) if frequencies is None else torch.as_tensor(frequencies, dtype=torch.float64).cpu()
            assert frequencies.shape == (rotary // 2,) and rotary % 2 == 0 and rotary <= self.dim, "SequenceBlock: a frequency for each of rotary / 2 pairs"
            self._radians = frequencies
            self.register_buffer("frequencies", frequencies, persistent=False)
        if head_norm:
            self.q_norm, self.k_norm = Parameter(torch.ones(self.dim)), Parameter(torch.ones(self.dim))
        self.out = nn.Linear(features, features)
        hidden = 4 * features if hidden is None else hidden
        self.mlp = nn.Sequential(nn.Linear(features, hidden), nn.GELU(), nn.Linear(hidden, features))
        self.drop1, self.drop2 = Dropout(p), Dropout(p)

    def _projected(self, x):
        return self.project(self.norm1(x)).unflatten(-1, (-1, self.dim)).split((self.heads, self.kv_heads, self.kv_heads), dim=2)

    def _apply(self, fn, recurse=True):
        super()._apply(fn, recurse)
        if self.rotary is not None:                        # float64 whatever the parameters' type
            self.frequencies = self._radians.to(self.frequencies.device)
        return self

    def _turning(self, q):
        weights = (self.q_norm.to(q.dtype), self.k_norm.to(q.dtype)) if self.head_norm else (None, None)
        return (self.frequencies,) + weights + (1e-6 if self.head_norm else None,)

    def _placed(self, x, positions):
        """queries, keys, values of positions from ``positions`` on, and what attention adds by position"""
        q, k, v = self._projected(x)
        if self.rotary is None:
            return q, k, v, (self.bias.weight.to(q.dtype), self.bias.buckets)
        return norm_rotate(q, k, *self._turning(q), positions=positions) + (v, (None, None))

    def _rest(self, x, a):
        x = self.drop1(self.out(a.flatten(2)).to(x.dtype), residual=x)
        return self.drop2(self.mlp(self.norm2(x)).to(x.dtype), residual=x)

    def forward(self, x, lengths=None):
        q, k, v, bias = self._placed(x, 0)
        a = attention(q, k, v, *bias, causal=self.causal, q_lengths=lengths, kv_lengths=lengths)
        return self._rest(x, a)

    def step(self, x, keys, values, filled):
        q, k, v, bias = self._placed(x, filled)
        assert x.size(1) <= keys.size(1), "step: more new positions than there is room"
        first = filled.clamp(0, keys.size(1) - x.size(1))
        at = first.long()[:, None] + torch.arange(x.size(1), device=x.device)
        which = torch.arange(x.size(0), device=x.device)[:, None]
        keys[which, at], values[which, at] = k, v
        a = attention(q, keys, values, *bias, causal=self.causal, q_start=filled, kv_lengths=filled + x.size(1))
        return self._rest(x, a.masked_fill((first != filled)[:, None, None, None], math.nan))

    def step_pages(self, x, keys, values, pages, filled, lengths=None):
        """x [batch, new, features], of which ``lengths`` (int32 [batch], None: all) are filled: new positions of sequences whose first
        ``filled`` (int32 [batch]) keys and values are kept in ``keys``, ``values`` [pages, page, kv_heads, dim].  Writes the new ones to
        their pages and answers for the new positions: NaN where a position has no page.  Without gradients."""
        with torch.no_grad():
            q, k, v = self._projected(x)
            turning = self._turning(q) if self.rotary is not None else ()
            q = norm_rotate_store(q, k, v, keys, values, pages, *turning, positions=filled, lengths=lengths)
            bias = (self.bias.weight.to(q.dtype), self.bias.buckets) if self.rotary is None else (None, None)
            a = paged_attention(q, keys, values, pages, *bias, causal=self.causal, q_start=filled, q_lengths=lengths,
                                kv_lengths=filled + (x.size(1) if lengths is None else lengths.clamp(max=x.size(1))))
            return self._rest(x, a)
