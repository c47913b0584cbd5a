"""Attention with a relative bias, layer norm and dropout against their definitions in 64 bits, at the sizes, strides and
masks where they can go wrong; their gradients against differences; their refusals.

Tolerances.  eps = 2^-24 (float32) or 2^-9 (bfloat16) is half a unit in the last place.

* A float32 result sums at most a few thousand products whose terms carry a few eps each; errors of single terms are
  independent, so that the 2-norm of the error stays near eps times a small factor.  5e-6 (80 eps) leaves room for that factor
  and for the relative 2^-22 of the exponential, and is far below what a wrong term, row or bucket would cause.
* A bfloat16 result is rounded once (relative 2^-9 at most, 2^-9 / sqrt 3 in the mean); weights and score gradients may be
  rounded to bfloat16 once more on the way to the tensor cores, and the output once where the backward pass reads it: 8e-3
  is four such roundings at their largest.
"""
import math

import numpy as np
import pytest
import torch

import backends
import s2cnn_b200 as S
from s2cnn_b200 import _lib

TOL = {torch.float32: 5e-6, torch.bfloat16: 8e-3}
F32, BF16 = torch.float32, torch.bfloat16


def rel(a, b):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    assert a.shape == b.shape
    assert bool((torch.isfinite(a) == torch.isfinite(b)).all())
    d, n = (a - b).norm().item(), b.norm().item()
    return d / n if n else d


def exact_attention(q, k, v, bias=None, buckets=None, causal=False, q_start=0, q_lengths=None, kv_lengths=None, grad=None):
    """(out, dq, dk, dv, dbias) in float64, query by query; masked keys are left out, whatever they hold."""
    q, k, v = (t.detach().double().cpu() for t in (q, k, v))
    B, Lq, H, D = q.shape
    Lk, Hk = k.shape[1:3]
    out, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    table = bias.detach().double().cpu() if bias is not None else None
    dbias = torch.zeros_like(table) if table is not None else None
    reach = len(buckets) // 2 if buckets is not None else 0
    buckets = buckets.cpu().long() if buckets is not None else None
    for b in range(B):
        start = int(q_start[b]) if isinstance(q_start, torch.Tensor) else q_start
        nq = Lq if q_lengths is None else min(max(int(q_lengths[b]), 0), Lq)
        nk = Lk if kv_lengths is None else min(max(int(kv_lengths[b]), 0), Lk)
        for i in range(nq):
            n = min(nk, max(0, i + start + 1)) if causal else nk
            if n == 0:
                continue
            for h in range(H):
                kh = h // (H // Hk)
                s = k[b, :n, kh] @ q[b, i, h] / math.sqrt(D)
                if table is not None:
                    w = buckets[(torch.arange(n) - i - start).clamp(-reach, reach) + reach]
                    ok = (w >= 0) & (w < len(table))
                    s = s + torch.where(ok, table[w.clamp(0, len(table) - 1), h], 0.0)
                p = torch.softmax(s, 0)
                out[b, i, h] = p @ v[b, :n, kh]
                if grad is not None:
                    g = grad[b, i, h].detach().double().cpu()
                    dv[b, :n, kh] += p[:, None] * g
                    dp = v[b, :n, kh] @ g
                    ds = p * (dp - p @ dp)
                    dq[b, i, h] = ds @ k[b, :n, kh] / math.sqrt(D)
                    dk[b, :n, kh] += ds[:, None] * q[b, i, h] / math.sqrt(D)
                    if table is not None:
                        dbias[:, h].index_add_(0, w[ok], ds[ok])
    return out, dq, dk, dv, dbias


def normal(gen, dev, dtype, *shape):
    return torch.randn(shape, generator=gen).to(dtype).to(dev)


def check_attention(dev, dtype, B, Lq, Lk, H, Hk, D, bias=None, seed=0, packed=False, **kw):
    gen = torch.Generator().manual_seed(seed)
    if packed:
        qkv = normal(gen, dev, dtype, B, Lq, H + 2 * Hk, D)
        q, k, v = qkv.split((H, Hk, Hk), 2)
    else:
        q, k, v = (normal(gen, dev, dtype, B, *s, D) for s in ((Lq, H), (Lk, Hk), (Lk, Hk)))
    table = buckets = None
    if bias:
        table, buckets = normal(gen, dev, dtype, bias[0], H), S.relative_buckets(*bias, device=dev)
    kw = {n: torch.tensor(x, dtype=torch.int32, device=dev) if isinstance(x, list) else x for n, x in kw.items()}
    g = normal(gen, dev, dtype, B, Lq, H, D)
    want = exact_attention(q, k, v, table, buckets, grad=g, **kw)
    with torch.no_grad():
        inferred = S.attention(q, k, v, table, buckets, **kw)
    args = [t.detach().requires_grad_(True) for t in ((q, k, v) if table is None else (q, k, v, table))]
    out = S.attention(*args[:3], args[3] if table is not None else None, buckets, **kw)
    grads = torch.autograd.grad(out, args, g)
    assert rel(inferred, want[0]) <= TOL[dtype]          # (where a bias gradient may follow, weights are kept more exactly)
    for name, a, b in zip(("out", "dq", "dk", "dv", "dbias"), (out,) + tuple(grads), want):
        # one key or one bucket per row makes score gradients that are zero up to rounding: measured against what their terms are
        err = (a.double().cpu() - b).norm().item() if b.norm() < 1e-3 * g.double().norm().cpu() and name in ("dq", "dk", "dbias") else None
        assert a.dtype == dtype
        if err is not None:
            assert err <= TOL[dtype] * g.double().norm().item() * 4, (name, err)
        else:
            assert rel(a, b) <= TOL[dtype], (name, rel(a, b))
    return out


SMALL = [
    # B, Lq, Lk, H, Hk, D, bias, kw
    (1, 1, 1, 1, 1, 1, None, {}),
    (1, 12, 12, 4, 4, 10, (8, 6), {}),
    (2, 5, 9, 2, 1, 16, (8, 3), {}),
    (1, 65, 70, 2, 2, 20, (16, 30), {}),                                  # one past a tile; 40-byte rows in bfloat16
    (2, 33, 33, 4, 2, 25, (8, 6), {"causal": True}),                       # rows of odd length
    (1, 17, 129, 3, 3, 64, (32, 128), {"causal": True, "q_start": 112}),
    (3, 20, 24, 2, 2, 32, (8, 4), {"kv_lengths": [24, 0, 7], "q_lengths": [20, 20, 3]}),
    (3, 20, 24, 2, 1, 40, (8, 4), {"kv_lengths": [24, 1, 30], "q_lengths": [0, -3, 99], "causal": True, "q_start": [4, 0, -7]}),
    (2, 3, 140, 4, 1, 50, (16, 64), {"causal": True, "q_start": [137, 20], "kv_lengths": [140, 23]}),   # few rows
    (1, 2, 300, 2, 2, 128, None, {}),
]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("case", SMALL, ids=lambda c: "x".join(map(str, c[:6])))
@pytest.mark.parametrize("backend", backends.BACKENDS)
def test_attention_and_gradients(backend, case, dtype):
    with backends.active(backend) as (_, dev):
        B, Lq, Lk, H, Hk, D, bias, kw = case
        check_attention(dev, dtype, B, Lq, Lk, H, Hk, D, bias, packed=Lq == Lk, **kw)


LARGE = [
    (2, 1, 1500, 16, 1, 128, (32, 128), {"causal": True, "q_start": [1400, 37]}),          # one query, all heads on one key head
    (3, 2, 777, 10, 2, 25, (32, 64), {"kv_lengths": [777, 0, 513]}),                       # rows of 50 bytes
    (1, 4, 2000, 8, 2, 34, (16, 30), {"causal": True, "q_start": 1996}),                   # rows of 68 bytes
    (1, 1, 600, 16, 1, 128, (32, 2048), {}),                                               # bias tables beyond the shared memory
    (2, 128, 128, 2, 2, 64, (32, 128), {}),
    (1, 257, 257, 2, 2, 128, (32, 30), {"causal": True}),
    (2, 400, 400, 4, 2, 64, (32, 128), {"kv_lengths": [400, 133], "q_lengths": [400, 133], "causal": True}),
    (1, 150, 700, 3, 1, 100, (16, 64), {"q_start": 550, "causal": True}),
    (1, 700, 150, 2, 2, 16, (16, 64), {"q_start": -300, "causal": True}),
    (1, 384, 384, 2, 2, 80, (32, 400), {}),                                # the reach covers every tile
    (2, 300, 300, 1, 1, 64, None, {"kv_lengths": [0, 300]}),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("case", LARGE, ids=lambda c: "x".join(map(str, c[:6])))
def test_attention_over_many_tiles(case, dtype):
    B, Lq, Lk, H, Hk, D, bias, kw = case
    check_attention("cuda", dtype, B, Lq, Lk, H, Hk, D, bias, packed=Lq == Lk, **kw)


@pytest.mark.parametrize("backend", backends.BACKENDS)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("few", [True, False])
def test_attention_does_not_read_what_is_masked(backend, dtype, few):
    """NaN and infinities behind the lengths and where no query of the call looks reach no result and no gradient."""
    with backends.active(backend) as (_, dev):
        gen = torch.Generator().manual_seed(3)
        Lq, Lk = (2, 90) if few else (70, 90)
        q, k, v = (normal(gen, dev, dtype, 2, n, 2, 24) for n in (Lq, Lk, Lk))
        g = normal(gen, dev, dtype, 2, Lq, 2, 24)
        for kw in ({"kv_lengths": [50, 0]}, {"causal": True, "q_start": [90 - Lq - 20, 3]}, {"q_lengths": [1, 0], "kv_lengths": [90, 90]}):
            kw = {n: torch.tensor(x, dtype=torch.int32, device=dev) if isinstance(x, list) else x for n, x in kw.items()}
            q2, k2, v2, g2 = (t.clone() for t in (q, k, v, g))
            for b in range(2):
                nk = int(kw["kv_lengths"][b]) if "kv_lengths" in kw else Lk
                nq = int(kw["q_lengths"][b]) if "q_lengths" in kw else Lq
                if "causal" in kw:
                    nk = min(nk, int(kw["q_start"][b]) + Lq)
                k2[b, nk:], v2[b, nk:] = math.nan, math.inf
                q2[b, nq:], g2[b, nq:] = math.inf, math.nan
            results = []
            for qq, kk, vv, gg in ((q, k, v, g), (q2, k2, v2, g2)):
                args = [t.clone().requires_grad_(True) for t in (qq, kk, vv)]
                out = S.attention(*args, **kw)
                results.append((out,) + torch.autograd.grad(out, args, gg))
            for a, b in zip(*results):
                assert bool(torch.isfinite(b.float()).all()) and torch.equal(a, b)


@pytest.mark.parametrize("backend", backends.BACKENDS)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lq", [3, 70])
def test_bias_of_the_lowest_value_masks(backend, dtype, lq):
    """A bucket with the type's lowest value, or with -infinity, takes no weight; a row of the lowest value alone is a plain mean."""
    with backends.active(backend) as (_, dev):
        gen = torch.Generator().manual_seed(4)
        q, k, v = (normal(gen, dev, dtype, 1, n, 2, 16) for n in (lq, 80, 80))
        g = normal(gen, dev, dtype, 1, lq, 2, 16)
        buckets = S.relative_buckets(8, 4, device=dev)
        for low in (torch.finfo(dtype).min, -math.inf):
            table = torch.zeros(8, 2, dtype=dtype, device=dev)
            table[4:] = low                                      # keys behind the query
            args = [t.clone().requires_grad_(True) for t in (q, k, v)]
            out = S.attention(*args, table, buckets)
            grads = torch.autograd.grad(out, args, g)
            for a, b in zip((out,) + grads, exact_attention(q, k, v, causal=True, grad=g)):
                assert rel(a, b) <= TOL[dtype]
        table = torch.full((8, 2), torch.finfo(dtype).min, dtype=dtype, device=dev)
        vv = v.clone().requires_grad_(True)
        out = S.attention(q, k, vv, table, buckets)
        mean = v.double().cpu().mean(1, keepdim=True).expand(1, lq, 2, 16)
        assert (out.double().cpu() - mean).abs().max() <= TOL[dtype] * 4
        dv, = torch.autograd.grad(out, vv, g)
        assert rel(dv, (g.double().sum(1, keepdim=True) / 80).expand_as(v)) <= TOL[dtype]


@pytest.mark.parametrize("backend", backends.BACKENDS)
def test_attention_takes_any_strides(backend):
    with backends.active(backend) as (_, dev):
        gen = torch.Generator().manual_seed(5)
        base = normal(gen, dev, F32, 2, 4, 21, 15)               # [batch, heads, length, dim + 2]: odd rows, heads outside
        q = base.transpose(1, 2)[..., 1:14]
        k = normal(gen, dev, F32, 13, 2, 21, 4).permute(1, 2, 3, 0)           # dim outermost: copied
        v = normal(gen, dev, F32, 1, 21, 1, 13).expand(2, 21, 4, 13)          # broadcast
        want = exact_attention(q, k, v, grad=torch.ones(2, 21, 4, 13))
        vv = v[:1, :, :1].clone().requires_grad_(True)
        out = S.attention(q, k, vv.expand(2, 21, 4, 13))
        assert rel(out, want[0]) <= TOL[F32]
        dv, = torch.autograd.grad(out.sum(), vv)
        assert rel(dv, want[3].sum((0, 2), keepdim=True)) <= TOL[F32]


@pytest.mark.parametrize("backend", backends.BACKENDS)
def test_attention_without_positions(backend):
    with backends.active(backend) as (_, dev):
        for shape_q, shape_k in (((0, 3, 2, 8), (0, 4, 2, 8)), ((2, 0, 2, 8), (2, 4, 2, 8)), ((2, 3, 2, 8), (2, 0, 2, 8)), ((2, 30, 2, 8), (2, 0, 2, 8))):
            q, k = torch.ones(shape_q, device=dev, requires_grad=True), torch.ones(shape_k, device=dev, requires_grad=True)
            table = torch.zeros(8, 2, device=dev, requires_grad=True)
            out = S.attention(q, k, k, table, S.relative_buckets(8, 2, device=dev))
            assert out.shape == q.shape and not out.any()
            for g in torch.autograd.grad(out.sum(), (q, k, table)):
                assert not g.any()


@pytest.mark.parametrize("backend", backends.BACKENDS)
@pytest.mark.parametrize("lq", [2, 20])
def test_attention_gradient_against_differences(backend, lq):
    """Central differences of a weighted sum, step 1e-2: their own error is h^2 / 6 times a third derivative of order one
    (2e-5) and 2^-24 |f| / h (2e-5 for |f| of some 5)."""
    with backends.active(backend) as (_, dev):
        gen = torch.Generator().manual_seed(6)
        args = [normal(gen, dev, F32, *s) for s in ((1, lq, 2, 6), (1, 18, 1, 6), (1, 18, 1, 6), (8, 2))]
        weight = normal(gen, dev, F32, 1, lq, 2, 6) / math.sqrt(12 * lq)
        buckets = S.relative_buckets(8, 5, device=dev)
        f = lambda *a: (S.attention(*a, buckets, causal=True, q_start=18 - lq).double() * weight).sum()  # noqa: E731
        leaves = [a.clone().requires_grad_(True) for a in args]
        grads = torch.autograd.grad(f(*leaves), leaves)
        for n, (a, g) in enumerate(zip(args, grads)):
            way = normal(gen, dev, F32, *a.shape)
            way /= way.norm()
            moved = [[x + (s * 1e-2 * way if m == n else 0) for m, x in enumerate(args)] for s in (1, -1)]
            with torch.no_grad():
                slope = ((f(*moved[0]) - f(*moved[1])) / 2e-2).item()
            assert abs(slope - (g * way).sum().item()) <= 1e-4, n


@pytest.mark.gpu
def test_attention_gradients_are_reproducible():
    gen = torch.Generator().manual_seed(7)
    for dtype in (F32, BF16):
        q, k, v = (normal(gen, "cuda", dtype, 2, 300, n, 64).requires_grad_(True) for n in (4, 2, 2))
        table = normal(gen, "cuda", dtype, 16, 4).requires_grad_(True)
        g = normal(gen, "cuda", dtype, 2, 300, 4, 64)
        buckets = S.relative_buckets(16, 64, device="cuda")
        runs = []
        for _ in range(3):
            out = S.attention(q, k, v, table, buckets, causal=True)
            runs.append((out,) + torch.autograd.grad(out, (q, k, v, table), g))
        for other in runs[1:]:
            assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("case", [(8, 1000, 8, 8, 64, True), (8, 1000, 8, 8, 64, False), (5, 1000, 8, 8, 128, True), (4, 1100, 8, 8, 64, False),
                                  (13, 333, 8, 4, 128, True), (40, 64, 8, 2, 64, True), (38, 130, 4, 4, 32, False)],
                         ids=lambda c: "x".join(map(str, c)))
def test_attention_of_several_waves(case, dtype):
    """More blocks than run at once, with a last wave of any size: against whole matrices in 64 bits, and the same in every call."""
    B, L, H, Hk, D, causal = case
    gen = torch.Generator().manual_seed(17)
    q, k, v = (normal(gen, "cuda", dtype, B, L, n, D) for n in (H, Hk, Hk))
    table, g = normal(gen, "cuda", dtype, 32, H) * 2, normal(gen, "cuda", dtype, B, L, H, D)
    buckets = S.relative_buckets(32, 128, device="cuda")
    args = [t.requires_grad_(True) for t in (q, k, v, table)]
    ref = [t.detach().double().requires_grad_(True) for t in args]
    rel_pos = torch.arange(L, device="cuda") - torch.arange(L, device="cuda")[:, None]
    which = buckets.long()[rel_pos.clamp(-128, 128) + 128]
    scores = torch.einsum("bihd,bjhd->bhij", ref[0], ref[1].repeat_interleave(H // Hk, 2)) / math.sqrt(D) + ref[3][which].permute(2, 0, 1)
    if causal:
        scores = scores.masked_fill(rel_pos > 0, -math.inf)
    want = torch.einsum("bhij,bjhd->bihd", torch.softmax(scores, -1), ref[2].repeat_interleave(H // Hk, 2))
    want = (want.detach(),) + torch.autograd.grad(want, ref, g.double())
    del scores
    first = None
    for _ in range(4):
        with torch.no_grad():
            inferred = S.attention(*args, buckets, causal=causal)
        out = S.attention(*args, buckets, causal=causal)
        now = (inferred, out) + torch.autograd.grad(out, args, g)
        for name, a, b in zip(("inferred", "out", "dq", "dk", "dv", "dbias"), now, want[:1] + want):
            assert rel(a, b) <= TOL[dtype], (name, rel(a, b))
        first = first or now
        assert all(torch.equal(a, b) for a, b in zip(first, now))


@pytest.mark.gpu
def test_few_queries_agree_with_many():
    """One query of a long cache, split over the keys, beside the same query among others."""
    gen = torch.Generator().manual_seed(8)
    for dtype in (F32, BF16):
        q, k, v = (normal(gen, "cuda", dtype, 2, n, h, 64) for n, h in ((40, 4), (3000, 2), (3000, 2)))
        table, buckets = normal(gen, "cuda", dtype, 32, 4), S.relative_buckets(32, 128, device="cuda")
        every = S.attention(q, k, v, table, buckets, causal=True, q_start=2960)
        one = S.attention(q[:, 39:], k, v, table, buckets, causal=True, q_start=2999)
        assert rel(one, every[:, 39:]) <= 2 * TOL[dtype]


@pytest.mark.gpu
@pytest.mark.parametrize("lq", [1, 130])
def test_offsets_beyond_32_bits(lq):
    """Keys and values 131072 elements apart: the last of 20000 lie 2.6e9 elements behind the first."""
    gen = torch.Generator().manual_seed(16)
    k, v = (normal(gen, "cuda", BF16, 1, 20000, 1, 64) for _ in range(2))
    q = normal(gen, "cuda", BF16, 1, lq, 2, 64)
    room = torch.empty(20000, 1024, 128, dtype=BF16, device="cuda")
    far_k, far_v = room[:, :1, :64].unsqueeze(0), room[:, 1:2, 64:].unsqueeze(0)
    far_k.copy_(k)
    far_v.copy_(v)
    assert far_k.stride(1) * 19999 > 2 ** 31
    kw = {"causal": True, "q_start": 20000 - lq}
    assert torch.equal(S.attention(q, far_k, far_v, **kw), S.attention(q, k, v, **kw))
    if lq > 1:
        g = normal(gen, "cuda", BF16, 1, lq, 2, 64)
        results = []
        for kk, vv in ((far_k, far_v), (k, v)):
            args = [t.detach().requires_grad_(True) for t in (q, kk, vv)]
            results.append(torch.autograd.grad(S.attention(*args, **kw), args, g))
        assert all(torch.equal(a, b) for a, b in zip(*results))


# ---- layer norm ---------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("backend", backends.BACKENDS)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (70, 8), (5, 33), (9, 128), (2, 200), (3, 257), (2, 1000), (1, 1100)])
def test_layer_norm(backend, dtype, rows, cols):
    with backends.active(backend) as (_, dev):
        check_layer_norm(dev, dtype, rows, cols)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,cols", [(1000, 1024), (4000, 40), (33, 2048), (7, 4095), (5, 8192), (3, 16384), (20000, 24), (400, 1501)])
def test_layer_norm_wide_and_long(dtype, rows, cols):
    check_layer_norm("cuda", dtype, rows, cols)


def check_layer_norm(dev, dtype, rows, cols):
    gen = torch.Generator().manual_seed(rows * 10007 + cols)
    x, g = normal(gen, dev, dtype, rows, cols) * 2 + 3, normal(gen, dev, dtype, rows, cols)
    w, b = normal(gen, dev, dtype, cols), normal(gen, dev, dtype, cols)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    y = S.layer_norm(*leaves)
    got = (y,) + torch.autograd.grad(y, leaves, g)
    exact = [t.double().cpu().requires_grad_(True) for t in (x, w, b)]
    mean = exact[0].mean(-1, keepdim=True)
    hat = (exact[0] - mean) / ((exact[0] - mean).square().mean(-1, keepdim=True) + 1e-5).sqrt()
    want_y = hat * exact[1] + exact[2]
    want = (want_y,) + torch.autograd.grad(want_y, exact, g.double().cpu())
    # a single column is all mean: its gradient is 0 but for rounding
    for name, a, e in zip(("y", "dx", "dw", "db"), got, want):
        if cols == 1 and name in ("dx", "dw"):
            assert a.abs().max() <= 1e-4
        else:
            assert rel(a, e) <= TOL[dtype], (name, rel(a, e))
    assert torch.equal(S.layer_norm(x, w, b), y)


@pytest.mark.parametrize("backend", backends.BACKENDS)
def test_layer_norm_forms(backend):
    with backends.active(backend) as (_, dev):
        gen = torch.Generator().manual_seed(9)
        x = normal(gen, dev, F32, 2, 3, 12)
        hat = (x - x.mean(-1, keepdim=True)) / (x.var(-1, unbiased=False, keepdim=True) + 1e-3).sqrt()
        w = normal(gen, dev, F32, 12)
        assert rel(S.layer_norm(x, eps=1e-3), hat) <= TOL[F32]
        assert rel(S.layer_norm(x, w, eps=1e-3), hat * w) <= TOL[F32]
        assert rel(S.layer_norm(x, None, w, eps=1e-3), hat + w) <= TOL[F32]
        wide = normal(gen, dev, F32, 4, 30)
        assert torch.equal(S.layer_norm(wide[:, 5:18]), S.layer_norm(wide[:, 5:18].clone()))     # rows apart, unaligned
        off = torch.zeros(4 * 12 + 1, device=dev)[1:].view(4, 12).copy_(wide[:, :12])            # 4 bytes past 16
        assert torch.equal(S.layer_norm(off), S.layer_norm(wide[:, :12].clone()))
        big = 1e4 + normal(gen, dev, F32, 4, 64)                                                # mean far above the deviation
        ref = big.double().cpu()
        ref = (ref - ref.mean(-1, keepdim=True)) / (ref.var(-1, unbiased=False, keepdim=True) + 1e-5).sqrt()
        assert rel(S.layer_norm(big), ref) <= 2e-3                    # 1e4 2^-24 / 1 per value of the mean
        none = torch.zeros(0, 12, device=dev, requires_grad=True)
        w.requires_grad_(True)
        y = S.layer_norm(none, w)
        gx, gw = torch.autograd.grad(y.sum(), (none, w))
        assert y.shape == (0, 12) and gx.shape == (0, 12) and not gw.any()
        x.requires_grad_(True)                                        # single gradients
        gx, = torch.autograd.grad(S.layer_norm(x, w.detach()).square().sum(), x)
        gw, = torch.autograd.grad(S.layer_norm(x.detach(), w).square().sum(), w)
        assert rel(gw, (2 * S.layer_norm(x, w) * S.layer_norm(x)).sum((0, 1))) <= TOL[F32] and gx.shape == x.shape


# ---- dropout ------------------------------------------------------------------------------------------------------------


def words(n, seed, step):
    """The generator's words in whole numbers of Python."""
    out = []
    for block in range(-(-n // 4)):
        a, b, c, d = block & 0xFFFFFFFF, block >> 32, step & 0xFFFFFFFF, step >> 32
        k0, k1 = seed & 0xFFFFFFFF, seed >> 32
        for _ in range(7):
            x, y = 0xD2511F53 * a, 0xCD9E8D57 * c
            a, b, c, d = (y >> 32) ^ b ^ k0, y & 0xFFFFFFFF, (x >> 32) ^ d ^ k1, x & 0xFFFFFFFF
            k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
        out += [a, b, c, d]
    return np.array(out[:n], dtype=np.uint64)


@pytest.mark.parametrize("backend", backends.BACKENDS)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [1, 4, 7, 64, 1023, 5000])
def test_dropout(backend, dtype, n):
    with backends.active(backend) as (_, dev):
        gen = torch.Generator().manual_seed(n)
        x, r, g = (normal(gen, dev, dtype, n) for _ in range(3))
        for p, seed, step in ((0.1, 5, 0), (0.5, 2 ** 62 + 12345, 2 ** 40 + 7), (0.0, 1, 1), (0.999, 3, 2)):
            keep = torch.from_numpy(words(n, seed, step) >= np.uint64(int(p * 2 ** 32)))
            f = keep.double() / (1 - p)
            xx, rr = x.clone().requires_grad_(True), r.clone().requires_grad_(True)
            y = S.dropout(xx, p, seed, step, residual=rr)
            gx, gr = torch.autograd.grad(y, (xx, rr), g)
            for a, e in ((S.dropout(x, p, seed, step), x.double().cpu() * f), (y, r.double().cpu() + x.double().cpu() * f), (gx, g.double().cpu() * f)):
                assert rel(a, e) <= TOL[dtype]
            assert torch.equal(gx != 0, (keep.to(dev) & (g != 0))) and torch.equal(gr, g)


@pytest.mark.parametrize("backend", backends.BACKENDS)
def test_dropout_mask_does_not_depend_on_shape_or_alignment(backend):
    with backends.active(backend) as (_, dev):
        x = torch.ones(6, 50, device=dev)
        y = S.dropout(x, 0.3, 11, 4)
        off = torch.ones(301, device=dev)[1:]
        assert torch.equal(S.dropout(off, 0.3, 11, 4), y.flatten())
        assert torch.equal(S.dropout(torch.ones(50, 6, device=dev).t(), 0.3, 11, 4), y)
        assert torch.equal(S.dropout(x.to(BF16), 0.3, 11, 4) != 0, y != 0)
        assert not torch.equal(S.dropout(x, 0.3, 11, 5), y) and not torch.equal(S.dropout(x, 0.3, 12, 4), y)
        assert S.dropout(torch.zeros(0, device=dev), 0.3, 1).shape == (0,)
        nan = torch.full((40,), math.nan, device=dev)                 # a dropped NaN is gone
        z = S.dropout(nan, 0.5, 1, 1, residual=torch.zeros(40, device=dev))
        assert torch.equal(torch.isnan(z), S.dropout(torch.ones(40, device=dev), 0.5, 1, 1) != 0)


@pytest.mark.gpu
def test_dropout_keeps_the_expected_share():
    """2^24 elements: the share kept is 1 - p within five standard deviations, sqrt(p (1 - p) 2^-24) each."""
    x = torch.ones(1 << 24, device="cuda")
    for p in (0.1, 0.5):
        share = (S.dropout(x, p, 77, 3) != 0).double().mean().item()
        assert abs(share - (1 - p)) <= 5 * math.sqrt(p * (1 - p) / (1 << 24))


# ---- refusals -------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("backend", backends.BACKENDS)
def test_refusals(backend):
    with backends.active(backend) as (ops, dev):
        t = lambda *s, d=F32: torch.zeros(s, dtype=d, device=dev)  # noqa: E731
        i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
        q, k = t(2, 3, 4, 8), t(2, 5, 2, 8)
        buckets, table = S.relative_buckets(8, 4, device=dev), t(8, 4)
        for call in (lambda: S.attention(q, k, t(2, 5, 2, 7)), lambda: S.attention(q, t(2, 5, 3, 8), t(2, 5, 3, 8)),
                     lambda: S.attention(q, t(1, 5, 2, 8), t(1, 5, 2, 8)), lambda: S.attention(q[0], k, k), lambda: S.attention(q, k, k, table),
                     lambda: S.attention(q, k, k, None, buckets), lambda: S.attention(q, k, k, t(8, 3), buckets),
                     lambda: S.attention(q, k, k, table, buckets[1:]), lambda: S.attention(q, k, k, kv_lengths=i32(1)),
                     lambda: S.attention(q, k, k, q_start=i32(1, 2, 3)), lambda: S.attention(q, k, k, q_lengths=i32(1, 2, 3, 4)[::2]),
                     lambda: S.layer_norm(t(3, 4), t(5)), lambda: S.layer_norm(t()), lambda: S.layer_norm(t(3, 4), eps=-1.0),
                     lambda: S.dropout(t(3), 1.0, 1), lambda: S.dropout(t(3), -0.1, 1), lambda: S.dropout(t(3), 0.1, -1),
                     lambda: S.dropout(t(3), 0.1, 1, residual=t(4)), lambda: S.relative_buckets(7, 10), lambda: S.relative_buckets(32, 3)):
            with pytest.raises(AssertionError):
                call()
        for call in (lambda: S.attention(t(2, 3, 4, 8, d=torch.float16), k, k), lambda: S.attention(q, k.to(BF16), k),
                     lambda: S.attention(q, k, k, table.to(BF16), buckets), lambda: S.attention(q, k, k, table, buckets.long()),
                     lambda: S.attention(q, k, k, kv_lengths=torch.zeros(2, device=dev)), lambda: S.layer_norm(t(3, 4, d=torch.float64)),
                     lambda: S.layer_norm(t(3, 4), t(4, d=BF16)), lambda: S.dropout(t(3, d=torch.int32), 0.1, 1)):
            with pytest.raises(TypeError):
                call()
        for call in (lambda: S.attention(t(1, 1, 1, 129), t(1, 1, 1, 129), t(1, 1, 1, 129)), lambda: S.layer_norm(t(1, 16385)),
                     lambda: S.attention(q, k, k, t(2000, 4), buckets), lambda: S.attention(q, k, k, table, i32(*[0] * 4099)),
                     lambda: S.attention(q, k, k, scale=math.inf)):
            with pytest.raises(_lib.S2cError):
                call()
        if dev.type == "cuda":
            with pytest.raises(_lib.S2cError):
                S.attention(q.cpu(), k.cpu(), k.cpu())
            with pytest.raises((TypeError, AssertionError, _lib.S2cError)):
                S.layer_norm(q, torch.zeros(8))


@pytest.mark.parametrize("backend", backends.BACKENDS)
def test_buckets_outside_the_table_add_nothing(backend):
    with backends.active(backend) as (_, dev):
        gen = torch.Generator().manual_seed(12)
        q, k, v, g = (normal(gen, dev, F32, 1, 30, 2, 8) for _ in range(4))
        buckets = torch.tensor([0, -5, 2, 1000000, 1, -2 ** 31, 2 ** 31 - 1], dtype=torch.int32, device=dev)
        table = normal(gen, dev, F32, 3, 2)
        want = exact_attention(q, k, v, table, buckets, grad=g)
        tt = table.clone().requires_grad_(True)
        out = S.attention(q, k, v, tt, buckets)
        assert rel(out, want[0]) <= TOL[F32] and rel(torch.autograd.grad(out, tt, g)[0], want[4]) <= TOL[F32]


@pytest.mark.parametrize("backend", backends.BACKENDS)
def test_workspaces_are_checked(backend):
    with backends.active(backend) as (ops, dev):
        x = torch.zeros(100, 64, device=dev)
        stats = torch.zeros(100, 2, device=dev)
        stream = torch.cuda.current_stream().cuda_stream if dev.type == "cuda" else None
        need = ops.lib.s2c_layer_norm_backward_workspace(100, 64)
        assert need > 0 and ops.lib.s2c_layer_norm_backward_workspace(0, 64) == 0
        args = (0, x.data_ptr(), None, stats.data_ptr(), x.data_ptr(), x.data_ptr(), x.data_ptr(), None, 100, 64)
        with pytest.raises(_lib.S2cError, match="status 3"):
            ops.lib.call("s2c_layer_norm_backward", *args, None, need, stream)
        with pytest.raises(_lib.S2cError, match="status 3"):
            ops.lib.call("s2c_layer_norm_backward", *args, x.data_ptr(), need - 1, stream)
        with pytest.raises(_lib.S2cError, match="status 1"):
            ops.lib.call("s2c_dropout", 2, x.data_ptr(), None, x.data_ptr(), 10, 0.5, 1, 1, stream)
        with pytest.raises(_lib.S2cError, match="status 1"):
            ops.lib.call("s2c_attention", None, None, None, None, None, None, None, None, 0, stream)


# ---- together -------------------------------------------------------------------------------------------------------------


def plain_block(m, x, mask):
    """SequenceBlock in float64 from its parameters, dropout off; mask [batch, query, key]."""
    p = {n: t.detach().double().cpu() for n, t in m.state_dict().items()}
    norm = lambda t, n: torch.nn.functional.layer_norm(t, t.shape[-1:], p[n + ".weight"], p[n + ".bias"])  # noqa: E731
    linear = lambda t, n: t @ p[n + ".weight"].t() + p[n + ".bias"]  # noqa: E731
    q, k, v = linear(norm(x, "norm1"), "project").unflatten(-1, (-1, m.dim)).split((m.heads, m.kv_heads, m.kv_heads), 2)
    k, v = (t.repeat_interleave(m.heads // m.kv_heads, 2) for t in (k, v))
    n, buckets = x.size(1), m.bias.buckets.cpu().long()
    reach = len(buckets) // 2
    d = (torch.arange(n) - torch.arange(n)[:, None]).clamp(-reach, reach) + reach
    s = torch.einsum("bihd,bjhd->bhij", q, k) / math.sqrt(m.dim) + p["bias.weight"][buckets[d]].permute(2, 0, 1)
    a = torch.einsum("bhij,bjhd->bihd", torch.softmax(s.masked_fill(~mask[:, None], -math.inf), -1), v).flatten(2)
    x = x + linear(a, "out")
    return x + linear(torch.nn.functional.gelu(linear(norm(x, "norm2"), "mlp.0")), "mlp.2")


@pytest.mark.parametrize("backend", backends.BACKENDS)
def test_block_whole_and_step_by_step(backend):
    with backends.active(backend) as (_, dev):
        torch.manual_seed(13)
        m = S.SequenceBlock(24, 4, kv_heads=2, causal=True, p=0.2, num_buckets=8, reach=6).to(dev).eval()
        with torch.no_grad():
            m.bias.weight.normal_()
            x = torch.randn(2, 9, 24, device=dev)
            seen = torch.ones(9, 9, dtype=torch.bool).tril().expand(2, 9, 9)
            whole = m(x)
            assert rel(whole, plain_block(m, x.double().cpu(), seen)) <= 4 * TOL[F32]
            keys, values = (torch.full((2, 16, 2, 6), math.nan, device=dev) for _ in range(2))
            parts, filled = [], torch.zeros(2, dtype=torch.int32, device=dev)
            for n in (4, 1, 1, 3):
                parts.append(m.step(x[:, int(filled[0]):int(filled[0]) + n], keys, values, filled))
                filled = filled + n
            assert rel(torch.cat(parts, 1), whole) <= 4 * TOL[F32]
        m.train()
        a, b = m(x), m(x)
        assert not torch.equal(a, b)                       # every call a mask of its own
        a.sum().backward()
        assert all(t.grad is not None and bool(torch.isfinite(t.grad).all()) for t in m.parameters())


@pytest.mark.parametrize("backend", backends.BACKENDS)
def test_network_over_sequences_of_signals(backend):
    """What is padded changes no answer, the signals' order does, and every parameter has a gradient."""
    with backends.active(backend) as (_, dev):
        torch.manual_seed(14)
        m = S.models.SphereSequenceNet(f1=2, f2=8, f_output=3, b_in=4, b_l1=3, b_l2=2, heads=2, num_buckets=8, reach=3).to(dev).eval()
        x = torch.randn(2, 5, 1, 8, 8, device=dev)
        lengths = torch.tensor([5, 3], dtype=torch.int32, device=dev)
        with torch.no_grad():
            for block in m.blocks:
                block.bias.weight.normal_()
            y = m(x, lengths)
            other = x.clone()
            other[1, 3:] = torch.randn(2, 1, 8, 8, device=dev)
            assert torch.equal(m(other, lengths), y)
            assert rel(m(x[1:, :3], None), y[1:]) <= 4 * TOL[F32]
            assert rel(m(x[:1].flip(1), None), y[:1]) > 1e-3
        m.train()
        m(x, lengths).square().sum().backward()
        for name, t in m.named_parameters():
            assert t.grad is not None and bool(torch.isfinite(t.grad).all()), name


@pytest.mark.gpu
@pytest.mark.parametrize("mode", [1, 2])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_either_kind_of_kernels_takes_every_size(mode, dtype):
    """The tiles on the FP32 pipes at many tiles, the tensor cores at parts of one."""
    lib = _lib.cuda_lib()
    lib.s2c_debug_attention(mode)
    try:
        cases = SMALL[1:] if mode == 2 else LARGE[:4] + LARGE[-7:]
        for B, Lq, Lk, H, Hk, D, bias, kw in cases:
            check_attention("cuda", dtype, B, Lq, Lk, H, Hk, D, bias, packed=Lq == Lk, **kw)
    finally:
        lib.s2c_debug_attention(0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_operators_on_another_stream_and_in_a_graph(dtype):
    """Work and scratch space follow the current stream, and a captured forward pass gives what the call gave."""
    gen = torch.Generator().manual_seed(15)
    q, k, v = (normal(gen, "cuda", dtype, 2, 200, n, 64) for n in (4, 2, 2))
    table, buckets = normal(gen, "cuda", dtype, 16, 4), S.relative_buckets(16, 64, device="cuda")
    x, w = normal(gen, "cuda", dtype, 200, 96), normal(gen, "cuda", dtype, 96)

    def run():
        return (S.attention(q, k, v, table, buckets), S.attention(q[:, :1], k, v, table, buckets), S.layer_norm(x, w, w),
                S.dropout(x, 0.2, 9, 1, residual=x))

    want = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
