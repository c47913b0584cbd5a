"""Norm of heads and rotation by position against their definition in 64 bits, at the head sizes, layouts, strides and positions where
they can go wrong; their gradients against the formula's and against differences; their refusals.

Tolerances (2-norms, relative).  float32: a value is a sum of two products of values that carry some ten roundings of 2^-24 and
the series of sine and cosine (2^-24); the sum of squares has at most 128 terms: 2e-6 is 32 units of 2^-24.  The gradient through a norm is a difference, rstd (h - x^ mean(h x^)),
whose error is that of its terms: 2e-6 of ||rstd h||, which the difference may be far below (heads of two values: by a
factor of hundreds; of one value: it is 0).  A weight gradient sums heads x
positions products in float32 in chains of up to some hundred: 5e-6.  bfloat16: a result is rounded once, by 2^-8 of the value at most:
4e-3 is that and the float32 error before it.
"""
import math
from fractions import Fraction

import pytest
import torch

import backends
import s2cnn_b200 as S

F32, BF16 = torch.float32, torch.bfloat16
TOL = {F32: 2e-6, BF16: 4e-3}
TOL_SUM = {F32: 5e-6, BF16: 4e-3}


def rel(a, b):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    assert a.shape == b.shape
    d, n = (a - b).norm().item(), b.norm().item()
    return d / n if n else d


def normal(gen, dev, dtype, *shape, scale=1.0, shift=0.0):
    return (torch.randn(shape, generator=gen) * scale + shift).to(dtype).to(dev)


def where(positions, batch, length):
    """[batch, length] of Python's whole numbers"""
    if not isinstance(positions, torch.Tensor):
        return [[positions + i for i in range(length)] for _ in range(batch)]
    p = positions.tolist()
    return p if positions.dim() == 2 else [[a + i for i in range(length)] for a in p]


TWO_PI = 2 * Fraction("3.14159265358979323846264338327950288419716939937510582097494459")


def exact(x, w, frequencies, eps, positions, interleaved, magnitude, fixed=False):
    """In float64; angles by whole numbers of Python, modulo a turn.  ``fixed``: the norm's divisor is taken as a constant."""
    x = x.double().cpu()
    B, L, H, D = x.shape
    if eps is not None:
        size = (x.square().mean(-1, keepdim=True) + eps).sqrt()
        x = x / (size.detach() if fixed else size)
        if w is not None:
            x = x * w.double().cpu()
    f = [] if frequencies is None else frequencies.cpu().tolist()
    at = where(positions, B, L)
    turns = torch.tensor([[[float(Fraction(a) * p / TWO_PI % 1) for a in f] for p in row] for row in at], dtype=torch.float64).view(B, L, 1, len(f))
    c, s = torch.cos(2 * math.pi * turns) * magnitude, torch.sin(2 * math.pi * turns) * magnitude
    n = len(f)
    first, second = (list(range(0, 2 * n, 2)), list(range(1, 2 * n, 2))) if interleaved else (list(range(n)), list(range(n, 2 * n)))
    parts = [None] * D
    a, b = x[..., first], x[..., second]
    ta, tb = a * c - b * s, a * s + b * c
    for k in range(n):
        parts[first[k]], parts[second[k]] = ta[..., k], tb[..., k]
    for k in range(2 * n, D):
        parts[k] = x[..., k]
    return torch.stack(parts, -1)


def check(dev, dtype, B, L, H, Hk, D, pairs, interleaved=False, eps=1e-6, weights=True, positions=0, magnitude=1.0, seed=0, packed=True):
    gen = torch.Generator().manual_seed(seed)
    if packed:
        q, k, _ = normal(gen, dev, dtype, B, L, H + 2 * Hk, D, scale=1.5).split((H, Hk, Hk), 2)
    else:
        q, k = normal(gen, dev, dtype, B, L, H, D), normal(gen, dev, dtype, B, L, Hk, D)
    wq, wk = (normal(gen, dev, dtype, D, scale=0.3, shift=1.0) for _ in range(2)) if weights and eps is not None else (None, None)
    f = S.rotary_frequencies(2 * pairs, device=dev) if pairs else None
    if isinstance(positions, list):
        positions = torch.tensor(positions, dtype=torch.int32, device=dev)
    gq, gk = normal(gen, dev, dtype, B, L, H, D), normal(gen, dev, dtype, B, L, Hk, D)
    how = dict(positions=positions, interleaved=interleaved, magnitude=magnitude)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, wq, wk) if t is not None]
    ref = [t.detach().double().cpu().requires_grad_(True) for t in leaves]
    args = lambda t: (t[0], t[1], f) + (tuple(t[2:]) if len(t) == 4 else (None, None)) + (eps,)  # noqa: E731
    out = S.norm_rotate(*args(leaves), **how)
    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(out, S.norm_rotate(*args(leaves), **how)))
    want = [exact(x, w, f, eps, positions, interleaved, magnitude) for x, w in zip(ref[:2], ref[2:] or (None, None))]
    grads, exact_grads = torch.autograd.grad(out, leaves, (gq, gk)), torch.autograd.grad(want, ref, (gq.double().cpu(), gk.double().cpu()))
    fixed = [exact(x, w, f, eps, positions, interleaved, magnitude, True) for x, w in zip(ref[:2], ref[2:] or (None, None))]
    terms = dict(zip(("dq", "dk"), torch.autograd.grad(fixed, ref[:2], (gq.double().cpu(), gk.double().cpu()))))
    for name, a, b in zip(("q", "k", "dq", "dk", "dwq", "dwk"), tuple(out) + grads, tuple(want) + exact_grads):
        assert a.dtype == dtype and a.is_contiguous() and a.shape == b.shape
        error, size = (a.detach().double().cpu() - b).norm().item(), b.norm().item()
        bound = (TOL_SUM if name.startswith("dw") else TOL)[dtype] * size + (TOL[F32] * terms[name].norm().item() if name in terms else 0)
        assert error <= bound, (name, error, size)


CASES = [
    # B, L, H, Hk, D, pairs, kw
    (1, 1, 1, 1, 1, 0, {}),
    (1, 1, 1, 1, 2, 1, {"positions": 3}),
    (2, 5, 4, 4, 10, 5, {}),
    (2, 5, 4, 2, 10, 5, {"interleaved": True, "positions": [7, 900]}),
    (1, 9, 2, 1, 25, 12, {"positions": -4}),
    (1, 9, 2, 1, 25, 12, {"interleaved": True, "eps": None}),
    (1, 7, 3, 1, 25, 5, {"magnitude": 1.3}),                                # parts of odd length stay
    (2, 3, 5, 1, 32, 16, {"positions": [[5, 3, 1], [0, 100, 7]]}),
    (1, 3, 1, 1, 33, 8, {"interleaved": True, "magnitude": 0.5}),
    (1, 6, 6, 2, 64, 32, {"eps": None, "positions": 40}),
    (1, 6, 6, 2, 64, 16, {"weights": False}),
    (2, 2, 3, 3, 80, 20, {"packed": False}),
    (1, 5, 2, 2, 100, 50, {"interleaved": True}),
    (1, 4, 9, 1, 128, 64, {"positions": 1000}),
    (1, 4, 2, 2, 128, 64, {"interleaved": True, "eps": 0.5}),
    (1, 4, 2, 2, 128, 24, {}),
    (1, 3, 2, 2, 16, 0, {}),                                                # a norm alone
]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c[:6])))
@pytest.mark.parametrize("backend", backends.BACKENDS)
def test_norm_rotate_and_gradients(backend, case, dtype):
    with backends.active(backend) as (_, dev):
        B, L, H, Hk, D, pairs, kw = case
        check(dev, dtype, B, L, H, Hk, D, pairs, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("case", [(4, 700, 16, 4, 128, 64, {}), (2, 1001, 8, 8, 25, 12, {"interleaved": True, "positions": [100000, 5]}), (32, 60, 4, 4, 10, 5, {}),
                                  (1, 2049, 12, 4, 64, 16, {"eps": None})], ids=lambda c: "x".join(map(str, c[:6])))
def test_norm_rotate_of_many_blocks(case, dtype):
    B, L, H, Hk, D, pairs, kw = case
    check("cuda", dtype, B, L, H, Hk, D, pairs, **kw)


@pytest.mark.parametrize("backend", backends.BACKENDS)
@pytest.mark.parametrize("interleaved", [False, True])
def test_far_positions(backend, interleaved):
    """Up to 2^31 - 1, and negative ones.  f / 2 pi is rounded by 2^-53 of itself and held in units of 2^-64 turns: 2^31 positions
    away that is an angle of at most 2^31 (2^-53 + 2 pi 2^-64) < 3e-7, beside 2^-24 of the series."""
    with backends.active(backend) as (_, dev):
        gen = torch.Generator().manual_seed(1)
        q = normal(gen, dev, F32, 1, 8, 1, 64)
        f = S.rotary_frequencies(64, device=dev)
        at = torch.tensor([[2 ** 31 - 1, 2 ** 30 + 12345, -(2 ** 31), -77777777, 131072, 1000003, -1, 0]], dtype=torch.int32, device=dev)
        out, none = S.norm_rotate(q, None, f, positions=at, interleaved=interleaved)
        assert none is None
        assert rel(out, exact(q, None, f, None, at, interleaved, 1.0)) <= TOL[F32]
        # the positions that follow a first one pass 2^31 without turning round
        out, _ = S.norm_rotate(q, None, f, positions=torch.tensor([2 ** 31 - 3], dtype=torch.int32, device=dev), interleaved=interleaved)
        assert rel(out, exact(q, None, f, None, 2 ** 31 - 3, interleaved, 1.0)) <= TOL[F32]


@pytest.mark.parametrize("backend", backends.BACKENDS)
def test_scores_depend_on_the_distance_alone(backend):
    with backends.active(backend) as (_, dev):
        gen = torch.Generator().manual_seed(2)
        q, k = normal(gen, dev, F32, 1, 1, 1, 32), normal(gen, dev, F32, 1, 1, 1, 32)
        f = S.rotary_frequencies(32, device=dev)
        scores = []
        for at in (0, 1000, 12345678):
            a, _ = S.norm_rotate(q, None, f, positions=at + 17)
            _, b = S.norm_rotate(None, k, f, positions=at)
            scores.append((a * b).sum().item())
        assert max(scores) - min(scores) <= 32 * 2e-6 * (q.norm() * k.norm()).item() / 4


@pytest.mark.parametrize("backend", backends.BACKENDS)
def test_gradient_against_differences(backend):
    """Central differences, step 1e-2: h^2 / 6 times a third derivative of order one (2e-5) and 2^-24 |f| / h (2e-5)."""
    with backends.active(backend) as (_, dev):
        gen = torch.Generator().manual_seed(3)
        args = [normal(gen, dev, F32, *s) for s in ((1, 3, 2, 10), (1, 3, 1, 10), (10,), (10,))]
        gq, gk = normal(gen, dev, F32, 1, 3, 2, 10) / 8, normal(gen, dev, F32, 1, 3, 1, 10) / 8
        f = S.rotary_frequencies(8, device=dev)

        def value(q, k, wq, wk):
            a, b = S.norm_rotate(q, k, f, wq, wk, eps=0.1, positions=5, magnitude=1.2)
            return (a.double() * gq).sum() + (b.double() * gk).sum()

        leaves = [a.clone().requires_grad_(True) for a in args]
        grads = torch.autograd.grad(value(*leaves), leaves)
        for n, (a, g) in enumerate(zip(args, grads)):
            way = normal(gen, dev, F32, *a.shape)
            way /= way.norm()
            moved = [[x + (s * 1e-2 * way if m == n else 0) for m, x in enumerate(args)] for s in (1, -1)]
            with torch.no_grad():
                slope = ((value(*moved[0]) - value(*moved[1])) / 2e-2).item()
            assert abs(slope - (g * way).sum().item()) <= 1e-4, n


@pytest.mark.parametrize("backend", backends.BACKENDS)
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides_and_alignment(backend, dtype):
    """The same values however they lie: results to the last bit, gradients of broadcast heads as sums."""
    with backends.active(backend) as (_, dev):
        gen = torch.Generator().manual_seed(4)
        f = S.rotary_frequencies(16, device=dev)
        w = normal(gen, dev, dtype, 16)
        q = normal(gen, dev, dtype, 2, 3, 4, 16)
        want, _ = S.norm_rotate(q, None, f, w, eps=1e-6, positions=2)
        room = torch.zeros(2, 4, 3, 21, dtype=dtype, device=dev)
        room[..., 3:19] = q.transpose(1, 2)
        odd = room[..., 3:19].transpose(1, 2)                                   # heads outside, rows off every boundary
        flat = torch.zeros(q.numel() + 1, dtype=dtype, device=dev)[1:].view(q.shape).copy_(q)
        turned = q.permute(3, 0, 1, 2).contiguous().permute(1, 2, 3, 0)         # dim outermost
        for x in (odd, flat, turned):
            assert torch.equal(S.norm_rotate(x, None, f, w, eps=1e-6, positions=2)[0], want)
        one = q[:, :, :1].clone().requires_grad_(True)
        a, _ = S.norm_rotate(one.expand(2, 3, 4, 16), None, f, eps=1e-6)
        b, _ = S.norm_rotate(one, None, f, eps=1e-6)
        g = normal(gen, dev, dtype, 2, 3, 4, 16)
        ga, = torch.autograd.grad(a, one, g)
        gb, = torch.autograd.grad(b, one, g.float().sum(2, keepdim=True).to(dtype))
        # (bfloat16: four roundings of 2^-9 in the mean are summed, and the sum rounded on either side)
        assert rel(ga, gb) <= {F32: 4e-6, BF16: 1.6e-2}[dtype]


@pytest.mark.parametrize("backend", backends.BACKENDS)
def test_single_outputs_and_inputs(backend):
    with backends.active(backend) as (_, dev):
        gen = torch.Generator().manual_seed(5)
        f = S.rotary_frequencies(12, device=dev)
        q, k = normal(gen, dev, F32, 2, 3, 4, 12).requires_grad_(True), normal(gen, dev, F32, 2, 3, 2, 12).requires_grad_(True)
        w = normal(gen, dev, F32, 12).requires_grad_(True)
        a, b = S.norm_rotate(q, k, f, w, w, eps=1e-6)
        assert torch.equal(S.norm_rotate(q, None, f, w, eps=1e-6)[0], a) and torch.equal(S.norm_rotate(None, k, f, None, w, eps=1e-6)[1], b)
        both = torch.autograd.grad(a.square().sum() + b.sum(), (q, k, w), retain_graph=True)
        alone = torch.autograd.grad(S.norm_rotate(q, None, f, w, eps=1e-6)[0].square().sum(), (q, w))
        rest = torch.autograd.grad(S.norm_rotate(None, k, f, None, w, eps=1e-6)[1].sum(), (k, w))
        assert torch.equal(both[0], alone[0]) and torch.equal(both[1], rest[0]) and rel(both[2], alone[1] + rest[1]) <= TOL[F32]
        only, none, _ = torch.autograd.grad(a.square().sum(), (q, k, w), allow_unused=True)          # one output alone
        assert torch.equal(only, alone[0]) and (none is None or not none.any())
        gw, = torch.autograd.grad(S.norm_rotate(q.detach(), k.detach(), f, w, None, eps=1e-6)[0].square().sum(), w)
        assert torch.equal(gw, alone[1])


@pytest.mark.parametrize("backend", backends.BACKENDS)
def test_without_rows(backend):
    with backends.active(backend) as (_, dev):
        f = S.rotary_frequencies(8, device=dev)
        for shape in ((0, 3, 2, 8), (2, 0, 2, 8), (2, 3, 0, 8)):
            q, w = torch.ones(shape, device=dev, requires_grad=True), torch.ones(8, device=dev, requires_grad=True)
            k = torch.ones(shape[:2] + (1, 8), device=dev, requires_grad=True)
            a, b = S.norm_rotate(q, k, f, w, w, eps=1e-6)
            assert a.shape == q.shape and b.shape == k.shape
            gq, gw = torch.autograd.grad(a.sum(), (q, w))
            assert gq.shape == q.shape and not gw.any()


@pytest.mark.parametrize("backend", backends.BACKENDS)
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_what_is_no_number_stays_in_its_head(backend, dtype):
    """Without a norm: in its pair; what is not turned passes as it is."""
    with backends.active(backend) as (_, dev):
        gen = torch.Generator().manual_seed(6)
        f = S.rotary_frequencies(8, device=dev)
        q = normal(gen, dev, dtype, 1, 4, 3, 12)
        want, _ = S.norm_rotate(q, None, f, positions=3)
        bad = q.clone()
        bad[0, 1, 2, 2], bad[0, 2, 0, 10], bad[0, 3, 1, 9] = math.inf, math.inf, math.nan
        out, _ = S.norm_rotate(bad, None, f, positions=3)
        assert not torch.isfinite(out[0, 1, 2, [2, 6]]).any() and out[0, 2, 0, 10] == math.inf and out[0, 3, 1, 9].isnan()
        out[0, 1, 2, [2, 6]], out[0, 2, 0, 10], out[0, 3, 1, 9] = want[0, 1, 2, [2, 6]], want[0, 2, 0, 10], want[0, 3, 1, 9]
        assert torch.equal(out, want)
        normed, _ = S.norm_rotate(bad, None, f, eps=1e-6)
        fine, _ = S.norm_rotate(q, None, f, eps=1e-6)
        keep = torch.ones(1, 4, 3, dtype=torch.bool, device=dev)
        keep[0, 1, 2] = keep[0, 2, 0] = keep[0, 3, 1] = False
        assert torch.equal(normed[keep], fine[keep])
        # a head of zeros is one of zeros, and a large one does not overflow its own norm's result
        zero, _ = S.norm_rotate(torch.zeros(1, 1, 1, 12, dtype=dtype, device=dev), None, f, eps=1e-6)
        assert not zero.any()


@pytest.mark.parametrize("backend", backends.BACKENDS)
def test_gradients_are_reproducible_and_refuse_seconds(backend):
    with backends.active(backend) as (_, dev):
        gen = torch.Generator().manual_seed(7)
        f = S.rotary_frequencies(32, device=dev)
        q, w = normal(gen, dev, F32, 2, 40, 4, 32).requires_grad_(True), normal(gen, dev, F32, 32).requires_grad_(True)
        g = normal(gen, dev, F32, 2, 40, 4, 32)
        runs = [torch.autograd.grad(S.norm_rotate(q, None, f, w, eps=1e-6)[0], (q, w), g) for _ in range(3)]
        for other in runs[1:]:
            assert all(torch.equal(a, b) for a, b in zip(runs[0], other))
        first, = torch.autograd.grad(S.norm_rotate(q, None, f, w, eps=1e-6)[0].square().sum(), q, create_graph=True)
        with pytest.raises(RuntimeError, match="second derivative"):
            torch.autograd.grad(first.sum(), q)


@pytest.mark.parametrize("backend", backends.BACKENDS)
@pytest.mark.filterwarnings("ignore")
def test_traced_calls(backend):
    with backends.active(backend) as (_, dev):
        gen = torch.Generator().manual_seed(8)
        fr = S.rotary_frequencies(8, device=dev)
        w, k = normal(gen, dev, F32, 8), normal(gen, dev, F32, 1, 30, 1, 8)
        f = lambda x: S.norm_rotate(x, k, fr, w, None, eps=1e-6, positions=3)  # noqa: E731
        x, y = normal(gen, dev, F32, 1, 30, 2, 8), normal(gen, dev, F32, 1, 30, 2, 8)
        traced = torch.jit.trace(f, x.clone().requires_grad_(True), check_trace=False)
        assert all(torch.equal(a, b) for a, b in zip(traced(y), f(y)))
        a, b = y.clone().requires_grad_(True), y.clone().requires_grad_(True)
        traced(a)[0].square().sum().backward()
        f(b)[0].square().sum().backward()
        assert torch.equal(a.grad, b.grad)


def test_frequencies():
    f = S.rotary_frequencies(8, base=100.0)
    assert f.dtype == torch.float64 and torch.allclose(f, torch.tensor([1.0, 100 ** -0.25, 0.1, 100 ** -0.75], dtype=torch.float64), rtol=1e-15)
    assert torch.allclose(S.rotary_frequencies(8, base=100.0, factor=4.0), f / 4, rtol=1e-15)
    g = S.rotary_frequencies(64, factor=8.0, length=2000)
    f = S.rotary_frequencies(64)
    turns = f * 2000 / (2 * math.pi)
    assert torch.equal(g[turns > 32], f[turns > 32]) and torch.allclose(g[turns < 1], f[turns < 1] / 8, rtol=1e-15)
    assert bool(((g <= f) & (g >= f / 8 - 1e-18)).all()) and bool((g[1:] < g[:-1]).all())


@pytest.mark.parametrize("backend", backends.BACKENDS)
def test_refusals(backend):
    with backends.active(backend) as (_, dev):
        q, f = torch.zeros(2, 3, 2, 8, device=dev), S.rotary_frequencies(8, device=dev)
        w = torch.ones(8, device=dev)
        for error, call in [
            (AssertionError, lambda: S.norm_rotate(None, None, f)),
            (AssertionError, lambda: S.norm_rotate(q[0], None, f)),
            (AssertionError, lambda: S.norm_rotate(q, q[:, :2], f)),
            (AssertionError, lambda: S.norm_rotate(q, q[..., :6], f)),
            (RuntimeError, lambda: S.norm_rotate(torch.zeros(1, 1, 1, 129, device=dev))),
            (AssertionError, lambda: S.norm_rotate(q[..., :0])),
            (AssertionError, lambda: S.norm_rotate(q[..., :6], None, f)),
            (AssertionError, lambda: S.norm_rotate(q, None, f[None])),
            (TypeError, lambda: S.norm_rotate(q, None, f.float())),
            (TypeError, lambda: S.norm_rotate(q.half(), None, f)),
            (TypeError, lambda: S.norm_rotate(q.bfloat16(), q, f)),
            (TypeError, lambda: S.norm_rotate(q, None, f, w.bfloat16(), eps=1e-6)),
            (AssertionError, lambda: S.norm_rotate(q, None, f, w)),
            (AssertionError, lambda: S.norm_rotate(q, None, f, w[:7], eps=1e-6)),
            (AssertionError, lambda: S.norm_rotate(q, None, f, eps=-1e-6)),
            (AssertionError, lambda: S.norm_rotate(q, None, f, eps=math.nan)),
            (AssertionError, lambda: S.norm_rotate(q, None, f, magnitude=math.inf)),
            (AssertionError, lambda: S.norm_rotate(q, None, f, positions=1 << 31)),
            (TypeError, lambda: S.norm_rotate(q, None, f, positions=torch.zeros(2, device=dev))),
            (TypeError, lambda: S.norm_rotate(q, None, f, positions=torch.zeros(2, dtype=torch.int64, device=dev))),
            (AssertionError, lambda: S.norm_rotate(q, None, f, positions=torch.zeros(3, dtype=torch.int32, device=dev))),
            (AssertionError, lambda: S.norm_rotate(q, None, f, positions=torch.zeros(2, 2, dtype=torch.int32, device=dev))),
        ]:
            with pytest.raises(error):
                call()
