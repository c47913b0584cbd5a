"""Attention at the lines of its rules: what a query sees that is no number, a reach beside which tables or tiles no longer fit, a
few rows more than the kernel of few rows takes, and calls that are recorded by a tracer or refused in forward mode."""
import math

import pytest
import torch
import torch.autograd.forward_ad as fwd

import backends
import s2cnn_b200 as S
from test_sequence_ops import check_attention

F32, BF16 = torch.float32, torch.bfloat16


@pytest.mark.parametrize("backend", backends.BACKENDS)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lq,dim", [(3, 24), (20, 24), (130, 24), (130, 100)])
def test_an_infinity_that_is_seen_stays_in_its_column(backend, dtype, lq, dim):
    """A value that is no number makes its column of every output that sees it infinite or NaN, and changes no other column."""
    with backends.active(backend) as (_, dev):
        gen = torch.Generator().manual_seed(80)
        q, k, v = (torch.randn(1, n, 2, dim, generator=gen).to(dtype).to(dev) for n in (lq, 140, 140))
        want = S.attention(q, k, v)
        for bad in (math.inf, -math.inf, math.nan):
            w = v.clone()
            w[0, 77, 1, 5] = bad
            out = S.attention(q, k, w)
            assert not torch.isfinite(out[0, :, 1, 5]).any()
            out[0, :, 1, 5] = want[0, :, 1, 5]
            assert torch.equal(out, want)


WIDE_REACH = [
    # B, Lq, Lk, H, Hk, D, bias, kw
    (1, 200, 200, 2, 2, 128, (32, 2048), {}),                                         # two tables and the tiles of the gradients
    (1, 200, 200, 2, 1, 64, (32, 2048), {"causal": True}),
    (1, 1, 900, 16, 1, 128, (32, 256), {}),                                           # tables of sixteen heads
    (1, 2, 900, 8, 1, 100, (32, 512), {"causal": True, "q_start": 898}),
    (1, 8, 700, 2, 1, 128, (32, 1700), {}),
    (1, 1, 900, 16, 1, 128, (32, 1000), {}),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("case", WIDE_REACH, ids=lambda c: "x".join(map(str, c[:6])))
def test_wide_reach(case, dtype):
    B, Lq, Lk, H, Hk, D, bias, kw = case
    check_attention("cuda", dtype, B, Lq, Lk, H, Hk, D, bias, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [(16, 1), (4, 4), (17, 1), (5, 4), (16, 4), (64, 1)], ids=str)
def test_a_chunk_of_new_positions_over_kept_keys(dtype, rows):
    """Queries times heads per key head of 16, 17 and more over thousands of keys of different lengths."""
    lq, group = rows
    check_attention("cuda", dtype, 2, lq, 3000, 2 * group, 2, 64, (32, 128), causal=True, q_start=[3000 - lq, 700], kv_lengths=[3000, 700 + lq])


def calls(dev):
    gen = torch.Generator().manual_seed(81)
    k, table = torch.randn(1, 30, 2, 8, generator=gen).to(dev), torch.randn(8, 2, generator=gen).to(dev)
    w, buckets = torch.randn(8, generator=gen).to(dev), S.relative_buckets(8, 4, device=dev)
    numbers = torch.tensor([5, 6], device=dev)
    return {"attention": lambda x: S.attention(x, k, k, table, buckets, causal=True), "norm": lambda x: S.layer_norm(x, w),
            "dropout": lambda x: S.dropout(x, 0.3, 5, 6, residual=x), "dropout by numbers": lambda x: S.dropout(x, 0.3, numbers)}


@pytest.mark.parametrize("backend", backends.BACKENDS)
@pytest.mark.filterwarnings("ignore")
def test_traced_calls_give_the_eager_values_and_gradients(backend):
    with backends.active(backend) as (_, dev):
        for name, f in calls(dev).items():
            x, y = (torch.randn(1, 30, 2, 8, generator=torch.Generator().manual_seed(n)).to(dev) for n in (82, 83))
            traced = torch.jit.trace(f, x.clone().requires_grad_(True), check_trace=False)
            assert torch.equal(traced(y), f(y)), name
            a, b = y.clone().requires_grad_(True), y.clone().requires_grad_(True)
            traced(a).square().sum().backward()
            f(b).square().sum().backward()
            assert torch.equal(a.grad, b.grad), name


@pytest.mark.parametrize("backend", backends.BACKENDS)
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(backend, grad):
    with backends.active(backend) as (_, dev):
        for name, f in calls(dev).items():
            x = torch.randn(1, 30, 2, 8, device=dev).requires_grad_(grad)
            with fwd.dual_level(), pytest.raises(NotImplementedError, match="jvp"):
                f(fwd.make_dual(x, torch.ones_like(x)))
