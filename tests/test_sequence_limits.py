"""Attention at the lines of its rules: what a query sees that is no number, a reach beside which tables or tiles no longer fit, a
few rows more than the kernel of few rows takes."""
import math

import pytest
import torch

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
