"""Attention at the lines of its rules: what a query sees that is no number."""
import math

import pytest
import torch

import backends
import s2cnn_b200 as S

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
