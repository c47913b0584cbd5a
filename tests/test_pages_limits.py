"""Turned heads and kept keys in pages where they could go wrong: numbers at the ends of float32, memory that is not there, widths, many items.

Tolerances: as in test_norm_rotate.py and test_pages.py; what is compared without one is bits.
"""
import math

import pytest
import torch

import backends
import s2cnn_b200 as S
from test_norm_rotate import normal

F32, BF16 = torch.float32, torch.bfloat16


# ---- heads --------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("backend", backends.BACKENDS)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(24, 8, False), (24, 24, False), (40, 16, False), (80, 80, False), (128, 64, False), (20, 20, True), (44, 8, True), (25, 24, True)], ids=str)
def test_squares_that_overflow(backend, dtype, shape):
    """Where the sum of a head's squares is no float32 its inverse root is 0: the head is zeros, its gradient too, and it adds nothing to the
    weight's.  Other heads are as they were.  (1e20 is in the range of both types; its square is not.)"""
    with backends.active(backend) as (_, dev):
        D, turned, interleaved = shape
        gen = torch.Generator().manual_seed(60)
        f, w = S.rotary_frequencies(turned, device=dev), normal(gen, dev, dtype, D, scale=0.3, shift=1.0).requires_grad_(True)
        q, g = normal(gen, dev, dtype, 1, 7, 5, D), normal(gen, dev, dtype, 1, 7, 5, D)
        large, none = q.clone(), q.clone()
        for place in range(0, D, 3):
            i, h = place // 3 % 7, place // 3 % 5
            large[0, i, h, place] = 1e20
            none[0, i, h] = 0
        grads = []
        for x in (large, none):
            x.requires_grad_(True)
            y, _ = S.norm_rotate(x, None, f, w, eps=1e-6, positions=5, interleaved=interleaved)
            grads.append((y.detach(),) + torch.autograd.grad(y, (x, w), g))
        zeros = (none == 0).all(-1)
        for a, b in zip(grads[0][:2], grads[1][:2]):
            assert not a[zeros].any() and torch.equal(a[~zeros], b[~zeros])
        assert torch.equal(grads[0][2], grads[1][2])
