"""What lies in padded signals and at positions that nobody looks at reaches no answer and no gradient, whatever it is."""
import math

import pytest
import torch

import backends
import s2cnn_b200 as S

F32, BF16 = torch.float32, torch.bfloat16


@pytest.mark.parametrize("backend", backends.BACKENDS)
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_padded_signals_change_no_answer_and_no_gradient(backend, value):
    with backends.active(backend) as (_, dev):
        torch.manual_seed(30)
        m = S.models.SphereSequenceNet(f1=2, f2=8, f_output=3, b_in=4, b_l1=3, b_l2=2, heads=2, num_buckets=8, reach=3).to(dev).eval()
        x = torch.randn(3, 5, 1, 8, 8, device=dev)
        lengths = torch.tensor([5, 3, 0], dtype=torch.int32, device=dev)
        results = []
        for fill in (1.0, value):
            x[1, 3:] = fill
            x[2] = fill
            m.zero_grad()
            leaf = x.clone().requires_grad_(True)
            y = m(leaf, lengths)
            y.square().sum().backward()
            assert not leaf.grad[1, 3:].any() and not leaf.grad[2].any()
            results.append([y.detach(), leaf.grad] + [p.grad.clone() for p in m.parameters()])
        for a, b in zip(*results):
            assert bool(torch.isfinite(b).all()) and torch.equal(a, b)
