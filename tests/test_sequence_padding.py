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


@pytest.mark.parametrize("backend", backends.BACKENDS)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lq", [2, 70])
def test_a_query_that_sees_nothing_gives_zero_beside_others(backend, dtype, lq):
    """Where other queries of the block see an infinity or a NaN, one that sees no key still gives 0, and no gradient of its own."""
    with backends.active(backend) as (_, dev):
        gen = torch.Generator().manual_seed(31)
        q, k, v, g = (torch.randn(2, n, 2, 24, generator=gen).to(dtype).to(dev) for n in (lq, 200, 200, lq))
        k[:, 0, :, 3], v[:, 0, :, 5], v[:, 0, :, 6] = math.nan, math.inf, math.nan
        ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
        for kw, seen in (({"q_lengths": ints(1, 0)}, [1, 0]), ({"causal": True, "q_start": ints(1 - lq, -lq)}, [-1, 0])):
            args = [t.clone().requires_grad_(True) for t in (q, k, v)]
            out = S.attention(*args, **kw)
            dq, = torch.autograd.grad(out, args[:1], g)
            for b in range(2):
                rest = slice(seen[b], None) if seen[b] >= 0 else slice(0, seen[b])
                assert not out[b, rest].any() and not dq[b, rest].any()
                assert not seen[b] or bool(torch.isnan(out[b, 0 if seen[b] > 0 else -1, :, 6]).all())
