"""SequenceBlock and SphereSequenceNet with their matrix products and attention in bfloat16: under autocast, and with the blocks'
parameters in bfloat16 behind the float32 spherical layers.

Tolerance: a block's output is its input plus what attention and the linear layers add; each of the some ten roundings to bfloat16 on
the way (2^-9 at most each) enters the sum with a factor below one: 1.6e-2 is eight of them at their largest, all of one sign."""
import pytest
import torch

import backends
import s2cnn_b200 as S

F32, BF16 = torch.float32, torch.bfloat16
TOL = 1.6e-2


def gradients(module, y):
    module.zero_grad()
    (y.float() * torch.linspace(-1, 1, y.numel(), device=y.device).view(y.shape)).sum().backward()
    return [p.grad for p in module.parameters()]


def near(a, b, tol=TOL):
    return (a.double() - b.double()).norm() <= tol * b.double().norm()


@pytest.mark.parametrize("backend", backends.BACKENDS)
def test_block_under_autocast_and_in_bfloat16(backend):
    with backends.active(backend) as (_, dev):
        torch.manual_seed(50)
        m = S.SequenceBlock(32, 4, kv_heads=2, causal=True, p=0.0, num_buckets=8, reach=6).to(dev)
        with torch.no_grad():
            m.bias.weight.normal_()
        x = torch.randn(2, 70, 32, device=dev)
        want = m(x)
        wanted = gradients(m, want)
        with torch.autocast(dev.type, dtype=BF16):
            cast = m(x)
            short = m(x.to(BF16))
        assert cast.dtype == F32 and near(cast, want) and short.dtype == BF16 and near(short, want)
        for p, g, w in zip(m.parameters(), gradients(m, cast), wanted):
            assert g.dtype == F32 and near(g, w, 8 * TOL)          # (sums over rows of terms that nearly cancel)
        half = S.SequenceBlock(32, 4, kv_heads=2, causal=True, p=0.0, num_buckets=8, reach=6).to(dev)
        half.load_state_dict(m.state_dict())
        half.to(BF16)
        assert near(half(x), want) and half(x).dtype == F32        # what goes around the block stays float32
        assert near(half(x.to(BF16)), want) and half(x.to(BF16)).dtype == BF16
        with torch.no_grad(), torch.autocast(dev.type, dtype=BF16):
            keys, values = (torch.zeros(2, 80, 2, 8, dtype=BF16, device=dev) for _ in range(2))
            filled = torch.zeros(2, dtype=torch.int32, device=dev)
            parts = []
            for n in (66, 1, 3):
                parts.append(m.step(x[:, int(filled[0]):int(filled[0]) + n], keys, values, filled))
                filled = filled + n
        assert near(torch.cat(parts, 1), want)


@pytest.mark.parametrize("backend", backends.BACKENDS)
def test_network_with_bfloat16_blocks(backend):
    with backends.active(backend) as (_, dev):
        torch.manual_seed(51)
        m = S.models.SphereSequenceNet(f1=2, f2=16, f_output=3, b_in=4, b_l1=3, b_l2=2, heads=2, num_buckets=8, reach=3, p=0.1).to(dev).eval()
        x = torch.randn(2, 5, 1, 8, 8, device=dev)
        lengths = torch.tensor([5, 3], dtype=torch.int32, device=dev)
        with torch.no_grad():
            want = m(x, lengths)
            with torch.autocast(dev.type, dtype=BF16):
                assert near(m(x, lengths), want)
            m.blocks.to(BF16)
            y = m(x, lengths)
            assert y.dtype == F32 and near(y, want)
        m.train()
        m(x, lengths).square().sum().backward()
        for name, p in m.named_parameters():
            assert p.grad is not None and p.grad.dtype == p.dtype and bool(torch.isfinite(p.grad).all()), name


@pytest.mark.parametrize("backend", backends.BACKENDS)
def test_other_types_are_refused(backend):
    with backends.active(backend) as (_, dev):
        for m in (S.LayerNorm(32).to(dev), S.SequenceBlock(32, 4).to(dev)):
            for dtype in (torch.float16, torch.float64, torch.int32):
                with pytest.raises(TypeError):
                    m(torch.ones(2, 5, 32, dtype=dtype, device=dev))
