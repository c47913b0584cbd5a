"""``SequenceBlock.step`` where the room for kept positions ends."""
import pytest
import torch

import backends
import s2cnn_b200 as S


@pytest.mark.parametrize("backend", backends.BACKENDS)
def test_a_sequence_without_room_gives_nan_and_disturbs_no_other(backend):
    with backends.active(backend) as (_, dev):
        torch.manual_seed(70)
        m = S.SequenceBlock(24, 4, kv_heads=2, causal=True, p=0.0, num_buckets=8, reach=6).to(dev).eval()
        with torch.no_grad():
            kept = torch.randn(4, 16, 2, 6, device=dev), torch.randn(4, 16, 2, 6, device=dev)
            x = torch.randn(4, 3, 24, device=dev)
            fits = torch.tensor([13, 4, 0, 7], dtype=torch.int32, device=dev)
            want = m.step(x, *(t.clone() for t in kept), fits)
            filled = torch.tensor([13, 14, -1, 2 ** 30], dtype=torch.int32, device=dev)        # 16 of 16; one and more too many; none
            keys, values = (t.clone() for t in kept)
            y = m.step(x, keys, values, filled)
            assert torch.equal(y[0], want[0]) and bool(torch.isnan(y[1:]).all())
            assert torch.equal(keys[0, :13], kept[0][0, :13]) and not torch.equal(keys[0, 13:], kept[0][0, 13:])
            assert torch.equal(m.step(x, keys, values, fits), want)
            with pytest.raises(AssertionError):
                m.step(torch.randn(4, 17, 24, device=dev), keys, values, fits)
