"""Where the masks of ``Dropout`` come from: torch's generator, call by call, so that a call repeated under activation
checkpointing draws the mask of the first one, a copy or a resumed run does as torch's own dropout does, and a captured training
step has a new mask in every replay."""
import copy

import pytest
import torch
from torch.utils.checkpoint import checkpoint

import backends
import s2cnn_b200 as S

F32, BF16 = torch.float32, torch.bfloat16


def gradients(block, x, call, dev):
    torch.manual_seed(21)
    block.zero_grad()
    x = x.clone().requires_grad_(True)
    y = call(x)
    y.square().sum().backward()
    return [y.detach(), x.grad] + [p.grad.clone() for p in block.parameters()]


@pytest.mark.parametrize("backend", backends.BACKENDS)
@pytest.mark.parametrize("reentrant", [True, False])
def test_checkpointed_block_has_the_gradients_of_the_plain_one(backend, reentrant):
    """The second call, in the backward pass, computes what the first one did: the same kernels on the same inputs, equal to the
    last bit but for what torch's matrix products may do; 1e-6 is a few units in the last place, another mask is off by 0.1."""
    with backends.active(backend) as (_, dev):
        torch.manual_seed(20)
        block = S.SequenceBlock(24, 4, p=0.3, num_buckets=8, reach=6).to(dev).train()
        x = torch.randn(2, 9, 24, device=dev)
        plain = gradients(block, x, block, dev)
        again = gradients(block, x, lambda t: checkpoint(block, t, use_reentrant=reentrant), dev)
        for a, b in zip(plain, again):
            assert (a - b).norm() <= 1e-6 * a.norm()


@pytest.mark.parametrize("backend", backends.BACKENDS)
def test_masks_follow_the_state_of_the_generator(backend):
    with backends.active(backend) as (_, dev):
        x = torch.ones(4, 300, device=dev)
        m = S.Dropout(0.5).train()
        other = copy.deepcopy(m)
        get = torch.cuda.get_rng_state if dev.type == "cuda" else torch.get_rng_state
        put = torch.cuda.set_rng_state if dev.type == "cuda" else torch.set_rng_state
        state = get()
        masks = [m(x), other(x), m(x)]
        assert not any(torch.equal(a, b) for a, b in ((masks[0], masks[1]), (masks[1], masks[2]), (masks[0], masks[2])))
        put(state)                                   # what a resumed run does
        fresh = S.Dropout(0.5).train()
        assert all(torch.equal(fresh(x), a) for a in masks)


@pytest.mark.parametrize("backend", backends.BACKENDS)
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_seed_and_step_in_memory(backend, dtype):
    """An int64 tensor of seed and step gives what the two numbers give, forward and backward."""
    with backends.active(backend) as (_, dev):
        x, g = torch.randn(3, 41).to(dtype).to(dev), torch.randn(3, 41).to(dtype).to(dev)
        seed, step = 2 ** 62 + 12345, 2 ** 40 + 7
        results = []
        for numbers in ((seed, step), (torch.tensor([seed, step], device=dev),)):
            leaf = x.clone().requires_grad_(True)
            y = S.dropout(leaf, 0.3, *numbers, residual=x)
            results.append((y, torch.autograd.grad(y, leaf, g)[0]))
        assert all(torch.equal(a, b) for a, b in zip(*results))
        for bad in (torch.tensor([1], device=dev), torch.tensor([[1, 2]], device=dev), torch.tensor([1, 2, 3, 4], device=dev)[::2]):
            with pytest.raises(AssertionError):
                S.dropout(x, 0.3, bad)
        with pytest.raises(TypeError):
            S.dropout(x, 0.3, torch.tensor([1, 2], dtype=torch.int32, device=dev))
        with pytest.raises(AssertionError):          # the step is the tensor's second number
            S.dropout(x, 0.3, torch.tensor([1, 2], device=dev), 5)
        if dev.type == "cuda":
            with pytest.raises(TypeError):
                S.dropout(x, 0.3, torch.tensor([1, 2]))


@pytest.mark.gpu
def test_replays_of_a_captured_training_step_differ():
    """The mask is drawn on the device: every replay has a new one, the same forward and backward."""
    m = S.Dropout(0.5).train()
    x = torch.ones(4, 300, device="cuda", requires_grad=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(m(x).sum(), x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = m(x)
        g, = torch.autograd.grad(y.sum(), x)
    seen = []
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, g)                     # 0 or 2, both
        seen.append(y.detach().clone())
    assert not torch.equal(seen[0], seen[1]) and not torch.equal(seen[1], seen[2])
