"""``fuse`` on the network over sequences: the spherical layers in the fused kernels, the blocks as they are."""
import pytest
import torch

import backends
import s2cnn_b200 as S


@pytest.mark.parametrize("backend", backends.BACKENDS)
@pytest.mark.parametrize("with_lengths", [True, False])
def test_fused_network_over_sequences(backend, with_lengths):
    """Answers and gradients of the fused network are the plain one's up to the order of float32 sums (2e-5: a few hundred units in
    the last place over the network's sums)."""
    with backends.active(backend) as (_, dev):
        torch.manual_seed(60)
        m = S.models.SphereSequenceNet(f1=2, f2=8, f_output=3, b_in=4, b_l1=3, b_l2=2, heads=2, num_buckets=8, reach=3, p=0.2).to(dev)
        fused = S.fuse(m)
        kinds = [n.target for n in fused.graph.nodes if n.op == "call_module"]
        assert {"conv1", "conv2", "blocks.0", "blocks.1"} <= set(kinds)
        by_name = {n.target: n.kwargs for n in fused.graph.nodes if n.op == "call_module"}
        assert by_name["conv1"].get("relu_so3_fft") and by_name["conv2"].get("relu_integrate")
        for train in (False, True):
            m.train(train)
            fused.train(train)
            # (another batch, another length than any that was traced)
            for batch, n in ((2, 5), (3, 4)):
                x = torch.randn(batch, n, 1, 8, 8, device=dev)
                lengths = (torch.tensor([n] + [2] * (batch - 1), dtype=torch.int32, device=dev),) if with_lengths else ()
                results = []
                for net in (m, fused):
                    m.zero_grad()
                    torch.manual_seed(61)
                    y = net(x, *lengths)
                    y.square().sum().backward()
                    results.append([y.detach()] + [p.grad.clone() for p in m.parameters()])
                for a, b in zip(*results):
                    assert (a - b).norm() <= 2e-5 * a.norm().clamp_min(1e-6)


@pytest.mark.parametrize("backend", backends.BACKENDS)
def test_own_functions_in_a_fused_model(backend):
    """The functions and modules on sequences in a model of a user's own."""
    class Net(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.norm, self.drop = S.LayerNorm(12), S.Dropout(0.3)
            self.bias = S.RelativeBias(2, 8, 4)

        def forward(self, x):
            y = S.layer_norm(self.norm(x), eps=1e-3).unflatten(-1, (2, 6))
            a = S.attention(y, y, y, self.bias.weight, self.bias.buckets, causal=True).flatten(2)
            return self.drop(S.dropout(a, 0.25, 7, residual=x), residual=a)

    with backends.active(backend) as (_, dev):
        m = Net().to(dev)
        fused = S.fuse(m)
        x = torch.randn(2, 9, 12, device=dev)
        for train in (False, True):
            m.train(train)
            fused.train(train)
            torch.manual_seed(62)
            want = m(x)
            torch.manual_seed(62)
            assert torch.equal(fused(x), want)
