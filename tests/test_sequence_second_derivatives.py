"""Gradients of gradients: dropout is linear and has them, attention and layer norm refuse instead of leaving the term out."""
import pytest
import torch

import backends
import s2cnn_b200 as S


@pytest.mark.parametrize("backend", backends.BACKENDS)
def test_dropout_twice(backend):
    """y = m x with a fixed mask m: what goes through the first gradient is a product of the same factors."""
    with backends.active(backend) as (_, dev):
        x, w = torch.randn(5, 9, device=dev, requires_grad=True), torch.randn(5, 9, device=dev, requires_grad=True)
        r = torch.randn(5, 9, device=dev, requires_grad=True)
        for numbers in ((3, 4), (torch.tensor([3, 4], device=dev),)):
            factor = S.dropout(torch.ones_like(x), 0.4, *numbers).detach()
            y = S.dropout(x, 0.4, *numbers, residual=r)
            gx, gr = torch.autograd.grad((w * y).sum(), (x, r), create_graph=True)
            assert torch.equal(gx, factor * w)
            second, = torch.autograd.grad((gx * gx).sum() + gr.sum(), w, create_graph=True)
            assert torch.equal(second, 2 * (factor * w) * factor + 1)
            third, = torch.autograd.grad(second.sum(), w)
            assert torch.equal(third, 2 * factor * factor)


@pytest.mark.parametrize("backend", backends.BACKENDS)
def test_attention_and_layer_norm_refuse(backend):
    with backends.active(backend) as (_, dev):
        q, k, v, b = (torch.randn(*s, device=dev, requires_grad=True) for s in ((1, 5, 2, 8), (1, 5, 2, 8), (1, 5, 2, 8), (8, 2)))
        x, w = torch.randn(4, 6, device=dev, requires_grad=True), torch.randn(6, device=dev, requires_grad=True)
        buckets = S.relative_buckets(8, 4, device=dev)
        for f, leaves in ((lambda: S.attention(q, k, v, b, buckets), (q, k, v, b)), (lambda: S.attention(q, k, v), (q, k, v)),
                          (lambda: S.layer_norm(x, w), (x, w)), (lambda: S.layer_norm(x), (x,))):
            plain = torch.autograd.grad(f().square().sum(), leaves)
            grads = torch.autograd.grad(f().square().sum(), leaves, create_graph=True)
            for a, g in zip(plain, grads):
                assert torch.equal(a, g) and not a.requires_grad and g.requires_grad
                with pytest.raises(RuntimeError, match="second derivative"):
                    torch.autograd.grad(g.square().sum() + sum(t.sum() for t in leaves), leaves, retain_graph=True)
                with pytest.raises(RuntimeError, match="second derivative"):
                    (g.square().sum() + leaves[0].sum()).backward(retain_graph=True)
        # a loss beside the gradient's own graph is not held up
        y = S.layer_norm(x, w)
        g, = torch.autograd.grad(y.sum(), x, create_graph=True)
        (y.sum() + g.detach().sum()).backward()
