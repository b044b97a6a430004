"""The train nodes among other autograd operations: what they cannot give is refused, not
left out of a gradient."""
import pytest
import torch

import fused_rope_attn_b200 as fr

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
BF = torch.bfloat16


def leaf(g, *shape, scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).to(DEV, BF).requires_grad_(True)


def penalty(y, x):
    """A loss on the gradient itself: |d(sum y^2) / dx|^2."""
    (gx,) = torch.autograd.grad(y.float().square().sum(), x, create_graph=True)
    return gx.float().square().sum()


@pytest.mark.parametrize("checkpoint", [False, True])
@pytest.mark.parametrize("act", ["none", "gelu"])
def test_linear_node_refuses_a_second_derivative(act, checkpoint):
    """With a residual the gradient keeps a graph through dout, so that the missing terms
    would not show."""
    g = torch.Generator().manual_seed(0)
    x, w, b = leaf(g, 8, 64), leaf(g, 64, 64, scale=0.1), leaf(g, 64)
    y = fr.linear_act_train(x, w, b, activation=act, residual=x, checkpoint=checkpoint)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        penalty(y, x).backward()


@pytest.mark.parametrize("checkpoint", [False, True])
def test_norm_node_refuses_a_second_derivative(checkpoint):
    g = torch.Generator().manual_seed(1)
    x, w, b = leaf(g, 8, 512), leaf(g, 512), leaf(g, 512)
    y = fr.layer_norm_train(x, w, b, checkpoint=checkpoint) + x
    with pytest.raises(RuntimeError, match="once_differentiable"):
        penalty(y, x).backward()


def test_first_derivatives_with_a_graph_are_the_same():
    g = torch.Generator().manual_seed(2)
    x, w, b = leaf(g, 8, 64), leaf(g, 64, 64, scale=0.1), leaf(g, 64)
    nw, nb = leaf(g, 64), leaf(g, 64)
    y = fr.linear_act_train(fr.layer_norm_train(x, nw, nb), w, b, activation="silu", residual=x)
    ps = (x, w, b, nw, nb)
    a = torch.autograd.grad(y.float().sum(), ps, retain_graph=True)
    c = torch.autograd.grad(y.float().sum(), ps, create_graph=True)
    assert all(torch.equal(s, t) for s, t in zip(a, c))


def test_attention_node_refuses_a_second_derivative():
    g = torch.Generator().manual_seed(3)
    q, k, v = (leaf(g, 96, 2, 64) for _ in range(3))
    cos, sin = torch.ones(96, 32, device=DEV), torch.zeros(96, 32, device=DEV)
    cu = torch.tensor([0, 40, 96], dtype=torch.int32, device=DEV)
    y = fr.fused_rope_attention_train(q, k, v, cos, sin, cu) + v
    with pytest.raises(RuntimeError, match="once_differentiable"):
        penalty(y, v).backward()
