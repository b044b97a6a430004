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


def test_writing_to_a_saved_tensor_shows():
    """out= writes in place, as any in-place operation does: a tensor that a node saved for
    its backward pass and that is overwritten before it is an error there."""
    g = torch.Generator().manual_seed(4)
    x, w, b = leaf(g, 8, 64), leaf(g, 64, 64, scale=0.1), leaf(g, 64)
    other = torch.randn(8, 64, generator=g).to(DEV, BF)
    p = fr.pack_activation(other)
    d = [t.detach() for t in (w, b)]
    writes = {
        "linear_act": lambda t: fr.linear_act(other, *d, out=t),
        "linear_act in place": lambda t: fr.linear_act(other, *d, residual=t, out=t),
        "layer_norm": lambda t: fr.layer_norm(other, out=t),
        "layer_norm in place": lambda t: fr.layer_norm(t, out=t),
        "unpack_activation": lambda t: fr.unpack_activation(p, out=t),
    }
    for name, write in writes.items():
        h = fr.layer_norm_train(x)
        y = fr.linear_act_train(h, w, b)
        before = h._version
        with torch.no_grad():
            write(h.detach())
        assert h._version > before, name
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.float().sum().backward()
    with torch.inference_mode():  # tensors without a version are written all the same
        t = torch.zeros(8, 64, dtype=BF, device=DEV)
        assert fr.layer_norm(other, out=t) is t and (t != 0).any()
    assert fr.unpack_activation(p, out=t) is t


def test_writing_to_a_saved_tensor_shows_for_the_attention():
    g = torch.Generator().manual_seed(5)
    T, H, D = 96, 2, 64
    q, k, v = (torch.randn(T, H, D, generator=g).to(DEV, BF) for _ in range(3))
    x, w = torch.randn(T, 64, generator=g).to(DEV, BF), torch.randn(3 * H * D, 64, generator=g).to(DEV, BF)
    cos, sin = torch.ones(T, D // 2, device=DEV), torch.zeros(T, D // 2, device=DEV)
    cu = torch.tensor([0, 40, T], dtype=torch.int32, device=DEV)
    pos = torch.zeros(T, 2, dtype=torch.int32, device=DEV)
    writes = {
        "fused_rope_attention": lambda t: fr.fused_rope_attention(q, k, v, cos, sin, cu, out=t),
        "fused_rope_attention_pos": lambda t: fr.fused_rope_attention_pos(q, k, v, pos, cu, max_position=1, out=t),
        "fused_attention_rotated": lambda t: fr.fused_attention_rotated(q, k, v, cu, out=t),
        "fused_rope_attention_fp8": lambda t: fr.fused_rope_attention_fp8(q, k, v, cos, sin, cu, out=t),
    }
    for name, write in writes.items():
        t = torch.zeros(T, H, D, dtype=BF, device=DEV)
        assert write(t) is t and t._version == 1, name
    t = torch.zeros(T, 3, H, D, dtype=BF, device=DEV)
    assert fr.qkv_rope_projection(x, w, None, cos, sin, H, out=t) is t and t._version == 1
