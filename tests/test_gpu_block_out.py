"""Outputs that the caller provides, on the GPU: in place and beside their inputs in one
buffer the same bits as into a new tensor, refused where they share memory."""
import pytest
import torch

import fused_rope_attn_b200 as fr
from fused_rope_attn_b200 import last_status

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
BF, HF, FF = torch.bfloat16, torch.float16, torch.float32


def randn(g, *shape, dtype=BF, scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).to(DEV, dtype)


@pytest.mark.parametrize("T,C,dt", [(1, 64, BF), (300, 1281, HF), (900, 1280, BF), (700, 333, FF), (1500, 100, BF),
                                    (5, 9000, BF), (400, 8200, HF)])
def test_layer_norm_in_place(T, C, dt):
    """Each kernel reads a row before it writes it (few rows, many, wider than 8192)."""
    g = torch.Generator().manual_seed(T)
    x, w, b = randn(g, T, C, dtype=dt), randn(g, C, dtype=dt), randn(g, C, dtype=dt)
    ref = fr.layer_norm(x, w, b)
    assert torch.equal(fr.layer_norm(x, w, b, out=x), ref)
    both = torch.zeros(T, 2 * C + 3, dtype=dt, device=DEV)  # input and output as columns of one buffer
    both[:, C:2 * C] = randn(torch.Generator().manual_seed(1), T, C, dtype=dt)
    ref = fr.layer_norm(both[:, C:2 * C].contiguous(), w, b).float()
    got = fr.layer_norm(both[:, C:2 * C], w, b, out=both[:, :C]).float()
    assert (got - ref).abs().max() <= 2.0 ** -5 * max(1.0, float(ref.abs().max()) / 8)  # vectors of another width


def test_linear_act_beside_its_inputs_in_one_buffer():
    g = torch.Generator().manual_seed(0)
    w, b = randn(g, 64, 96, scale=0.1), randn(g, 64)
    buf = torch.zeros(300, 96 + 64 + 64, dtype=BF, device=DEV)
    buf[:] = randn(g, 300, 224)
    x, r, out = buf[:, :96], buf[:, 96:160], buf[:, 160:]
    ref = fr.linear_act(x.contiguous(), w, b, activation="gelu", residual=r.contiguous())
    keep = buf[:, :160].clone()
    assert torch.equal(fr.linear_act(x, w, b, activation="gelu", residual=r, out=out), ref)
    assert torch.equal(buf[:, :160], keep)
    assert torch.equal(fr.linear_act(x, w, b, activation="gelu", residual=r, out=r), ref)


def test_refusals_of_shared_memory():
    g = torch.Generator().manual_seed(2)
    buf, w, b = randn(g, 65, 64), randn(g, 64, 64), randn(g, 64)
    x, low = buf[:64], buf[1:]
    p = fr.pack_activation(x)
    before = buf.clone()
    bad = [
        lambda: fr.linear_act(x, w, b, out=x), lambda: fr.linear_act(x, w, b, out=low), lambda: fr.linear_act(w, x, b, out=x),
        lambda: fr.linear_act(w, w, buf[3], out=x), lambda: fr.linear_act(w, w, b, residual=low, out=x),
        lambda: fr.layer_norm(x, out=low), lambda: fr.layer_norm(w, buf[2], b, out=x),
        lambda: fr.layer_norm(w, b, buf[2], out=x),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            print("accepted:", i)
    # a checkpoint of 32 rows of 16 values unpacked over the 4096 bytes that hold its codes
    codes = p.codes.view(-1)
    small = fr.PackedActivation(codes[:1024].view(32, 32), p.scales.view(-1)[:32].view(32, 1), 16, FF)
    with pytest.raises(ValueError, match="share memory with codes"):
        fr.unpack_activation(small, out=codes[:2048].view(FF).view(32, 16))
    assert torch.equal(buf, before)
    assert last_status(DEV) == 0
