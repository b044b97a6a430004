"""Calls that follow one another without a wait between them, each on what the one before
wrote: a kernel may start before the one in front of it has ended, but reads after it."""
import pytest
import torch

import fused_rope_attn_b200 as fr
from fused_rope_attn_b200 import last_status

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
BF, FF = torch.bfloat16, torch.float32


def randn(g, *shape, dtype=BF, scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).to(DEV, dtype)


@pytest.mark.parametrize("T,K,N", [(3, 64, 100), (130, 72, 333), (40, 320, 320), (700, 512, 264), (300, 5120, 640),
                                   (2100, 640, 1285)])
def test_residual_in_place_again_and_again(T, K, N):
    """out = residual on one buffer, whose rows share lines and pieces of 16 bytes between the
    tiles of different SMs, against new tensors each time."""
    g = torch.Generator().manual_seed(N)
    xs = [randn(g, T, K) for _ in range(4)]
    w, b = randn(g, N, K, scale=K ** -0.5), [randn(g, N) for _ in range(4)]
    r0 = randn(g, T, N)
    ref = r0
    for i in range(40):
        ref = fr.linear_act(xs[i % 4], w, b[i % 4], activation="silu", residual=ref)
        torch.cuda.synchronize()
    acc = r0.clone()
    for i in range(40):
        fr.linear_act(xs[i % 4], w, b[i % 4], activation="silu", residual=acc, out=acc)
    assert torch.equal(acc, ref)
    assert last_status(DEV) == 0


@pytest.mark.parametrize("T,C,dt", [(5, 333, BF), (150, 1281, FF), (900, 1281, BF), (30, 8200, BF), (400, 9001, BF)])
def test_norm_of_its_own_output_with_parameters_just_written(T, C, dt):
    """Rows, weight and bias are all written by the calls right in front."""
    g = torch.Generator().manual_seed(C)
    x0, p0 = randn(g, T, C, dtype=dt), randn(g, 2, C, dtype=dt)

    def chain(wait):
        x, p = x0.clone(), p0.clone()
        for _ in range(12):
            fr.layer_norm(p, out=p)
            if wait:
                torch.cuda.synchronize()
            fr.layer_norm(x, p[0], p[1], out=x)
            if wait:
                torch.cuda.synchronize()
            m = torch.zeros(T, device=DEV)
            x, dw, db = fr.layer_norm_backward(x, x, p[0], m, m + 1)
            p = torch.stack((dw, db))
            if wait:
                torch.cuda.synchronize()
        return x, p

    a, c = chain(False), chain(True)
    assert all(torch.equal(s, t) for s, t in zip(a, c)) and torch.isfinite(a[0]).all()
