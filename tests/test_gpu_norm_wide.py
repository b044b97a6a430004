"""Layer norm where one row takes most of a block: teams of five to eight warps, fewer blocks
to an SM than the registers would allow, and more rows than run at once.

Tolerances as for the other widths: u is one rounding of the output (2^-8 bf16, 2^-11 fp16
with spacing 2^-24 near zero, 2^-24 fp32), a sum of n terms in 32 bits is off by at most
n 2^-23 of the sum of their magnitudes."""
import numpy as np
import pytest
import torch

import fused_rope_attn_b200 as fr
from oracle import block_oracle as B

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
BF, HF, FF = torch.bfloat16, torch.float16, torch.float32
U = {BF: 2.0 ** -8, HF: 2.0 ** -11, FF: 2.0 ** -24}
TINY = {BF: 0.0, HF: 2.0 ** -25, FF: 0.0}


def f64(t):
    return t.detach().double().cpu().numpy()


def near(got, ref, dtype, slack):
    g = f64(got)
    assert got.dtype == dtype and g.shape == ref.shape
    over = np.abs(g - ref) - (1.01 * U[dtype] * (np.abs(ref) + slack) + TINY[dtype] + slack)
    assert np.isfinite(g).all() and (over <= 0).all(), f"worst excess {over.max():.3e} at {np.unravel_index(over.argmax(), over.shape)}"


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("T,C,dt", [
    (593, 5376, BF), (2000, 5121, HF), (1500, 6400, BF), (593, 7680, HF), (900, 8192, BF), (1801, 8192, BF), (593, 8191, BF),
    (593, 4608, FF), (900, 4101, FF), (593, 8192, FF), (1200, 6401, FF),
])
def test_rows_of_a_block_each(T, C, dt, packed):
    g = torch.Generator().manual_seed(C)
    x = (torch.randn(T, C, generator=g) * torch.exp(0.5 * torch.randn(C, generator=g))
         + 3 * torch.randn(T, 1, generator=g)).to(dt)
    w, b = 1 + 0.2 * torch.randn(C, generator=g), 0.3 * torch.randn(C, generator=g)
    dy = torch.randn(T, C, generator=g).to(dt)
    y, mean, rstd = fr.layer_norm(x.to(DEV), w.to(DEV), b.to(DEV), return_stats=True)
    ry, rm, rr = B.layer_norm(f64(x), f64(w), f64(b), 1e-6)
    eps = (C + 16) * 2.0 ** -23
    ax = np.abs(f64(x))
    near(y, ry, dt, eps * (ax + ax.mean(1, keepdims=True)) * rr[:, None] * np.abs(f64(w)) + 2.0 ** -22 * np.abs(f64(b)))
    arg, xv = x.to(DEV), f64(x)
    if packed:
        arg = fr.pack_activation(arg)
        xv = B.unpack(arg.codes.cpu().numpy(), arg.scales.cpu().numpy(), C)
    m, r = f64(mean), f64(rstd)
    dx, dw, db = fr.layer_norm_backward(dy.to(DEV), arg, w.to(DEV), mean, rstd)
    rx, rw, rb = B.layer_norm_bwd(f64(dy), xv, f64(w), m, r)
    h = (np.abs(xv) + np.abs(m)[:, None]) * r[:, None]
    gw = np.abs(f64(dy) * f64(w))
    near(dx, rx, dt, eps * r[:, None] * (gw + gw.mean(1, keepdims=True) + h * (gw * h).mean(1, keepdims=True)))
    near(dw, rw, FF, (T + 8) * 2.0 ** -23 * (np.abs(f64(dy)) * h).sum(0))
    near(db, rb, FF, (T + 8) * 2.0 ** -23 * np.abs(f64(dy)).sum(0))


@pytest.mark.parametrize("packed", [False, True])
def test_more_rows_than_blocks_above_8192_columns(packed):
    T, C = 700, 8200
    g = torch.Generator().manual_seed(0)
    x, dy = (torch.randn(T, C, generator=g) + 1).to(BF), torch.randn(T, C, generator=g).to(BF)
    w, b = 1 + 0.2 * torch.randn(C, generator=g), 0.3 * torch.randn(C, generator=g)
    y, mean, rstd = fr.layer_norm(x.to(DEV), w.to(DEV), b.to(DEV), return_stats=True)
    ry, rm, rr = B.layer_norm(f64(x), f64(w), f64(b), 1e-6)
    eps = (C + 16) * 2.0 ** -23
    ax = np.abs(f64(x))
    near(y, ry, BF, eps * (ax + ax.mean(1, keepdims=True)) * rr[:, None] * np.abs(f64(w)) + 2.0 ** -22 * np.abs(f64(b)))
    arg, xv = x.to(DEV), f64(x)
    if packed:
        arg = fr.pack_activation(arg)
        xv = B.unpack(arg.codes.cpu().numpy(), arg.scales.cpu().numpy(), C)
    m, r = f64(mean), f64(rstd)
    dx, dw, db = fr.layer_norm_backward(dy.to(DEV), arg, w.to(DEV), mean, rstd)
    rx, rw, rb = B.layer_norm_bwd(f64(dy), xv, f64(w), m, r)
    h = (np.abs(xv) + np.abs(m)[:, None]) * r[:, None]
    gw = np.abs(f64(dy) * f64(w))
    near(dx, rx, BF, eps * r[:, None] * (gw + gw.mean(1, keepdims=True) + h * (gw * h).mean(1, keepdims=True)))
    near(dw, rw, FF, (T + 8) * 2.0 ** -23 * (np.abs(f64(dy)) * h).sum(0))
    near(db, rb, FF, (T + 8) * 2.0 ** -23 * np.abs(f64(dy)).sum(0))
