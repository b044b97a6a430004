"""Activations of the linear layer where their result is small or their argument large.

z reaches the epilogue exactly: K = 1 and x = 1, so z is the weight itself. An output is
rounded once (u = 2^-8 bf16, 2^-11 fp16 with spacing 2^-24 near zero).

silu and gelu_tanh are z times a sigmoid 1 / (1 + 2^v). In front of the rounding the
factor is off by what rounds v: |v| <= 60 in 32 bits with four roundings and constants
of 24 bits, 60 x 6 x 2^-24 ln 2 < 2^-15 of itself, and by ex2, rcp and the sum, some 2^-22
each: 2^-14 of the result is asked for. Where the sigmoid is below 2^-58 the result counts as zero: below
41 x 2^-59 or 7.4 x 2^-58 in magnitude, so 2^-52 absolute is allowed besides.
"""
import math

import numpy as np
import pytest
import torch

import fused_rope_attn_b200 as fr
from fused_rope_attn_b200 import last_status
from oracle import block_oracle as B

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
BF, HF = torch.bfloat16, torch.float16
U = {BF: 2.0 ** -8, HF: 2.0 ** -11}
TINY = {BF: 2.0 ** -134, HF: 2.0 ** -25}  # half the spacing of the subnormals


def forward(z, act, T=1):
    x = torch.ones(T, 1, dtype=z.dtype, device=DEV)
    y = fr.linear_act(x, z.view(-1, 1).to(DEV), activation=act)
    assert last_status(DEV) == 0
    return y


def formula(z, act):
    """In 64 bits and without the cancellation of 1 + tanh for negative z."""
    with np.errstate(over="ignore"):
        if act == "gelu_tanh":
            return z / (1 + np.exp(-2 * np.sqrt(2 / np.pi) * (z + 0.044715 * z ** 3)))
        return B.act(z, act)


def check(y, z, act, rel, floor):
    zz = z.double().numpy()
    ref = formula(zz, act)
    got = y.double().cpu().numpy()
    assert np.isfinite(got).all()
    over = np.abs(got - ref) - (1.01 * U[z.dtype] * np.abs(ref) + TINY[z.dtype] + rel * np.abs(ref) + floor)
    at = np.unravel_index(over.argmax(), over.shape)[-1]
    assert (over <= 0).all(), f"{act}({zz[at]:.4g}): worst excess {over.max():.3e}"


@pytest.mark.parametrize("T", [1, 9000])
@pytest.mark.parametrize("act", ["gelu_tanh", "silu"])
@pytest.mark.parametrize("dt", [BF, HF])
def test_sigmoid_activations_to_the_ends_of_the_type(dt, act, T):
    """Down to the largest negative value the result is zero, not a fraction of z."""
    mag = torch.logspace(-6, float(np.log10(torch.finfo(dt).max)) - 1e-3, 800, dtype=torch.float64)
    edge = torch.tensor([7.3, 7.4, 7.5, 8.0, 40.0, 41.0, 41.5, 42.0, 60.0, 88.0, 89.0, 104.0], dtype=torch.float64)
    z = torch.cat([-mag, -edge, edge, mag]).to(dt)
    z = torch.cat([z, torch.tensor([torch.finfo(dt).min, torch.finfo(dt).max], dtype=dt)])
    y = forward(z, act, T)
    for row in (0, T - 1):
        check(y[row], z, act, 2.0 ** -14, 2.0 ** -52)
    assert (y[0].cpu()[z < -1e3] == 0).all()


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
def test_an_infinite_argument_shows(act):
    """z times a factor that is 0 at minus infinity: NaN, as in the formula's own arithmetic."""
    z = torch.tensor([-float("inf"), float("inf"), float("nan"), 1.0, -1.0, 0.0], dtype=BF)
    y = forward(z, act)[0].cpu()
    assert torch.isnan(y[0]) and y[1] == float("inf") and torch.isnan(y[2]) and torch.isfinite(y[3:]).all()


@pytest.mark.parametrize("T", [1, 9000])
@pytest.mark.parametrize("dt", [BF, HF])
def test_gelu_of_negative_values(dt, T):
    """In the negative tail gelu is z times the small distribution function itself: within
    2^-14 of itself before the rounding. That is the polynomial's 2^-14.8 and what rounds the
    exponent, |z^2 / (2 ln 2)| <= 122 in 32 bits: 122 x 2.5 x 2^-24 ln 2 = 2^-16.2."""
    z = -torch.cat([torch.logspace(-3, 0, 100), torch.linspace(1, 13, 1200)]).double().to(dt)
    y = forward(z, "gelu", T)
    zz = z.double().numpy()
    cdf = np.array([0.5 * math.erfc(-v / math.sqrt(2)) for v in zz])
    for row in (0, T - 1):
        got = y[row].double().cpu().numpy()
        over = np.abs(got - zz * cdf) - ((1.01 * U[dt] + 2.0 ** -14) * np.abs(zz * cdf) + TINY[dt])
        assert (over <= 0).all(), f"gelu({zz[over.argmax()]:.4g}): worst excess {over.max():.3e}"


@pytest.mark.parametrize("dt", [BF, HF])
def test_gelu_gradient_of_negative_values(dt):
    """cdf + z pdf: each term within 2^-14 of itself, as above."""
    z = -torch.cat([torch.logspace(-3, 0, 100), torch.linspace(1, 13, 1200)]).double().to(dt)
    N = z.numel()
    one = torch.ones(1, 1, dtype=dt, device=DEV)
    _, _, db = fr.linear_act_backward(torch.ones(1, N, dtype=dt, device=DEV), one, z.view(N, 1).to(DEV),
                                      z.view(1, N).to(DEV), activation="gelu")
    zz = z.double().numpy()
    cdf = np.array([0.5 * math.erfc(-v / math.sqrt(2)) for v in zz])
    zpdf = zz * np.exp(-zz * zz / 2) / math.sqrt(2 * math.pi)
    over = np.abs(db.double().cpu().numpy() - (cdf + zpdf)) - (
        1.01 * U[dt] * np.abs(cdf + zpdf) + 2.0 ** -14 * (cdf + np.abs(zpdf)) + TINY[dt])
    assert (over <= 0).all(), f"at {zz[over.argmax()]:.4g}: worst excess {over.max():.3e}"
    assert last_status(DEV) == 0
