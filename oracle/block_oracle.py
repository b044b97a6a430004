"""CPU oracle of the transformer-block operators — TEST INFRASTRUCTURE ONLY.

Plain numpy in 64 bits, from the definitions in include/frattn.h: layer norm, the
linear layer with bias, activation and residual, their gradients, and the 8-bit
checkpoint format. The reference project has none of these operators.
"""
from __future__ import annotations

import math

import numpy as np

BLOCK = 32
_erf = np.vectorize(math.erf, otypes=[np.float64])


def layer_norm(x, w, b, eps):
    x = x.astype(np.float64)
    mean = x.mean(1)
    d = x - mean[:, None]
    rstd = 1 / np.sqrt((d * d).mean(1) + eps)
    y = d * rstd[:, None]
    return (y if w is None else y * w) + (0 if b is None else b), mean, rstd


def layer_norm_bwd(dy, x, w, mean, rstd):
    h = (x - mean[:, None]) * rstd[:, None]
    g = dy if w is None else dy * w
    dx = rstd[:, None] * (g - g.mean(1, keepdims=True) - h * (g * h).mean(1, keepdims=True))
    return dx, (dy * h).sum(0), dy.sum(0)


def act(z, name):
    if name == "relu":
        return np.maximum(z, 0)
    if name == "gelu":
        return 0.5 * z * (1 + _erf(z / math.sqrt(2)))
    if name == "gelu_tanh":
        return 0.5 * z * (1 + np.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    if name == "silu":
        return z / (1 + np.exp(-z))
    return z


def act_grad(z, name):
    if name == "relu":
        return (z > 0).astype(np.float64)
    if name == "gelu":
        return 0.5 * (1 + _erf(z / math.sqrt(2))) + z * np.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = np.tanh(c * (z + 0.044715 * z ** 3))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    if name == "silu":
        s = 1 / (1 + np.exp(-z))
        return s * (1 + z * (1 - s))
    return np.ones_like(z)


def linear(x, w, b):
    return x @ w.T + (0 if b is None else b)


def linear_act_bwd(dy, x, w, z, name):
    dz = dy if name == "none" else dy * act_grad(z, name)
    return dz, dz @ w, dz.T @ x, dz.sum(0)


def pack(x):
    """(codes [T, 32 nb], scale bytes [T, nb]) of x [T, C]."""
    t, c = x.shape
    nb = -(-c // BLOCK)
    v = np.zeros((t, nb * BLOCK))
    v[:, :c] = x
    v = v.reshape(t, nb, BLOCK)
    bad = ~np.isfinite(v).all(-1)
    v = np.where(bad[..., None], 0, v)
    _, q = np.frexp(np.abs(v).max(-1))
    zero = np.abs(v).max(-1) == 0
    e = np.maximum(q - 7, -126)
    codes = np.clip(np.rint(np.ldexp(v, -e[..., None])), -127, 127)
    scale = np.where(bad, 255, np.where(zero, 1, e + 127))  # an all-zero block has the smallest scale
    return codes.reshape(t, -1).astype(np.int8), scale.astype(np.uint8)


def unpack(codes, scales, width):
    t, nb = scales.shape
    step = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(np.int64) - 127))
    return (codes.reshape(t, nb, BLOCK) * step[..., None]).reshape(t, -1)[:, :width]
