"""Transformer-block operators without a GPU: the oracle against differences, the
checkpoint format's properties, and the refusals of the public entry points."""
import numpy as np
import pytest
import torch

import fused_rope_attn_b200 as fr
from fused_rope_attn_b200 import _lib
from oracle import block_oracle as B

ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]


@pytest.mark.parametrize("name", ACTS)
def test_oracle_activation_gradient(name):
    z = np.linspace(-6, 6, 241) + 0.013  # off relu's corner
    h = 1e-5
    num = (B.act(z + h, name) - B.act(z - h, name)) / (2 * h)
    # central differences: h^2 f''' / 6 + rounding 2^-52 |f| / h
    assert np.abs(num - B.act_grad(z, name)).max() < 1e-9


def test_oracle_layer_norm_gradient():
    rng = np.random.default_rng(0)
    x, dy = rng.normal(size=(3, 7)), rng.normal(size=(3, 7))
    w, b = rng.normal(size=7), rng.normal(size=7)
    _, mean, rstd = B.layer_norm(x, w, b, 1e-6)
    dx, dw, db = B.layer_norm_bwd(dy, x, w, mean, rstd)
    h = 1e-6

    def loss(x, w, b):
        return (B.layer_norm(x, w, b, 1e-6)[0] * dy).sum()

    for v, g, at in ((x, dx, (1, 2)), (w, dw, (3,)), (b, db, (5,))):
        p, m = v.copy(), v.copy()
        p[at] += h
        m[at] -= h
        a = [(p if t is v else t, m if t is v else t) for t in (x, w, b)]
        num = (loss(*(t[0] for t in a)) - loss(*(t[1] for t in a))) / (2 * h)
        assert abs(num - g[at]) < 1e-7


def test_oracle_pack_error_bound():
    """Each value is off by at most half a step, one step where it is above 127 steps;
    the step is at most 2^-6 of the block's largest magnitude."""
    rng = np.random.default_rng(1)
    x = rng.normal(size=(50, 75)) * np.exp(rng.normal(size=(50, 1)) * 5)
    codes, scales = B.pack(x)
    back = B.unpack(codes, scales, 75)
    step = np.repeat(np.ldexp(1.0, scales.astype(int) - 127), 32, 1)[:, :75]
    err = np.abs(back - x)
    assert (err <= np.where(np.abs(x) > 127 * step, step, step / 2)).all()
    amax = np.abs(np.pad(x, ((0, 0), (0, 21))).reshape(50, 3, 32)).max(-1)
    assert (np.ldexp(1.0, scales.astype(int) - 127) <= amax * 2.0 ** -6).all()
    c2, s2 = B.pack(back)  # packing what a checkpoint stands for gives it again
    assert (B.unpack(c2, s2, 75) == back).all()


def _refuses(f, *words):
    with pytest.raises(ValueError) as e:
        f()
    for w in words:
        assert w in str(e.value), str(e.value)


def test_refusals_of_cpu_tensors():
    x, w = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(8, 64, dtype=torch.bfloat16)
    _refuses(lambda: fr.layer_norm(x), "x must be on CUDA")
    _refuses(lambda: fr.layer_norm_backward(x, x, None, x, x), "dout must be on CUDA")
    _refuses(lambda: fr.linear_act(x, w), "x must be on CUDA")
    _refuses(lambda: fr.linear_act_backward(x, x, w), "dout must be on CUDA")
    _refuses(lambda: fr.pack_activation(x), "x must be on CUDA")
    p = fr.PackedActivation(torch.zeros(4, 64, dtype=torch.int8), torch.zeros(4, 2, dtype=torch.uint8), 64,
                            torch.bfloat16)
    assert p.shape == (4, 64)
    _refuses(lambda: fr.unpack_activation(p), "must be on CUDA")
    _refuses(lambda: fr.unpack_activation(p._replace(width=70)), "do not hold rows of 70 values")
    _refuses(lambda: fr.unpack_activation(p._replace(codes=p.codes.float())), "must be int8")


def _norm(lib, **kw):
    a = dict(x=16, xs=64, w=16, b=16, pd=_lib.BF16, T=4, C=64, eps=1e-6, dt=_lib.BF16, out=16, os=64, mean=16,
             rstd=16)
    a.update(kw)
    return lib.frattn_layer_norm(a["x"], a["xs"], a["w"], a["b"], a["pd"], a["T"], a["C"], a["eps"], a["dt"],
                                 a["out"], a["os"], a["mean"], a["rstd"], None)


def test_layer_norm_abi_checks():
    lib = _lib.load()
    assert _norm(lib, T=0, x=None) == 0  # nothing to do
    assert _norm(lib, x=None) == _lib.E_NULL
    assert _norm(lib, C=0) == _lib.E_SHAPE
    assert _norm(lib, T=-1) == _lib.E_SHAPE
    assert _norm(lib, os=63) == _lib.E_SHAPE
    assert _norm(lib, eps=-1.0) == _lib.E_SHAPE
    assert _norm(lib, eps=float("nan")) == _lib.E_SHAPE
    assert _norm(lib, dt=7) == _lib.E_DTYPE
    assert _norm(lib, pd=_lib.F16) == _lib.E_DTYPE
    assert _norm(lib, x=17) == _lib.E_ALIGN
    assert _norm(lib, mean=18) == _lib.E_ALIGN


def _norm_bwd(lib, **kw):
    a = dict(dy=16, dys=64, x=16, xs=64, codes=None, scales=None, w=16, pd=_lib.BF16, mean=16, rstd=16, T=4, C=64,
             dt=_lib.BF16, dx=16, dxs=64, dw=16, db=16, ws=256, wsb=1 << 20)
    a.update(kw)
    return lib.frattn_layer_norm_bwd(a["dy"], a["dys"], a["x"], a["xs"], a["codes"], a["scales"], a["w"], a["pd"],
                                     a["mean"], a["rstd"], a["T"], a["C"], a["dt"], a["dx"], a["dxs"], a["dw"],
                                     a["db"], a["ws"], a["wsb"], None)


def test_layer_norm_bwd_abi_checks():
    lib = _lib.load()
    for k in ("dy", "x", "mean", "rstd", "dx", "ws"):
        assert _norm_bwd(lib, **{k: None}) == _lib.E_NULL, k
    assert _norm_bwd(lib, codes=16, scales=16) == _lib.E_NULL  # x given twice
    assert _norm_bwd(lib, x=None, codes=16) == _lib.E_NULL
    assert _norm_bwd(lib, x=None, codes=24, scales=16) == _lib.E_ALIGN
    assert _norm_bwd(lib, dxs=10) == _lib.E_SHAPE
    assert _norm_bwd(lib, wsb=16) == _lib.E_WORKSPACE
    assert _lib.workspace_bytes_layer_norm_bwd(9216, 1280) >= 148 * 2 * 1280 * 4
    with pytest.raises(ValueError):
        _lib.workspace_bytes_layer_norm_bwd(4, 0)


def _linear(lib, **kw):
    a = dict(x=16, xs=64, w=16, ws_=64, b=16, r=16, rs=32, act=2, T=4, K=64, N=32, dt=_lib.BF16, out=16, os=32,
             z=None, zs=0, zc=None, zsc=None, ws=256, wsb=1 << 40)
    a.update(kw)
    return lib.frattn_linear_act(a["x"], a["xs"], a["w"], a["ws_"], a["b"], a["r"], a["rs"], a["act"], a["T"], a["K"],
                                 a["N"], a["dt"], a["out"], a["os"], a["z"], a["zs"], a["zc"], a["zsc"], a["ws"],
                                 a["wsb"], None, None)


def test_linear_abi_checks():
    lib = _lib.load()
    assert _linear(lib, T=0) == 0
    for k in ("x", "w", "out"):
        assert _linear(lib, **{k: None}) == _lib.E_NULL, k
    for k, v in (("K", 0), ("N", -1), ("T", -1), ("xs", 56), ("ws_", 8), ("os", 31), ("act", 5), ("act", -1)):
        assert _linear(lib, **{k: v}) == _lib.E_SHAPE, k
    assert _linear(lib, dt=_lib.F32) == _lib.E_DTYPE
    for k, v in (("x", 8), ("xs", 68), ("w", 24), ("ws_", 65), ("out", 17), ("r", 17), ("b", 3)):
        assert _linear(lib, **{k: v}) == _lib.E_ALIGN, k
    assert _linear(lib, z=16, zs=32, zc=16, zsc=16) == _lib.E_NULL  # both kinds of pre-activation
    assert _linear(lib, zc=16) == _lib.E_NULL
    assert _linear(lib, zc=8, zsc=16) == _lib.E_ALIGN


def _linear_bwd(lib, **kw):
    a = dict(dy=16, dys=32, x=16, xs=64, xc=None, xsc=None, w=16, ws_=64, z=16, zs=32, zc=None, zsc=None, act=2, T=4,
             K=64, N=32, dt=_lib.BF16, dx=16, dxs=64, dw=16, db=16, ws=256, wsb=1 << 40)
    a.update(kw)
    return lib.frattn_linear_act_bwd(a["dy"], a["dys"], a["x"], a["xs"], a["xc"], a["xsc"], a["w"], a["ws_"], a["z"],
                                     a["zs"], a["zc"], a["zsc"], a["act"], a["T"], a["K"], a["N"], a["dt"], a["dx"],
                                     a["dxs"], a["dw"], a["db"], a["ws"], a["wsb"], None, None)


def test_linear_bwd_abi_checks():
    lib = _lib.load()
    for k in ("dy", "x", "w", "z", "ws"):
        assert _linear_bwd(lib, **{k: None}) == _lib.E_NULL, k
    assert _linear_bwd(lib, xc=16, xsc=16) == _lib.E_NULL
    assert _linear_bwd(lib, zc=16, zsc=16) == _lib.E_NULL
    for k, v in (("K", 0), ("dxs", 8), ("xs", 8), ("ws_", 8), ("act", 9)):
        assert _linear_bwd(lib, **{k: v}) == _lib.E_SHAPE, k
    assert _linear_bwd(lib, dt=_lib.F32) == _lib.E_DTYPE
    for k, v in (("x", 8), ("xs", 68), ("w", 24), ("dy", 17), ("z", 17), ("ws", 128)):
        assert _linear_bwd(lib, **{k: v}) == _lib.E_ALIGN, k
    assert _linear_bwd(lib, wsb=64) == _lib.E_WORKSPACE
    assert _lib.workspace_bytes_linear_act_bwd(9216, 1280, 3424) > 9216 * 3424 * 2
