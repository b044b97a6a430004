"""Transformer-block operators on the GPU against the 64-bit oracle.

Tolerances. u is the unit roundoff of the output's type: half a unit in the last place
relative to the value, at most 2^-p for p significant bits (2^-8 bf16, 2^-11 fp16 with
its spacing near zero, 2^-24 fp32). A sum of n fp32
terms is off by at most n 2^-23 of the sum of their magnitudes, whatever its order
(2^-23, not 2^-24: the tensor core may truncate); activations have slopes of at most
1.13 and their own error is below 2^-20 of |z|. dz is rounded to the 16-bit type
before the two products of the backward pass, which adds u of the sum of magnitudes
at the worst. In the 2-norm a rounding is off by 0.42 u on average (its error is uniform
within half a unit, the mantissas spread over a factor of two) and errors are independent:
two of them stay below 0.6 u, and u is asked for.
"""
import numpy as np
import pytest
import torch

import fused_rope_attn_b200 as fr
from fused_rope_attn_b200 import last_status
from oracle import block_oracle as B

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}
BF, HF, FF = torch.bfloat16, torch.float16, torch.float32
ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]


def f64(t):
    return t.detach().double().cpu().numpy()


def near(got, ref, dtype, slack):
    """|got - ref| <= one rounding to dtype + slack (elementwise or a number)."""
    g = f64(got)
    assert got.dtype == dtype and g.shape == ref.shape
    over = np.abs(g - ref) - (1.01 * U[dtype] * (np.abs(ref) + slack) + TINY[dtype] + slack)
    assert np.isfinite(g).all() and (over <= 0).all(), f"worst excess {over.max():.3e} at {np.unravel_index(over.argmax(), over.shape)}"


def rel(got, ref):
    return np.linalg.norm(f64(got) - ref) / max(np.linalg.norm(ref), 1e-300)


def randn(g, *shape, dtype=FF, scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def wide_rows(t, extra):
    """t on the GPU as rows of a wider buffer."""
    big = torch.zeros(t.shape[0], t.shape[1] + extra, dtype=t.dtype, device=DEV)
    big[:, :t.shape[1]] = t.to(DEV)
    return big[:, :t.shape[1]]


def shifted(t, n):
    """t on the GPU, contiguous, its first element n elements into an allocation."""
    buf = torch.zeros(t.numel() + n, dtype=t.dtype, device=DEV)
    v = buf[n:].view(t.shape)
    v.copy_(t)
    return v


# --------------------------------------------------------------------------- layer norm
NORM_CASES = [
    (1, 1, BF, BF), (1, 32, FF, FF), (3, 31, BF, FF), (5, 33, HF, HF), (64, 1280, BF, BF), (700, 1280, BF, FF),
    (1000, 64, BF, BF), (9, 1281, HF, FF), (600, 1281, BF, BF), (37, 3420, HF, FF), (601, 3420, BF, BF),
    (3, 8192, BF, BF), (2, 8191, BF, FF), (2, 4100, FF, FF), (5, 8200, BF, BF), (3, 20001, HF, FF), (800, 100, FF, FF),
]


def norm_inputs(T, C, dt, pt, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(T, C, generator=g) * torch.exp(0.5 * torch.randn(C, generator=g))
         + 3 * torch.randn(T, 1, generator=g)).to(dt)
    return x, 1 + randn(g, C, scale=0.2).to(pt), randn(g, C, dtype=pt, scale=0.3), randn(g, T, C, dtype=dt)


def norm_slack(x, w, rstd, C):
    """Error of (x - mean) rstd w + b before its rounding: mean is off by C 2^-23 mean|x|,
    rstd by (C + 8) 2^-23 of itself (and by mean's error squared, smaller), each value's
    own four operations by 2^-22."""
    ax = np.abs(x)
    h = (ax + ax.mean(1, keepdims=True)) * rstd[:, None]
    return (C + 16) * 2.0 ** -23 * h * np.abs(w)


@pytest.mark.parametrize("T,C,dt,pt", NORM_CASES)
def test_layer_norm(T, C, dt, pt):
    x, w, b, _ = norm_inputs(T, C, dt, pt)
    y, mean, rstd = fr.layer_norm(x.to(DEV), w.to(DEV), b.to(DEV), eps=1e-5, return_stats=True)
    ry, rm, rr = B.layer_norm(f64(x), f64(w), f64(b), 1e-5)
    near(mean, rm, FF, C * 2.0 ** -23 * np.abs(f64(x)).mean(1) + 1e-30)
    if C > 1:
        near(rstd, rr, FF, (C + 8) * 2.0 ** -22 * rr * (1 + rm ** 2 * rr ** 2 * C * 2.0 ** -23))
        near(y, ry, dt, norm_slack(f64(x), f64(w), rr, C) + 2.0 ** -22 * np.abs(f64(b)))
    else:  # one column: the difference from the mean is 0
        near(y, ry, dt, 2.0 ** -22)


@pytest.mark.parametrize("extra,n", [(8, 0), (4, 0), (1, 0), (0, 1), (0, 4), (8, 3)])
def test_layer_norm_rows_of_any_alignment(extra, n):
    x, w, b, dy = norm_inputs(40, 320, BF, BF)
    ref = fr.layer_norm(x.to(DEV), w.to(DEV), b.to(DEV), return_stats=True)
    xv = wide_rows(x, extra) if n == 0 else shifted(x, n)
    out = wide_rows(torch.zeros(40, 320, dtype=BF), 3)
    got = fr.layer_norm(xv, shifted(w, 1), shifted(b, 3), out=out, return_stats=True)
    assert got[0].data_ptr() == out.data_ptr()
    for a, c in zip(got, ref):  # the same sums in another order
        assert (a.float() - c.float()).abs().max() <= 2.0 ** -5  # one unit in the last place below 8
    dyv = wide_rows(dy, extra) if n == 0 else shifted(dy, n)
    a = fr.layer_norm_backward(dyv, xv, w.to(DEV), ref[1], ref[2])
    c = fr.layer_norm_backward(dy.to(DEV), x.to(DEV), w.to(DEV), ref[1], ref[2])
    for s, t in zip(a, c):
        assert torch.allclose(s.float(), t.float(), rtol=2.0 ** -7, atol=2.0 ** -12 * 40)


def test_layer_norm_without_parameters_and_broadcast_rows():
    x, w, b, _ = norm_inputs(6, 200, FF, FF)
    near(fr.layer_norm(x.to(DEV)), B.layer_norm(f64(x), None, None, 1e-6)[0], FF,
         norm_slack(f64(x), 1.0, B.layer_norm(f64(x), None, None, 1e-6)[2], 200))
    one = x[:1].to(DEV).expand(6, 200)  # row stride 0
    got = fr.layer_norm(one, w.to(DEV), None)
    assert (got == got[:1]).all()
    near(got[:1], B.layer_norm(f64(x[:1]), f64(w), None, 1e-6)[0], FF,
         norm_slack(f64(x[:1]), f64(w), B.layer_norm(f64(x[:1]), None, None, 1e-6)[2], 200))


def test_layer_norm_constant_rows_and_nonfinite_rows_stay_apart():
    x = torch.full((4, 96), 2.5)
    x[1, 5] = float("nan")
    x[2, 7] = float("inf")
    y, mean, rstd = fr.layer_norm(x.to(DEV), eps=1e-6, return_stats=True)
    y = y.cpu()
    assert (y[0] == 0).all() and (y[3] == 0).all() and torch.isnan(y[1]).all() and torch.isnan(y[2]).any()
    assert abs(float(rstd[0]) - 1000.0) < 1e-3


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("T,C,dt,pt", NORM_CASES)
def test_layer_norm_backward(T, C, dt, pt, packed):
    x, w, b, dy = norm_inputs(T, C, dt, pt, seed=1)
    _, m, r = B.layer_norm(f64(x), f64(w), f64(b), 1e-5)
    m, r = torch.from_numpy(m).float(), torch.from_numpy(r).float()
    arg, xv = x.to(DEV), f64(x)
    if packed:
        arg = fr.pack_activation(arg)
        xv = B.unpack(arg.codes.cpu().numpy(), arg.scales.cpu().numpy(), C)
    dx, dw, db = fr.layer_norm_backward(dy.to(DEV), arg, w.to(DEV), m.to(DEV), r.to(DEV))
    rx, rw, rb = B.layer_norm_bwd(f64(dy), xv, f64(w), f64(m), f64(r))
    h = (np.abs(xv) + np.abs(f64(m))[:, None]) * f64(r)[:, None]  # magnitudes of h's terms
    g = np.abs(f64(dy) * f64(w))
    eps = (C + 16) * 2.0 ** -23
    near(dx, rx, dt, eps * f64(r)[:, None] * (g + g.mean(1, keepdims=True) + h * (g * h).mean(1, keepdims=True)))
    near(dw, rw, pt, (T + 8) * 2.0 ** -23 * (np.abs(f64(dy)) * h).sum(0))
    near(db, rb, pt, (T + 8) * 2.0 ** -23 * np.abs(f64(dy)).sum(0))


def test_layer_norm_no_rows():
    x = torch.empty(0, 48, dtype=BF, device=DEV)
    w = torch.ones(48, dtype=BF, device=DEV)
    y, mean, rstd = fr.layer_norm(x, w, w, return_stats=True)
    assert y.shape == (0, 48) and mean.shape == (0,)
    dx, dw, db = fr.layer_norm_backward(x, x, w, mean, rstd)
    assert dx.shape == (0, 48) and (dw == 0).all() and (db == 0).all()


def test_layer_norm_backward_same_bits_every_run():
    x, w, b, dy = norm_inputs(5000, 1280, BF, FF)
    _, m, r = fr.layer_norm(x.to(DEV), w.to(DEV), b.to(DEV), return_stats=True)
    runs = [fr.layer_norm_backward(dy.to(DEV), x.to(DEV), w.to(DEV), m, r) for _ in range(3)]
    for o in runs[1:]:
        assert all(torch.equal(a, c) for a, c in zip(o, runs[0]))


# --------------------------------------------------------------------------- checkpoints
@pytest.mark.parametrize("dt", [BF, HF, FF])
@pytest.mark.parametrize("T,C", [(1, 1), (3, 31), (4, 32), (5, 33), (7, 100), (64, 1280), (1000, 1281), (33, 3420), (2, 20000)])
def test_pack_matches_the_format_bit_for_bit(T, C, dt):
    g = torch.Generator().manual_seed(T * C)
    x = (torch.randn(T, C, generator=g) * torch.exp(2 * torch.randn(T, 1, generator=g))).to(dt)
    x[0, : min(C, 32)] = 0  # an all-zero block
    p = fr.pack_activation(x.to(DEV))
    codes, scales = B.pack(f64(x))
    assert np.array_equal(p.codes.cpu().numpy(), codes) and np.array_equal(p.scales.cpu().numpy(), scales)
    back = fr.unpack_activation(p)
    assert back.dtype == dt and np.array_equal(f64(back), B.unpack(codes, scales, C))
    assert torch.equal(fr.unpack_activation(fr.pack_activation(back)), back)


@pytest.mark.parametrize("dt", [BF, HF, FF])
def test_pack_extremes(dt):
    """Largest and smallest magnitudes of the type stay finite and exact where they fit 7
    bits; an infinity or a NaN turns its own block into NaN and no other."""
    fi = torch.finfo(dt)
    x = torch.zeros(6, 64, dtype=dt)
    x[0] = fi.max
    x[1, 3], x[1, 40] = -fi.max, fi.tiny
    x[2, :32] = torch.arange(32).to(dt) * fi.smallest_normal
    x[3, 1] = float("inf")
    x[4, 33] = float("nan")
    x[5, 0], x[5, 1] = 1.0, 127.0 / 128
    p = fr.pack_activation(x.to(DEV))
    codes, scales = B.pack(f64(x))
    assert np.array_equal(p.codes.cpu().numpy(), codes) and np.array_equal(p.scales.cpu().numpy(), scales)
    back = fr.unpack_activation(p).cpu()
    assert torch.isfinite(back[[0, 1, 2, 5]]).all()
    assert torch.isnan(back[3, :32]).all() and (back[3, 32:] == 0).all()
    assert torch.isnan(back[4, 32:]).all() and (back[4, :32] == 0).all()


@pytest.mark.parametrize("extra,n", [(8, 0), (4, 0), (1, 0), (0, 1), (0, 4)])
def test_pack_rows_of_any_alignment(extra, n):
    x = randn(torch.Generator().manual_seed(0), 20, 160, dtype=BF)
    xv = wide_rows(x, extra) if n == 0 else shifted(x, n)
    a, b = fr.pack_activation(xv), fr.pack_activation(x.to(DEV))
    assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
    out = wide_rows(torch.zeros(20, 160, dtype=BF), extra)
    assert torch.equal(fr.unpack_activation(a, out=out), fr.unpack_activation(b))
    e = fr.pack_activation(torch.empty(0, 40, dtype=BF, device=DEV))
    assert fr.unpack_activation(e).shape == (0, 40)


# --------------------------------------------------------------------------- linear layer
LINEAR_CASES = [  # T, K, N, dtype, act, bias, residual, save
    (1, 64, 64, BF, "none", True, False, None),
    (1, 1280, 3424, BF, "silu", True, False, None),
    (2, 1281, 70, HF, "gelu", True, True, "full"),
    (17, 200, 333, BF, "gelu_tanh", False, True, "packed"),
    (33, 8, 1, BF, "none", True, True, None),
    (64, 1280, 1280, BF, "none", True, True, None),
    (65, 72, 130, HF, "relu", True, False, "packed"),
    (77, 1, 40, BF, "silu", True, False, "full"),
    (129, 520, 257, BF, "gelu", True, True, "packed"),
    (200, 3420, 320, BF, "none", True, True, "full"),
    (333, 1280, 3420, HF, "gelu", True, False, "full"),
    (513, 640, 1024, BF, "silu", False, False, "packed"),
    (1030, 320, 520, BF, "gelu_tanh", True, True, "full"),
]


def linear_inputs(T, K, N, dt, bias, residual, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (randn(g, T, K, dtype=dt), randn(g, N, K, dtype=dt, scale=K ** -0.5),
            randn(g, N, dtype=dt, scale=0.3) if bias else None, randn(g, T, N, dtype=dt) if residual else None)


def linear_ref(x, w, b, r, act):
    x, w = f64(x), f64(w)
    z = B.linear(x, w, None if b is None else f64(b))
    mag = np.abs(x) @ np.abs(w).T + (0 if b is None else np.abs(f64(b)))
    y = B.act(z, act) + (0 if r is None else f64(r))
    return z, y, (x.shape[1] + 2) * 2.0 ** -23 * mag


def gpu(*ts):
    return [None if t is None else t.to(DEV) for t in ts]


def check_preact(kept, z, slack, dt):
    if isinstance(kept, fr.PackedActivation):
        back = f64(fr.unpack_activation(kept._replace(dtype=FF)))
        step = np.repeat(np.ldexp(1.0, f64(kept.scales).astype(int) - 127), 32, 1)[:, :z.shape[1]]
        # half a step of the scale in use, which may be its neighbour's where the largest
        # magnitude lies within the sum's error of a power of two
        assert (np.abs(back - z) <= np.where(np.abs(z) > 127 * step, step, step / 2) + slack).all()
        assert (f64(kept.codes)[:, z.shape[1]:] == 0).all()
    else:
        near(kept, z, dt, slack)


@pytest.mark.parametrize("T,K,N,dt,act,bias,residual,save", LINEAR_CASES)
def test_linear_act(T, K, N, dt, act, bias, residual, save):
    x, w, b, r = linear_inputs(T, K, N, dt, bias, residual)
    got = fr.linear_act(*gpu(x, w, b), activation=act, residual=gpu(r)[0], save_preact=save)
    torch.cuda.synchronize()
    assert last_status(DEV) == 0
    y, kept = got if save else (got, None)
    z, ry, slack = linear_ref(x, w, b, r, act)
    near(y, ry, dt, 1.13 * slack + 2.0 ** -20 * np.abs(z) + 2.0 ** -23 * np.abs(ry))
    if save:
        check_preact(kept, z, slack, dt)


def test_linear_act_strided_rows_out_and_in_place_residual():
    x, w, b, r = linear_inputs(150, 192, 264, BF, True, True)
    ref = fr.linear_act(*gpu(x, w, b), activation="silu", residual=r.to(DEV))
    wide = wide_rows(w, 24)
    for extra in (8, 1, 4):
        out = wide_rows(torch.zeros(150, 264, dtype=BF), extra)
        got = fr.linear_act(wide_rows(x, 8 * extra), wide, shifted(b, 1), activation="silu",
                            residual=wide_rows(r, extra), out=out)
        assert got.data_ptr() == out.data_ptr() and torch.equal(got, ref)
        assert (out._base[:, 264:] == 0).all()  # nothing past the row's end
    for n in (0, 1):
        acc = shifted(r, n)
        assert torch.equal(fr.linear_act(*gpu(x, w, b), activation="silu", residual=acc, out=acc), ref)
    assert torch.equal(fr.linear_act(shifted(x, 3), shifted(w, 1), b.to(DEV), activation="silu", residual=shifted(r, 5)),
                       ref)


def test_linear_act_rows_do_not_depend_on_each_other():
    """A NaN or an infinity in one row of x reaches that row alone."""
    for T in (5, 300):
        x, w, b, _ = linear_inputs(T, 256, 320, BF, True, False)
        clean = fr.linear_act(*gpu(x, w, b), activation="gelu")
        x[2, 7], x[4, 9] = float("nan"), float("inf")
        got = fr.linear_act(*gpu(x, w, b), activation="gelu")
        rest = [i for i in range(T) if i not in (2, 4)]
        assert torch.isnan(got[2]).all() and not torch.isfinite(got[4]).all()
        assert torch.equal(got[rest], clean[rest])


def test_linear_act_no_rows():
    x, w, b, _ = linear_inputs(3, 64, 40, BF, True, False)
    y, p = fr.linear_act(x[:0].to(DEV), *gpu(w, b), activation="gelu", save_preact="packed")
    assert y.shape == (0, 40) and p.shape == (0, 40)
    dx, dw, db = fr.linear_act_backward(y, x[:0].to(DEV), w.to(DEV), p, activation="gelu")
    assert dx.shape == (0, 64) and dw.shape == (40, 64) and (dw == 0).all() and (db == 0).all()


LINEAR_BWD_CASES = [  # T, K, N, dtype, act
    (1, 64, 64, BF, "none"), (1, 1280, 40, HF, "gelu"), (3, 33, 65, BF, "silu"), (64, 320, 320, BF, "none"),
    (65, 200, 333, HF, "relu"), (130, 1281, 70, BF, "gelu_tanh"), (257, 520, 264, BF, "gelu"),
    (700, 640, 1288, BF, "silu"), (1000, 1280, 172, HF, "gelu_tanh"), (2100, 136, 72, BF, "none"),
]


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("T,K,N,dt,act", LINEAR_BWD_CASES)
def test_linear_act_backward(T, K, N, dt, act, packed):
    x, w, _, dy = linear_inputs(T, K, N, dt, False, True, seed=3)
    z = randn(torch.Generator().manual_seed(4), T, N, dtype=dt)
    xa, za, xv, zv = x.to(DEV), z.to(DEV), f64(x), f64(z)
    if packed:
        xa, za = fr.pack_activation(xa), fr.pack_activation(za)
        xv, zv = (B.unpack(p.codes.cpu().numpy(), p.scales.cpu().numpy(), p.width) for p in (xa, za))
    dx, dw, db = fr.linear_act_backward(dy.to(DEV), xa, w.to(DEV), za if act != "none" else None, activation=act)
    torch.cuda.synchronize()
    assert last_status(DEV) == 0
    dz, rx, rw, rb = B.linear_act_bwd(f64(dy), xv, f64(w), zv, act)
    u = 0 if act == "none" else 1.01 * U[dt] + 2.0 ** -20
    ady = 1.13 * np.abs(f64(dy)) if act != "none" else np.abs(f64(dy))
    mx, mw = ady @ np.abs(f64(w)), ady.T @ np.abs(xv)
    near(dx, rx, dt, (u + (N + 2) * 2.0 ** -23) * mx + TINY[dt] * np.abs(f64(w)).sum(0))
    near(dw, rw, dt, (u + (T + 2) * 2.0 ** -23) * mw + TINY[dt] * np.abs(xv).sum(0))
    near(db, rb, dt, ((T + 2) * 2.0 ** -23 + 2.0 ** -20) * ady.sum(0))
    if T * N > 1000:
        assert rel(dx, rx) < U[dt] and rel(dw, rw) < U[dt]


def test_linear_act_backward_strided_inputs_and_need():
    x, w, _, dy = linear_inputs(90, 96, 136, BF, False, True)
    z = randn(torch.Generator().manual_seed(5), 90, 136, dtype=BF)
    ref = fr.linear_act_backward(*gpu(dy, x, w, z), activation="gelu")
    for extra in (8, 1):
        got = fr.linear_act_backward(wide_rows(dy, extra), wide_rows(x, 8 * extra), wide_rows(w, 8), wide_rows(z, extra),
                                     activation="gelu")
        assert all(torch.equal(a, b) for a, b in zip(got[:2], ref[:2]))
        near(got[2], f64(ref[2]), BF, 92 * 2.0 ** -22 * np.abs(f64(dy)).sum(0))  # another order of the same sum
    for need in ((True, False, False), (False, True, False), (False, False, True)):
        got = fr.linear_act_backward(*gpu(dy, x, w, z), activation="gelu", need=need)
        for a, b, n in zip(got, ref, need):
            assert (torch.equal(a, b)) if n else a is None
    for dyv in (wide_rows(dy, 1), wide_rows(dy, 8), dy.to(DEV)):  # no activation: dout itself is the operand
        a = fr.linear_act_backward(dyv, *gpu(x, w))
        b = fr.linear_act_backward(*gpu(dy, x, w))
        assert all(torch.equal(s, t) for s, t in zip(a[:2], b[:2]))


def test_linear_act_backward_same_bits_every_run():
    x, w, _, dy = linear_inputs(3000, 320, 640, BF, False, True)
    z = randn(torch.Generator().manual_seed(6), 3000, 640, dtype=BF)
    runs = [fr.linear_act_backward(*gpu(dy, x, w, z), activation="silu") for _ in range(3)]
    for o in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(o, runs[0]))


# --------------------------------------------------------------------------- autograd nodes
@pytest.mark.parametrize("checkpoint", [False, True])
def test_train_nodes_against_differences(checkpoint):
    """Directional derivatives of a norm + MLP pair: the nodes' gradients against central
    differences of the oracle's forward (64 bits). The gradients carry a few 16-bit
    roundings (2^-11 each, fp16), the checkpointed ones the 8-bit steps: at most 2^-7 of a
    block's largest value each, about 2^-8.5 of a typical one in the 2-norm, in x, in
    the pre-activation and in the norm's input."""
    T, C, N = 48, 64, 96
    g = torch.Generator().manual_seed(11)
    x = randn(g, T, C, dtype=HF)
    nw, nb_ = 1 + randn(g, C, scale=0.2), randn(g, C, scale=0.2)
    w1, b1 = randn(g, N, C, dtype=HF, scale=C ** -0.5), randn(g, N, dtype=HF, scale=0.2)
    w2, b2 = randn(g, C, N, dtype=HF, scale=N ** -0.5), randn(g, C, dtype=HF, scale=0.2)
    dy = randn(g, T, C, dtype=HF)
    ps = [t.to(DEV).requires_grad_(True) for t in (x, nw, nb_, w1, b1, w2, b2)]
    h = fr.layer_norm_train(ps[0], ps[1], ps[2], checkpoint=checkpoint)
    h = fr.linear_act_train(h, ps[3], ps[4], activation="gelu", checkpoint=checkpoint)
    y = fr.linear_act_train(h, ps[5], ps[6], residual=ps[0], checkpoint=checkpoint)
    y.backward(dy.to(DEV))

    def loss(v):
        a = B.layer_norm(v[0], v[1], v[2], 1e-6)[0]
        a = B.act(B.linear(a, v[3], v[4]), "gelu")
        return ((B.linear(a, v[5], v[6]) + v[0]) * f64(dy)).sum()

    vals = [f64(t) for t in ps]
    rng = np.random.default_rng(2)
    for i, p in enumerate(ps):
        # along the gradient itself: a derivative of the gradient's own size, no cancellation
        d = f64(p.grad) / np.linalg.norm(f64(p.grad))
        e = 1e-5
        up, dn = list(vals), list(vals)
        up[i], dn[i] = vals[i] + e * d, vals[i] - e * d
        num = (loss(up) - loss(dn)) / (2 * e)
        got = (f64(p.grad) * d).sum()
        assert abs(num - got) <= (2e-2 if checkpoint else 4e-3) * abs(num), (i, num, got)
        d = rng.normal(size=vals[i].shape)
        d /= np.linalg.norm(d)
        up[i], dn[i] = vals[i] + e * d, vals[i] - e * d
        num = (loss(up) - loss(dn)) / (2 * e)
        assert abs(num - (f64(p.grad) * d).sum()) <= (4e-2 if checkpoint else 8e-3) * np.linalg.norm(f64(p.grad)) + 1e-6


def test_operators_on_another_stream():
    x, w, b, r = linear_inputs(260, 320, 648, BF, True, True)
    xs = gpu(x, w, b, r)
    nw = torch.ones(320, dtype=BF, device=DEV)

    def step():
        y, m, s = fr.layer_norm(xs[0], nw, return_stats=True)
        o, z = fr.linear_act(y, xs[1], xs[2], activation="gelu", residual=xs[3], save_preact="packed")
        g = fr.linear_act_backward(xs[3], fr.pack_activation(y), xs[1], z, activation="gelu")
        return (o, *g, *fr.layer_norm_backward(g[0], xs[0], nw, m, s))

    ref = step()
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = step()
    st.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(got, ref))
    with torch.cuda.stream(st):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            cap = step()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(cap, ref))


# --------------------------------------------------------------------------- refusals
def test_gpu_refusals():
    x = torch.zeros(4, 64, dtype=BF, device=DEV)
    w = torch.zeros(8, 64, dtype=BF, device=DEV)
    f = torch.zeros(4, device=DEV)
    bad = [
        lambda: fr.layer_norm(x[0]), lambda: fr.layer_norm(x.double()), lambda: fr.layer_norm(x, x[0, :32]),
        lambda: fr.layer_norm(x, x[0].half()), lambda: fr.layer_norm(x, x[0].float(), x[0]),
        lambda: fr.layer_norm(x, eps=-1.0), lambda: fr.layer_norm(x, out=x[:2]),
        lambda: fr.layer_norm(x, out=x.float()), lambda: fr.layer_norm(x, x[0].cpu()),
        lambda: fr.layer_norm_backward(x, x[:2], None, f, f), lambda: fr.layer_norm_backward(x, x.half(), None, f, f),
        lambda: fr.layer_norm_backward(x, x, None, f[:2], f), lambda: fr.layer_norm_backward(x, x, None, f, f.double()),
        lambda: fr.layer_norm_backward(x, fr.pack_activation(x[:, :32]), None, f, f),
        lambda: fr.linear_act(x.float(), w.float()), lambda: fr.linear_act(x, w[:, :32]), lambda: fr.linear_act(x, w.half()),
        lambda: fr.linear_act(x, w, x[0]), lambda: fr.linear_act(x, w, activation="tanh"),
        lambda: fr.linear_act(x, w, residual=x), lambda: fr.linear_act(x, w, save_preact="8bit"),
        lambda: fr.linear_act(x, w, out=x), lambda: fr.linear_act(x, w.cpu()),
        lambda: fr.linear_act(x, w, out=torch.zeros(8, 4, dtype=BF, device=DEV).t()),
        lambda: fr.linear_act(x, w, out=torch.zeros(1, 8, dtype=BF, device=DEV).expand(4, 8)),
        lambda: fr.linear_act_backward(x[:, :8], x, w, activation="gelu"),
        lambda: fr.linear_act_backward(x, x, w), lambda: fr.linear_act_backward(x[:, :8], x[:2], w),
        lambda: fr.linear_act_backward(x[:, :8], x, w, x, activation="relu"),
        lambda: fr.linear_act_backward(x[:, :8], fr.pack_activation(x.half()), w),
        lambda: fr.pack_activation(x.to(torch.int32)), lambda: fr.pack_activation(x[:, :0]),
        lambda: fr.unpack_activation(fr.pack_activation(x), out=x[:2]),
    ]
    for i, f_ in enumerate(bad):
        with pytest.raises(ValueError):
            f_()
            print("accepted:", i)
    torch.cuda.synchronize()
    assert last_status(DEV) == 0


def test_gradients_of_broadcast_outputs():
    """y.sum().backward() hands an expanded gradient (strides 0) to the nodes, and a
    gradient whose rows are one row repeated (row stride 0) is read in place."""
    x, w, b, _ = linear_inputs(70, 64, 48, BF, True, False)
    ps = [t.to(DEV).requires_grad_(True) for t in (x, w, b)]
    fr.linear_act_train(*ps, activation="relu").sum().backward()
    one = torch.ones(70, 48, dtype=BF, device=DEV)
    z = fr.linear_act(*gpu(x, w, b), save_preact="full")[1]
    ref = fr.linear_act_backward(one, x.to(DEV), w.to(DEV), z, activation="relu")
    assert all(torch.equal(p.grad, r) for p, r in zip(ps, ref))
    for act in ("none", "relu"):
        got = fr.linear_act_backward(one[:1].expand(70, 48), x.to(DEV), w.to(DEV), z, activation=act)
        ref = fr.linear_act_backward(one, x.to(DEV), w.to(DEV), z, activation=act)
        assert all(torch.equal(s, t) for s, t in zip(got, ref))
    nx = x.to(DEV).requires_grad_(True)
    fr.layer_norm_train(nx).sum().backward()
    assert nx.grad.abs().max() <= 2.0 ** -6  # the sum of a row's outputs is constant


@pytest.mark.parametrize("act", ["relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("dt", [BF, HF])
def test_activations_over_their_whole_range(act, dt):
    """Every magnitude the type has, forward (K = 1, weight 1: z = x) and derivative: near the
    formula within the approximations' 2^-20 of |z| (1 + |z|) for the derivative's factor, and a
    NaN or an infinity changes no other column."""
    mag = torch.logspace(-6, 4.5, 400, dtype=torch.float64)
    z = torch.cat([mag, -mag, torch.zeros(1, dtype=torch.float64)]).to(dt)
    z = z[torch.isfinite(z)]
    N = z.numel()
    x = torch.ones(1, 1, dtype=dt, device=DEV)
    y = fr.linear_act(x, z.view(N, 1).to(DEV), activation=act)
    zz = f64(z)
    with np.errstate(over="ignore", invalid="ignore"):
        ry, rg = B.act(zz, act), B.act_grad(np.clip(zz, -1e3, 1e3), act)
    near(y[0], ry, dt, 2.0 ** -20 * np.abs(zz))
    eye = torch.eye(1, dtype=dt, device=DEV)
    _, _, db = fr.linear_act_backward(torch.ones(1, N, dtype=dt, device=DEV), eye, z.view(N, 1).to(DEV), z.view(1, N).to(DEV),
                                      activation=act)
    near(db, rg, dt, 2.0 ** -20 * (1 + np.minimum(np.abs(zz), 64)))
    bad = z.clone()
    bad[7], bad[100] = float("nan"), float("inf")
    keep = [i for i in range(N) if i not in (7, 100)]
    yb = fr.linear_act(x, bad.view(N, 1).to(DEV), activation=act)
    assert torch.equal(yb[0][keep], y[0][keep]) and torch.isnan(yb[0, 7]) and yb[0, 100] == float("inf")
    _, _, gb = fr.linear_act_backward(torch.ones(1, N, dtype=dt, device=DEV), eye, z.view(N, 1).to(DEV), bad.view(1, N).to(DEV),
                                      activation=act)
    assert torch.equal(gb[keep], db[keep]) and torch.isnan(gb[7]) and gb[100] == 1


@pytest.mark.parametrize("T", [295, 296, 297, 591, 592, 593, 1777])
@pytest.mark.parametrize("C,dt", [(1280, BF), (1285, HF), (2600, BF), (5004, BF)])
def test_layer_norm_either_side_of_its_rules(T, C, dt):
    """Rows around the counts where the kernels change, widths of one to several warps: the
    same rows give the same outputs whatever the number of rows."""
    x, w, b, dy = norm_inputs(1777, C, dt, FF, seed=7)
    w, b = w.to(DEV), b.to(DEV)
    y, mean, rstd = fr.layer_norm(x[:T].to(DEV), w, b, return_stats=True)
    ry, rm, rr = B.layer_norm(f64(x[:T]), f64(w), f64(b), 1e-6)
    near(y, ry, dt, norm_slack(f64(x[:T]), f64(w), rr, C) + 2.0 ** -22 * np.abs(f64(b)))
    dx, dw, db = fr.layer_norm_backward(dy[:T].to(DEV), x[:T].to(DEV), w, mean, rstd)
    rx, rw, rb = B.layer_norm_bwd(f64(dy[:T]), f64(x[:T]), f64(w), f64(mean), f64(rstd))
    h = (np.abs(f64(x[:T])) + np.abs(f64(mean))[:, None]) * f64(rstd)[:, None]
    g = np.abs(f64(dy[:T]) * f64(w))
    eps = (C + 16) * 2.0 ** -23
    near(dx, rx, dt, eps * f64(rstd)[:, None] * (g + g.mean(1, keepdims=True) + h * (g * h).mean(1, keepdims=True)))
    near(dw, rw, FF, (T + 8) * 2.0 ** -23 * (np.abs(f64(dy[:T])) * h).sum(0))
    near(db, rb, FF, (T + 8) * 2.0 ** -23 * np.abs(f64(dy[:T])).sum(0))


@pytest.mark.parametrize("T,K,N,act,save", [
    (512, 512, 512, "gelu", "packed"), (2304, 128, 640, "silu", "full"), (4100, 640, 1288, "gelu_tanh", "packed"),
    (300, 5120, 640, "none", "packed"), (1100, 4096, 264, "relu", "full"), (2560, 2048, 256, "gelu", None),
    (1024, 8192, 512, "silu", "packed"), (1000, 8200, 500, "relu", "full"), (9216, 1288, 1000, "relu", None),
    (9000, 1280, 1280, "none", "packed"),
])
def test_linear_act_on_each_path(T, K, N, act, save):
    """Sizes that take the pair kernel in whole tiles and in split ones (of the forward: long
    reductions of few tiles; of the weight gradient: many rows) and the small kernel with
    several CTAs a tile, with a residual; checked on the GPU in 64 bits."""
    x, w, b, r = [t.to(DEV) for t in linear_inputs(T, K, N, BF, True, True, seed=9)]
    got = fr.linear_act(x, w, b, activation=act, residual=r, save_preact=save)
    y, kept = got if save else (got, None)
    xd, wd = x.double(), w.double()
    z = xd @ wd.t() + b.double()
    slack = f64((K + 2) * 2.0 ** -23 * (xd.abs() @ wd.abs().t() + b.double().abs()))
    zn = f64(z)
    ry = B.act(zn, act) + f64(r)
    near(y, ry, BF, 1.13 * slack + 2.0 ** -20 * np.abs(zn) + 2.0 ** -23 * np.abs(ry))
    if save:
        check_preact(kept, zn, slack, BF)
    acc = r.clone()
    assert torch.equal(fr.linear_act(x, w, b, activation=act, residual=acc, out=acc), y)
    z16 = torch.randn(T, N, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).to(BF)
    dx, dw, db = fr.linear_act_backward(r, x, w, z16, activation=act)
    dz = f64(r) * (1 if act == "none" else B.act_grad(f64(z16), act))
    d = torch.from_numpy(dz).to(DEV)
    assert rel(dx, f64(d @ wd)) < U[BF] and rel(dw, f64(d.t() @ xd)) < U[BF]
    near(db, dz.sum(0), BF, ((T + 2) * 2.0 ** -23 + 2.0 ** -20) * 1.13 * np.abs(f64(r)).sum(0))
    assert last_status(DEV) == 0
