"""Transformer-block operators around the attention: layer norm, linear layer with
bias, activation and residual in its epilogue, and 8-bit activation checkpoints.

The reference (sdan/fused-rope-attn) has the attention alone, forward only
(fused_attn.py:139-232). A block that is trained or served around it needs the
operators here; each calls hand-written sm_100a kernels through the C ABI
(include/frattn.h) on the current stream:

* ``layer_norm`` / ``layer_norm_backward``; ``layer_norm_train`` records the pair
  as an autograd node;
* ``linear_act`` / ``linear_act_backward``; ``linear_act_train`` likewise;
* ``pack_activation`` / ``unpack_activation``: a tensor kept for the backward pass
  in 8 bits (blocks of 32 values with a power-of-two scale each). Both backward
  passes take a ``PackedActivation`` in the place of the tensor it stands for, and
  the autograd nodes keep their inputs that way with ``checkpoint=True``.

Matrices are ``[T, C]`` with packed columns; rows may be strided (views of wider
buffers are read in place). The forms without ``_train`` record no gradient, whatever
their inputs require; ``out=`` is written in place and its version moves on.
"""
from __future__ import annotations

import functools
from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .fused_attn import _DT, _status_word, _written

__all__ = [
    "ACTIVATIONS",
    "PackedActivation",
    "pack_activation",
    "unpack_activation",
    "layer_norm",
    "layer_norm_backward",
    "layer_norm_train",
    "linear_act",
    "linear_act_backward",
    "linear_act_train",
]

PACK_BLOCK = 32

# Values of the FRATTN_ACT_* enum of include/frattn.h.
ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}


_entries: dict = {}
# The current stream's handle and device alone, where torch has them: the public calls
# build objects around them, a quarter of a small call's time.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _call(name: str, device: torch.device, *args) -> None:
    """Calls a C entry on ``device`` with its current stream as the last argument."""
    fn = _entries.get(name)
    if fn is None:
        fn = _entries[name] = getattr(_lib.load(), name)
    i = device.index
    if i is not None and i == _current_device():
        rc = fn(*args, _raw_stream(i) if _raw_stream is not None else torch.cuda.current_stream(device).cuda_stream)
    else:
        with torch.cuda.device(device):
            rc = fn(*args, torch.cuda.current_stream(device).cuda_stream)
    if rc:
        _lib.check(rc, name)


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(query, device, *sizes) -> int:
    """Workspace sizes are a function of the shape and the device."""
    with torch.cuda.device(device):
        return query(*sizes)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _workspace(nbytes: int, device) -> torch.Tensor:
    return torch.empty(nbytes, dtype=torch.uint8, device=device)


def _check_rows(name, t, dtypes):
    if not t.is_cuda:
        raise ValueError(f"{name} must be on CUDA, got device={t.device}")
    if t.ndim != 2:
        raise ValueError(f"{name} must be 2D [T, C], got {tuple(t.shape)}")
    if t.dtype not in dtypes:
        raise ValueError(f"{name} dtype must be one of {', '.join(str(d)[6:] for d in dtypes)}, got {t.dtype}")
    if t.shape[1] <= 0:
        raise ValueError(f"{name} must have at least one column, got {tuple(t.shape)}")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t with packed columns (rows may be strided); copied when they are not."""
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _rows16(t: torch.Tensor) -> tuple[torch.Tensor, int]:
    """t with rows that start on 16-byte boundaries (a TMA requirement), and their stride: t
    itself, or a copy in rows padded to a multiple of 8 elements. A weight whose width is
    not a multiple of 8 is best kept that way by its owner (a ``[:, :K]`` view of a
    padded buffer), so that no call copies it."""
    n, k = t.shape
    s, c = t.stride()
    if (c == 1 or k == 1) and t.data_ptr() % 16 == 0:
        if n == 1:
            return t, -(-k // 8) * 8
        if s % 8 == 0 and s >= k:
            return t, s
    kp = -(-k // 8) * 8
    return torch.empty(n, kp, dtype=t.dtype, device=t.device)[:, :k].copy_(t), kp


def _stride(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[1])


def _check_out_rows(out, shape, like, name="out"):
    if out is None:
        return torch.empty(shape, dtype=like.dtype, device=like.device)
    if tuple(out.shape) != tuple(shape) or out.dtype != like.dtype or out.device != like.device:
        raise ValueError(f"{name} must be {tuple(shape)} {like.dtype} on {like.device}, "
                         f"got {tuple(out.shape)} {out.dtype} on {out.device}")
    if out.stride(1) != 1 and out.shape[1] > 1 or out.shape[0] > 1 and out.stride(0) < out.shape[1]:
        raise ValueError(f"{name} must have packed columns and non-overlapping rows, got strides {out.stride()}")
    return out


def _bytes_of(t: torch.Tensor) -> tuple[int, int]:
    """Addresses of the first byte of t, a matrix or a vector, and past its last."""
    p, n, s = t.data_ptr(), t.shape, t.stride()
    last = (n[0] - 1) * s[0] + ((n[1] - 1) * s[1] if len(n) == 2 else 0)
    return p, p + t.element_size() * (last + 1)


def _apart(out: torch.Tensor, t: torch.Tensor, span: tuple[int, int] | None = None) -> bool:
    """Whether rows ``out`` (``span`` its addresses, where known) and a matrix or vector t,
    neither empty, have no byte in common: one ends before the other begins, or they are
    columns of one buffer that do not meet. (Rows of different strides that interleave
    count as sharing.)"""
    a, a_end = span or _bytes_of(out)
    b, b_end = _bytes_of(t)
    if a_end <= b or b_end <= a:
        return True
    row = out.stride(0) * out.element_size()
    if t.ndim != 2 or row <= 0 or row != t.stride(0) * t.element_size():
        return False
    at = (b - a) % row  # where t's columns begin in a row of out
    return out.shape[1] * out.element_size() <= at and at + t.shape[1] * t.element_size() <= row


def _check_apart(out, itself=None, **inputs):
    """Refuses an ``out`` that shares memory with an input of its call (None: not given). The input
    named ``itself`` may be exactly out: each row (or tile) of it is read before it is written."""
    span = _bytes_of(out)
    for name, t in inputs.items():
        if t is None or _apart(out, t, span):
            continue
        if name != itself:
            raise ValueError(f"out must not share memory with {name}")
        if t.data_ptr() != out.data_ptr() or t.stride(0) != out.stride(0) and t.shape[0] > 1:
            raise ValueError(f"out must be {name} itself or not share memory with it")


# --------------------------------------------------------------------------- 8-bit checkpoints
class PackedActivation(NamedTuple):
    """An ``[T, width]`` tensor kept in 8 bits: ``codes`` int8 ``[T, 32 * nb]`` and
    ``scales`` uint8 ``[T, nb]`` (biased exponents), ``nb = ceil(width / 32)``; ``dtype``
    is the type of the tensor it stands for. A value is ``code * 2**(scale - 127)``;
    a block that held an infinity or a NaN has scale 255 and stands for NaN."""

    codes: torch.Tensor
    scales: torch.Tensor
    width: int
    dtype: torch.dtype

    @property
    def shape(self):
        return torch.Size((self.scales.shape[0], self.width))

    @property
    def device(self):
        return self.codes.device


def _check_packed(name, p, dtype=None, shape=None):
    codes, scales, width, dt = p
    t, nb = scales.shape if scales.ndim == 2 else (-1, -1)
    if nb != -(-width // PACK_BLOCK) or width <= 0 or codes.shape != (t, nb * PACK_BLOCK):
        raise ValueError(f"{name}: codes {tuple(codes.shape)} and scales {tuple(scales.shape)} do not hold "
                         f"rows of {width} values in blocks of {PACK_BLOCK}")
    if codes.dtype is not torch.int8 or scales.dtype is not torch.uint8 or codes.device != scales.device:
        raise ValueError(f"{name}: codes must be int8 and scales uint8 on one device, got {codes.dtype} on "
                         f"{codes.device} and {scales.dtype} on {scales.device}")
    if not codes.is_cuda:
        raise ValueError(f"{name} must be on CUDA, got device={codes.device}")
    if not codes.is_contiguous() or not scales.is_contiguous() or codes.data_ptr() % 16:
        raise ValueError(f"{name}: codes and scales must be contiguous, codes 16-byte aligned")
    if shape is not None and (t, width) != tuple(shape):
        raise ValueError(f"{name} must stand for {tuple(shape)}, got {(t, width)}")
    if dtype is not None and dt != dtype:
        raise ValueError(f"{name} must stand for {dtype}, got {dt}")


def _empty_packed(rows, width, dtype, device) -> PackedActivation:
    nb = -(-width // PACK_BLOCK)
    return PackedActivation(torch.empty(rows, nb * PACK_BLOCK, dtype=torch.int8, device=device),
                            torch.empty(rows, nb, dtype=torch.uint8, device=device), width, dtype)


def pack_activation(x: torch.Tensor) -> PackedActivation:
    """``x`` ``[T, C]`` (float32, float16 or bfloat16) in 8 bits: 1 + 1/32 bytes a value.

    Per block of 32 columns with largest magnitude ``f * 2**q`` (1/2 <= f < 1) the step is
    ``2**max(q - 7, -126)`` and each value is rounded to the nearest multiple of it
    (ties to even; at most 127 steps)."""
    _check_rows("x", x, tuple(_DT))
    T, C = x.shape
    dt, dev = x.dtype, x.device
    xs, xc = x.stride()
    if xc != 1 and C > 1:
        x, xs = x.contiguous(), C
    p = _empty_packed(T, C, dt, dev)
    _call("frattn_act_pack", dev, x.data_ptr(), xs, T, C, _DT[dt], p.codes.data_ptr(), p.scales.data_ptr())
    return p


def unpack_activation(p: PackedActivation, *, out: torch.Tensor | None = None) -> torch.Tensor:
    """The values a checkpoint stands for, ``[T, width]`` of its dtype."""
    _check_packed("packed activation", p)
    if p.dtype not in _DT:
        raise ValueError(f"dtype must be float16, bfloat16 or float32, got {p.dtype}")
    codes, scales, C, dt = p
    T, dev = scales.shape[0], codes.device
    given = out is not None
    if not given:
        out, os = torch.empty((T, C), dtype=dt, device=dev), C
    else:
        out = _check_out_rows(out, (T, C), torch.empty(0, dtype=dt, device=dev))
        os = _stride(out)
        if T:
            _check_apart(out, codes=codes, scales=scales)
    _call("frattn_act_unpack", dev, codes.data_ptr(), scales.data_ptr(), T, C, _DT[dt], out.data_ptr(), os)
    return _written(out) if given else out


# --------------------------------------------------------------------------- layer norm
def _check_param(name, t, C, dtype, device):
    if t.shape != (C,):
        raise ValueError(f"{name} must be [{C}], got {tuple(t.shape)}")
    if t.dtype is not dtype and t.dtype is not torch.float32:
        raise ValueError(f"{name} dtype must be {dtype} or float32, got {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} must be on {device}, got {t.device}")
    return t.contiguous()


def layer_norm(
    x: torch.Tensor,
    weight: torch.Tensor | None = None,
    bias: torch.Tensor | None = None,
    *,
    eps: float = 1e-6,
    out: torch.Tensor | None = None,
    return_stats: bool = False,
):
    """Layer norm over the columns of ``x`` ``[T, C]`` (float32, float16 or bfloat16).

    ``weight`` and ``bias`` ``[C]`` in x's type or float32 (both the same). With
    ``return_stats`` also the fp32 ``mean`` and ``rstd`` ``[T]`` of the rows, which
    ``layer_norm_backward`` takes. ``out`` may be ``x`` itself, and shares no memory with
    the other inputs.
    """
    _check_rows("x", x, tuple(_DT))
    T, C = x.shape
    if not eps >= 0:
        raise ValueError(f"eps must be >= 0, got {eps}")
    dt, dev = x.dtype, x.device
    pd, wp, bp = dt, None, None
    if weight is not None:
        weight = _check_param("weight", weight, C, dt, dev)
        pd, wp = weight.dtype, weight.data_ptr()
    if bias is not None:
        bias = _check_param("bias", bias, C, dt, dev)
        if weight is not None and bias.dtype is not pd:
            raise ValueError(f"weight and bias must share a dtype, got {pd} and {bias.dtype}")
        pd, bp = bias.dtype, bias.data_ptr()
    xs, xc = x.stride()
    if xc != 1 and C > 1:
        x, xs = x.contiguous(), C
    given = out is not None
    if not given:
        out, os = torch.empty((T, C), dtype=dt, device=dev), C
    else:
        out = _check_out_rows(out, (T, C), x)
        os = _stride(out)
        if T:
            _check_apart(out, "x", x=x, weight=weight, bias=bias)
    if not return_stats:
        _call("frattn_layer_norm", dev, x.data_ptr(), xs, wp, bp, _DT[pd], T, C, eps, _DT[dt], out.data_ptr(), os, None, None)
        return _written(out) if given else out
    mean = torch.empty(T, dtype=torch.float32, device=dev)
    rstd = torch.empty_like(mean)
    _call("frattn_layer_norm", dev, x.data_ptr(), xs, wp, bp, _DT[pd], T, C, eps, _DT[dt], out.data_ptr(), os,
          mean.data_ptr(), rstd.data_ptr())
    return (_written(out) if given else out), mean, rstd


def layer_norm_backward(
    dout: torch.Tensor,
    x: torch.Tensor | PackedActivation,
    weight: torch.Tensor | None,
    mean: torch.Tensor,
    rstd: torch.Tensor,
    *,
    param_dtype: torch.dtype | None = None,
    need_param_grads: bool = True,
):
    """``(dx, dweight, dbias)`` of ``layer_norm`` for the output gradient ``dout`` ``[T, C]``.

    ``x`` is the forward's input or its checkpoint, ``mean`` / ``rstd`` the forward's (of the
    input itself, for a checkpoint too: they are not recomputed from the kept values).
    dweight and dbias come in ``weight``'s type (``param_dtype``, default x's, when
    weight is None); with ``need_param_grads=False`` they are not computed (None).
    """
    packed = isinstance(x, PackedActivation)
    _check_rows("dout", dout, tuple(_DT))
    T, C = dout.shape
    dev = dout.device
    if packed:
        _check_packed("x", x, dout.dtype, (T, C))
    else:
        _check_rows("x", x, tuple(_DT))
        if x.shape != dout.shape or x.dtype != dout.dtype:
            raise ValueError(f"x must match dout {tuple(dout.shape)} {dout.dtype}, got {tuple(x.shape)} {x.dtype}")
        x = _rows(x)
    if x.device != dev:
        raise ValueError(f"x must be on {dev}, got {x.device}")
    weight = None if weight is None else _check_param("weight", weight, C, dout.dtype, dev)
    pd = weight.dtype if weight is not None else param_dtype or dout.dtype
    if pd not in (dout.dtype, torch.float32):
        raise ValueError(f"param_dtype must be {dout.dtype} or float32, got {pd}")
    for name, t in (("mean", mean), ("rstd", rstd)):
        if t.shape != (T,) or t.dtype != torch.float32 or t.device != dev or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous float32 [{T}] on {dev}, got {tuple(t.shape)} {t.dtype}")
    dout = _rows(dout)
    dx = torch.empty(T, C, dtype=dout.dtype, device=dev)
    dw = db = ws = None
    nbytes = 0
    if need_param_grads:
        dw = torch.empty(C, dtype=pd, device=dev)
        db = torch.empty(C, dtype=pd, device=dev)
        nbytes = _workspace_bytes(_lib.workspace_bytes_layer_norm_bwd, dev, T, C)
        ws = _workspace(nbytes, dev)
    _call("frattn_layer_norm_bwd", dev, dout.data_ptr(), _stride(dout), None if packed else x.data_ptr(),
          0 if packed else _stride(x), x.codes.data_ptr() if packed else None,
          x.scales.data_ptr() if packed else None, _ptr(weight), _DT[pd], mean.data_ptr(), rstd.data_ptr(), T, C,
          _DT[dout.dtype], dx.data_ptr(), C, _ptr(dw), _ptr(db), _ptr(ws), nbytes)
    return dx, dw, db


class _LayerNorm(torch.autograd.Function):
    """Autograd node of ``layer_norm``; x is kept as it is or as a checkpoint."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps, checkpoint):
        out, mean, rstd = layer_norm(x, weight, bias, eps=eps, return_stats=True)
        ctx.has = (weight is not None, bias is not None)
        ctx.param_dtype = weight.dtype if weight is not None else bias.dtype if bias is not None else None
        ctx.packed = checkpoint
        if checkpoint:
            p = pack_activation(x)
            ctx.meta = (p.width, p.dtype)
            ctx.save_for_backward(p.codes, p.scales, weight, mean, rstd)
        else:
            ctx.save_for_backward(x, None, weight, mean, rstd)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        x, scales, weight, mean, rstd = ctx.saved_tensors
        if ctx.packed:
            x = PackedActivation(x, scales, *ctx.meta)
        need = any(ctx.needs_input_grad[1:3])
        dx, dw, db = layer_norm_backward(dout, x, weight, mean, rstd, param_dtype=ctx.param_dtype,
                                         need_param_grads=need)
        return dx, dw if ctx.has[0] else None, db if ctx.has[1] else None, None, None


def layer_norm_train(x, weight=None, bias=None, *, eps: float = 1e-6, checkpoint: bool = False) -> torch.Tensor:
    """``layer_norm`` with gradients for x, weight and bias, once differentiable (a second
    derivative through it raises). With ``checkpoint`` the node keeps x in 8 bits: the
    backward pass takes the kept values with the mean and rstd of x itself, so that the
    normalised row is off by the rounding of x alone."""
    return _LayerNorm.apply(x, weight, bias, eps, checkpoint)


# --------------------------------------------------------------------------- linear layer
_LINEAR_DT = (torch.float16, torch.bfloat16)


def _act_code(activation) -> int:
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {', '.join(ACTIVATIONS)}, got {activation!r}")
    return ACTIVATIONS[activation]


def _check_weight(weight, K, dtype, device):
    if weight.ndim != 2 or weight.shape[1] != K or weight.shape[0] <= 0:
        raise ValueError(f"weight must be [N, {K}], got {tuple(weight.shape)}")
    if weight.dtype != dtype or weight.device != device:
        raise ValueError(f"weight must be {dtype} on {device}, got {weight.dtype} on {weight.device}")


def linear_act(
    x: torch.Tensor,
    weight: torch.Tensor,
    bias: torch.Tensor | None = None,
    *,
    activation: str = "none",
    residual: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
    save_preact: str | None = None,
):
    """``act(x @ weight.T + bias) + residual`` in one pass, products and sums in fp32.

    ``x`` ``[T, K]``, ``weight`` ``[N, K]`` (``nn.Linear`` layout), ``bias`` ``[N]``,
    ``residual`` ``[T, N]``, all float16 or all bfloat16; ``activation`` one of
    ``ACTIVATIONS``. ``save_preact="full"`` also returns the pre-activation
    ``x @ weight.T + bias`` as a ``[T, N]`` tensor, ``"packed"`` as a
    ``PackedActivation``: ``(out, preact)``. ``out`` and ``residual`` may be strided
    rows; ``out`` may be ``residual`` itself (added in place), and shares no memory with
    the other inputs.
    """
    _check_rows("x", x, _LINEAR_DT)
    T, K = x.shape
    dev, dt = x.device, x.dtype
    act = _act_code(activation)
    _check_weight(weight, K, dt, dev)
    N = weight.shape[0]
    if bias is not None:
        if bias.shape != (N,) or bias.dtype != dt or bias.device != dev:
            raise ValueError(f"bias must be [{N}] {dt} on {dev}, got {tuple(bias.shape)} {bias.dtype} on {bias.device}")
        bias = bias.contiguous()
    if residual is not None:
        if residual.shape != (T, N) or residual.dtype != dt or residual.device != dev:
            raise ValueError(f"residual must be [{T}, {N}] {dt} on {dev}, got {tuple(residual.shape)} "
                             f"{residual.dtype} on {residual.device}")
        residual = _rows(residual)
    if save_preact not in (None, "none", "full", "packed"):
        raise ValueError(f"save_preact must be None, 'full' or 'packed', got {save_preact!r}")
    given = out is not None
    if not given:
        out, out_stride = torch.empty((T, N), dtype=dt, device=dev), N
    else:
        out = _check_out_rows(out, (T, N), x)
        out_stride = _stride(out)
    z = p = None
    if save_preact == "full":
        z = torch.empty(T, N, dtype=dt, device=dev)
    elif save_preact == "packed":
        p = _empty_packed(T, N, dt, dev)
    if T > 0:
        x, xs = _rows16(x)
        weight, ws_ = _rows16(weight)
        if given:
            _check_apart(out, "residual", x=x, weight=weight, bias=bias, residual=residual)
        nbytes = _workspace_bytes(_lib.workspace_bytes_linear_act, dev, T, K, N)
        ws = _workspace(nbytes, dev) if nbytes else None
        _call("frattn_linear_act", dev, x.data_ptr(), xs, weight.data_ptr(), ws_, _ptr(bias), _ptr(residual),
              0 if residual is None else _stride(residual), act, T, K, N, _DT[dt], out.data_ptr(), out_stride, _ptr(z), N, p.codes.data_ptr() if p is not None else None,
              p.scales.data_ptr() if p is not None else None, _ptr(ws), nbytes, _status_word(dev).data_ptr())
    if given:
        _written(out)
    if save_preact in (None, "none"):
        return out
    return out, (z if p is None else p)


def linear_act_backward(
    dout: torch.Tensor,
    x: torch.Tensor | PackedActivation,
    weight: torch.Tensor,
    preact: torch.Tensor | PackedActivation | None = None,
    *,
    activation: str = "none",
    need: tuple[bool, bool, bool] = (True, True, True),
):
    """``(dx, dweight, dbias)`` of ``linear_act`` for the output gradient ``dout`` ``[T, N]``.

    With ``dz = dout * act'(preact)``: ``dx = dz @ weight``, ``dweight = dz.T @ x``,
    ``dbias = dz.sum(0)``, in x's type. ``x`` and ``preact`` (what ``save_preact``
    returned; unused for activation "none") may be checkpoints. ``need`` says which
    of the three are wanted; the others come as None. The residual's gradient is
    ``dout``.
    """
    _check_rows("dout", dout, _LINEAR_DT)
    T, N = dout.shape
    dev, dt = dout.device, dout.dtype
    act = _act_code(activation)
    if weight.ndim != 2 or weight.shape[0] != N or weight.shape[1] <= 0:
        raise ValueError(f"weight must be [{N}, K], got {tuple(weight.shape)}")
    K = weight.shape[1]
    _check_weight(weight, K, dt, dev)
    xp, zp = isinstance(x, PackedActivation), isinstance(preact, PackedActivation)
    if xp:
        _check_packed("x", x, dt, (T, K))
    else:
        _check_rows("x", x, _LINEAR_DT)
        if x.shape != (T, K) or x.dtype != dt:
            raise ValueError(f"x must be [{T}, {K}] {dt}, got {tuple(x.shape)} {x.dtype}")
    if x.device != dev:
        raise ValueError(f"x must be on {dev}, got {x.device}")
    if act:
        if preact is None:
            raise ValueError(f"preact is needed for activation {activation!r}")
        if zp:
            _check_packed("preact", preact, dt, (T, N))
        else:
            _check_rows("preact", preact, _LINEAR_DT)
            if preact.shape != (T, N) or preact.dtype != dt:
                raise ValueError(f"preact must be [{T}, {N}] {dt}, got {tuple(preact.shape)} {preact.dtype}")
            preact = _rows(preact)
        if preact.device != dev:
            raise ValueError(f"preact must be on {dev}, got {preact.device}")
    else:
        preact, zp = None, False
    dout = _rows(dout)
    need_x, need_w, need_b = need
    dx = torch.empty(T, K, dtype=dt, device=dev) if need_x else None
    dw = torch.empty(N, K, dtype=dt, device=dev) if need_w else None
    db = torch.empty(N, dtype=dt, device=dev) if need_b else None
    if not (need_x or need_w or need_b):
        return dx, dw, db
    xs, ws_ = K, K
    if not xp:
        x, xs = _rows16(x) if need_w else (x, max(_stride(x), K))
    if need_x:
        weight, ws_ = _rows16(weight)
    nbytes = _workspace_bytes(_lib.workspace_bytes_linear_act_bwd, dev, T, K, N)
    ws = _workspace(nbytes, dev)
    _call("frattn_linear_act_bwd", dev, dout.data_ptr(), _stride(dout), None if xp else x.data_ptr(),
          0 if xp else xs, x.codes.data_ptr() if xp else None, x.scales.data_ptr() if xp else None,
          weight.data_ptr(), ws_, None if preact is None or zp else preact.data_ptr(),
          0 if preact is None or zp else _stride(preact), preact.codes.data_ptr() if zp else None,
          preact.scales.data_ptr() if zp else None, act, T, K, N, _DT[dt], _ptr(dx), K, _ptr(dw), _ptr(db),
          ws.data_ptr(), nbytes, _status_word(dev).data_ptr())
    return dx, dw, db


class _LinearAct(torch.autograd.Function):
    """Autograd node of ``linear_act``; x and the pre-activation are kept as they are
    or as checkpoints."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation, checkpoint):
        save = None if activation == "none" else "packed" if checkpoint else "full"
        T, N = x.shape[0], weight.shape[0]
        # rows of whole 16 bytes, so that a following linear layer reads them in place
        out = x.new_empty(T, -(-N // 8) * 8)[:, :N] if N % 8 and x.ndim == 2 else None
        got = linear_act(x, weight, bias, activation=activation, residual=residual, out=out, save_preact=save)
        out, z = got if save else (got, None)
        ctx.activation, ctx.packed = activation, checkpoint
        ctx.has_bias, ctx.has_res = bias is not None, residual is not None
        if checkpoint:
            p = pack_activation(x)
            ctx.meta = (p.width, z.width if z is not None else 0, x.dtype)
            ctx.save_for_backward(weight, p.codes, p.scales, *((z.codes, z.scales) if z is not None else ()))
        else:
            ctx.save_for_backward(weight, x, *((z,) if z is not None else ()))
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        weight, *kept = ctx.saved_tensors
        if ctx.packed:
            kx, kz, dt = ctx.meta
            x = PackedActivation(kept[0], kept[1], kx, dt)
            z = PackedActivation(kept[2], kept[3], kz, dt) if kz else None
        else:
            x, z = kept[0], kept[1] if len(kept) > 1 else None
        need = ctx.needs_input_grad
        dx, dw, db = linear_act_backward(dout, x, weight, z, activation=ctx.activation,
                                         need=(need[0], need[1], ctx.has_bias and need[2]))
        return dx, dw, db, dout if ctx.has_res and need[3] else None, None, None


def linear_act_train(x, weight, bias=None, *, activation: str = "none", residual=None,
                     checkpoint: bool = False) -> torch.Tensor:
    """``linear_act`` with gradients for x, weight, bias and residual, once
    differentiable (a second derivative through it raises). With ``checkpoint`` the node
    keeps x and the pre-activation in 8 bits, and the gradients are those at the values
    so kept."""
    return _LinearAct.apply(x, weight, bias, residual, activation, checkpoint)
