"""Outputs that the caller provides: which may share memory with an input. The check is on
addresses alone, so it is tested on the CPU against the addresses themselves."""
import random

import pytest
import torch

from fused_rope_attn_b200 import block_ops as ops


def bytes_of(t):
    """Every byte address that t's elements have."""
    e = t.element_size()
    at = [0]
    for n, s in zip(t.shape, t.stride()):
        at = [a + i * s * e for a in at for i in range(n)]
    return {t.data_ptr() + a + b for a in at for b in range(e)}


def test_apart_against_the_addresses():
    """Random views of one buffer: views that meet are never called apart, and those whose
    ranges of addresses are separate always are."""
    rng = random.Random(0)
    buf = torch.zeros(4096, dtype=torch.bfloat16)
    said = {True: 0, False: 0}
    for _ in range(4000):
        views = []
        for _ in range(2):
            rows, cols = rng.randint(1, 6), rng.randint(1, 24)
            stride = max(cols, rng.choice([cols, 24, 32, 40]))
            views.append(buf.as_strided((rows, cols), (stride, 1), rng.randint(0, 220)))
        out, t = views
        if rng.random() < 0.2:
            t = t[0]  # a vector
        a, b = bytes_of(out), bytes_of(t)
        apart = ops._apart(out, t)
        assert not (apart and a & b)
        assert apart or max(a) >= min(b) and max(b) >= min(a)
        said[apart] += 1
    assert min(said.values()) > 500


def test_columns_of_one_buffer_are_apart():
    buf = torch.zeros(9, 64)
    assert ops._apart(buf[:, :24], buf[:, 24:]) and ops._apart(buf[:, 24:], buf[:, :24])
    assert ops._apart(buf[:, 8:16], buf[:, 40:]) and ops._apart(buf[1:, :8], buf[:-1, 8:16])
    assert not ops._apart(buf[:, :24], buf[:, 23:]) and not ops._apart(buf[:, 32:], buf[1:, :33])
    half = buf.view(torch.bfloat16)  # the same rows as 128 values of 2 bytes
    assert ops._apart(buf[:, :24], half[:, 48:]) and not ops._apart(buf[:, :24], half[:, 47:])


def test_refusals_and_the_input_that_may_be_out_itself():
    buf = torch.zeros(10, 64)
    out = buf[:8]
    ops._check_apart(out, "residual", x=torch.zeros(8, 64), residual=out, bias=None)
    ops._check_apart(out, "residual", residual=buf[:8])
    ops._check_apart(buf[:1], "residual", residual=buf[:1].as_strided((1, 64), (7, 1)))  # one row: no stride
    for bad in (buf[1:9], buf[:8, 1:], buf[:8].as_strided((8, 64), (32, 1))):
        with pytest.raises(ValueError, match="residual itself or not share"):
            ops._check_apart(out, "residual", residual=bad)
    for name in ("x", "weight", "bias"):
        with pytest.raises(ValueError, match=f"share memory with {name}"):
            ops._check_apart(out, "residual", **{name: out})
