"""EncoderBlock: the norm, linear and attention operators together, against fp32 torch.

Tolerances, in the 2-norm. Eight 16-bit roundings of 0.42 u lie on the way to the
output and about twice as many on the way to a gradient (u = 2^-8): 0.42 u sqrt(16) is
below 0.01, and 0.03 leaves room for the attention's 16-bit probabilities. An 8-bit checkpoint
has steps of 2^-7 to 2^-6 of its block's largest value, for normal values about 2.1
times their spread: an error of 0.7 % of the spread a tensor, and a gradient depends on
up to six of them: 0.05."""
import pytest
import torch

from fused_rope_attn_b200 import EncoderBlock, compute_rope_2d, last_status
from fused_rope_attn_b200.encoder import rel_l2, rope_unfused
from fused_rope_attn_b200.utils import get_window_index, segments_per_image

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def inputs(grid, hidden, head_dim, window, seed=0):
    widx, cu = get_window_index(grid)
    cos, sin = compute_rope_2d(grid, head_dim, 2, 10000.0, DEV, torch.float32, window_idx=widx)
    if not window:
        cu = segments_per_image(grid)
    g = torch.Generator().manual_seed(seed)
    return torch.randn(cos.shape[0], hidden, generator=g).to(DEV, torch.bfloat16), cos, sin, cu.to(DEV)


def reference(blk, p, x, cos, sin, cu):
    """The block in fp32 torch operations on fp32 copies p of its parameters."""
    F = torch.nn.functional
    T = x.shape[0]
    h = F.layer_norm(x, (x.shape[1],), p["norm1_w"], p["norm1_b"], blk.eps)
    q, k, v = F.linear(h, p["qkv_w"], p["qkv_b"]).view(T, 3, blk.heads, blk.head_dim).unbind(1)
    q, k = rope_unfused(q, cos, sin), rope_unfused(k, cos, sin)
    o = []
    for a, b in zip(cu[:-1].tolist(), cu[1:].tolist()):
        s = torch.einsum("qhd,khd->hqk", q[a:b], k[a:b]) * blk.head_dim ** -0.5
        o.append(torch.einsum("hqk,khd->qhd", s.softmax(-1), v[a:b]))
    x = x + F.linear(torch.cat(o).reshape(T, -1), p["proj_w"], p["proj_b"])
    h = F.layer_norm(x, (x.shape[1],), p["norm2_w"], p["norm2_b"], blk.eps)
    h = F.gelu(F.linear(h, p["fc1_w"], p["fc1_b"]))
    return x + F.linear(h, p["fc2_w"], p["fc2_b"])


def make(hidden, heads, hd, mlp, checkpoint=False):
    blk = EncoderBlock(hidden, heads, hd, mlp, checkpoint=checkpoint, init_std=hidden ** -0.5, device=DEV)
    g = torch.Generator().manual_seed(5)
    with torch.no_grad():
        for n, p in blk.named_parameters():
            if n.endswith("_b"):
                p.copy_(torch.randn(p.shape, generator=g) * 0.1)
    return blk


SHAPES = [([(1, 16, 16)], 160, 2, 80, 428, True), ([(1, 12, 20), (1, 8, 8)], 256, 4, 64, 340, False)]


@pytest.mark.parametrize("grid,hidden,heads,hd,mlp,window", SHAPES)
def test_block_forward(grid, hidden, heads, hd, mlp, window):
    blk = make(hidden, heads, hd, mlp)
    x, cos, sin, cu = inputs(grid, hidden, hd, window)
    p = {n: t.detach().float() for n, t in blk.named_parameters()}
    ref = reference(blk, p, x.float(), cos, sin, cu)
    with torch.no_grad():
        y = blk(x, cos, sin, cu, max_seqlen=64 if window else None)
    assert y.shape == x.shape and rel_l2(y, ref) < 0.03
    yt = blk(x, cos, sin, cu, max_seqlen=64 if window else None)
    assert yt.requires_grad and rel_l2(yt, ref) < 0.03
    assert last_status(DEV) == 0


@pytest.mark.parametrize("checkpoint", [False, True])
@pytest.mark.parametrize("grid,hidden,heads,hd,mlp,window", SHAPES)
def test_block_gradients(grid, hidden, heads, hd, mlp, window, checkpoint):
    blk = make(hidden, heads, hd, mlp, checkpoint)
    x, cos, sin, cu = inputs(grid, hidden, hd, window, seed=1)
    dy = torch.randn(x.shape, generator=torch.Generator().manual_seed(2)).to(DEV, torch.bfloat16)
    x.requires_grad_(True)
    blk(x, cos, sin, cu).backward(dy)
    p = {n: t.detach().float().requires_grad_(True) for n, t in blk.named_parameters()}
    xr = x.detach().float().requires_grad_(True)
    reference(blk, p, xr, cos, sin, cu).backward(dy.float())
    bound = 0.05 if checkpoint else 0.03
    assert rel_l2(x.grad, xr.grad) < bound
    for n, t in blk.named_parameters():
        assert t.grad is not None and t.grad.dtype == t.dtype
        if n == "qkv_b":  # the keys' bias moves no score difference: its gradient is 0 but for rounding
            third = t.numel() // 3
            keep = [0, 2]
            for i in keep:
                sl = slice(i * third, (i + 1) * third)
                assert rel_l2(t.grad[sl], p[n].grad[sl]) < bound, n
        else:
            assert rel_l2(t.grad, p[n].grad) < bound, n
    assert last_status(DEV) == 0


def test_block_learns_and_checkpoints_use_less_memory():
    grid = [(1, 32, 32)]
    peak = {}
    for checkpoint in (False, True):
        blk = EncoderBlock(320, 4, 80, 856, checkpoint=checkpoint, device=DEV)
        x, cos, sin, cu = inputs(grid, 320, 80, True)
        target = torch.randn(x.shape, generator=torch.Generator().manual_seed(9)).to(DEV, torch.bfloat16)
        opt = torch.optim.SGD(blk.parameters(), lr=0.05)
        losses = []
        for _ in range(8):
            opt.zero_grad()
            torch.cuda.synchronize()
            torch.cuda.reset_peak_memory_stats()
            base = torch.cuda.memory_allocated()
            y = blk(x, cos, sin, cu, max_seqlen=64)
            peak[checkpoint] = torch.cuda.memory_allocated() - base
            loss = (y.float() - target.float()).square().sum() / x.shape[0]
            loss.backward()
            torch.nn.utils.clip_grad_norm_(blk.parameters(), 1.0)
            opt.step()
            losses.append(float(loss.detach()))
        assert losses[-1] < losses[0]
    # kept either way: q, k, v, the attention's output and the residual stream
    assert peak[True] < 0.85 * peak[False]
