"""EncoderBlock at a vision tower's size (1280 wide, 16 heads of 80, MLP 3420): products on CTA
pairs and norms through their rings, forward, gradients and checkpoints.

Bounds in the 2-norm as for the small blocks: 0.03 leaves room over some sixteen 16-bit
roundings of 0.42 x 2^-8 each, 0.05 over six 8-bit steps of 0.7 % besides."""
import pytest
import torch

from fused_rope_attn_b200 import last_status
from fused_rope_attn_b200.encoder import rel_l2
from test_gpu_block import DEV, inputs, make, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("checkpoint", [False, True])
def test_block_of_a_vision_tower(checkpoint):
    blk = make(1280, 16, 80, 3420, checkpoint)
    x, cos, sin, cu = inputs([(1, 40, 44), (1, 24, 32)], 1280, 80, True, seed=3)
    p = {n: t.detach().float().requires_grad_(True) for n, t in blk.named_parameters()}
    xr = x.float().requires_grad_(True)
    ref = reference(blk, p, xr, cos, sin, cu)
    with torch.no_grad():
        assert rel_l2(blk(x, cos, sin, cu, max_seqlen=64), ref.detach()) < 0.03
    x.requires_grad_(True)
    y = blk(x, cos, sin, cu, max_seqlen=64)
    assert rel_l2(y.detach(), ref.detach()) < 0.03
    dy = torch.randn(x.shape, generator=torch.Generator().manual_seed(4)).to(DEV, torch.bfloat16)
    y.backward(dy)
    ref.backward(dy.float())
    bound = 0.05 if checkpoint else 0.03
    assert rel_l2(x.grad, xr.grad) < bound
    for n, t in blk.named_parameters():
        if n != "qkv_b":  # (a third of it, the keys' bias, has no gradient but rounding)
            assert rel_l2(t.grad, p[n].grad) < bound, n
    assert last_status(DEV) == 0
