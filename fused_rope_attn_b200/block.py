"""A transformer block that is trained and served on this package's kernels.

Pre-norm block around the fused RoPE attention: layer norm, QKV projection,
attention, output projection with the residual added in its epilogue, layer norm, and
a two-matrix MLP with the activation and the residual in the epilogues. The
reference (sdan/fused-rope-attn) has the attention alone (fused_attn.py:139-232).

With gradients enabled every step records an autograd node whose backward pass is
this package's (``layer_norm_train``, ``linear_act_train``,
``fused_rope_attention_train``); ``checkpoint=True`` keeps the norms' and the linear
layers' inputs and pre-activations for it in 8 bits. Without gradients the rotation
moves into the QKV projection (``qkv_rope_projection``).
"""
from __future__ import annotations

import torch

from .block_ops import layer_norm, layer_norm_train, linear_act, linear_act_train
from .fused_attn import (QKV_ROPE_HEAD_DIMS, fused_attention_rotated, fused_rope_attention, fused_rope_attention_train,
                         qkv_rope_projection)

__all__ = ["EncoderBlock"]


class EncoderBlock(torch.nn.Module):
    """Pre-norm block of ``heads`` heads of ``head_dim`` and an MLP of width ``mlp``.

    Norm parameters are kept in float32, the matrices in ``dtype`` with rows padded to
    16 bytes (a width such as 3420 then costs no copies)."""

    def __init__(self, hidden: int = 1280, heads: int = 16, head_dim: int = 80, mlp: int = 3420, *,
                 activation: str = "gelu", eps: float = 1e-6, checkpoint: bool = False, init_std: float = 0.02,
                 seed: int = 0, device="cuda", dtype=torch.bfloat16):
        super().__init__()
        self.heads, self.head_dim, self.mlp = heads, head_dim, mlp
        self.activation, self.eps, self.checkpoint = activation, eps, checkpoint
        g = torch.Generator().manual_seed(seed)
        inner = heads * head_dim

        def matrix(n, k):
            rows = torch.zeros(n, -(-k // 8) * 8, dtype=dtype, device=device)
            rows[:, :k] = (torch.randn(n, k, generator=g) * init_std).to(device=device, dtype=dtype)
            return torch.nn.Parameter(rows[:, :k])

        def vector(n, value=0.0, dt=dtype):
            return torch.nn.Parameter(torch.full((n,), value, dtype=dt, device=device))

        self.norm1_w, self.norm1_b = vector(hidden, 1.0, torch.float32), vector(hidden, 0.0, torch.float32)
        self.qkv_w, self.qkv_b = matrix(3 * inner, hidden), vector(3 * inner)
        self.proj_w, self.proj_b = matrix(hidden, inner), vector(hidden)
        self.norm2_w, self.norm2_b = vector(hidden, 1.0, torch.float32), vector(hidden, 0.0, torch.float32)
        self.fc1_w, self.fc1_b = matrix(mlp, hidden), vector(mlp)
        self.fc2_w, self.fc2_b = matrix(hidden, mlp), vector(hidden)

    def forward(self, x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, cu_seqlens: torch.Tensor, *,
                max_seqlen: int | None = None) -> torch.Tensor:
        """``x`` ``[T, hidden]``; ``cos``, ``sin``, ``cu_seqlens`` and ``max_seqlen`` as for
        ``fused_rope_attention``."""
        if torch.is_grad_enabled() and (x.requires_grad or any(p.requires_grad for p in self.parameters())):
            return self._train(x, cos, sin, cu_seqlens, max_seqlen)
        return self._infer(x, cos, sin, cu_seqlens, max_seqlen)

    def _train(self, x, cos, sin, cu, max_seqlen):
        T, ck = x.shape[0], self.checkpoint
        h = layer_norm_train(x, self.norm1_w, self.norm1_b, eps=self.eps, checkpoint=ck)
        qkv = linear_act_train(h, self.qkv_w, self.qkv_b, checkpoint=ck)
        q, k, v = qkv.view(T, 3, self.heads, self.head_dim).unbind(1)
        o = fused_rope_attention_train(q, k, v, cos, sin, cu, max_seqlen=max_seqlen)
        x = linear_act_train(o.reshape(T, -1), self.proj_w, self.proj_b, residual=x, checkpoint=ck)
        h = layer_norm_train(x, self.norm2_w, self.norm2_b, eps=self.eps, checkpoint=ck)
        h = linear_act_train(h, self.fc1_w, self.fc1_b, activation=self.activation, checkpoint=ck)
        return linear_act_train(h, self.fc2_w, self.fc2_b, residual=x, checkpoint=ck)

    def _infer(self, x, cos, sin, cu, max_seqlen):
        T = x.shape[0]
        h = layer_norm(x, self.norm1_w, self.norm1_b, eps=self.eps)
        if self.head_dim in QKV_ROPE_HEAD_DIMS and self.qkv_w.shape[1] % 8 == 0:
            qkv = qkv_rope_projection(h, self.qkv_w, self.qkv_b, cos, sin, self.heads)
            o = fused_attention_rotated(qkv[:, 0], qkv[:, 1], qkv[:, 2], cu, max_seqlen=max_seqlen)
        else:
            q, k, v = linear_act(h, self.qkv_w, self.qkv_b).view(T, 3, self.heads, self.head_dim).unbind(1)
            o = fused_rope_attention(q, k, v, cos, sin, cu, max_seqlen=max_seqlen)
        x = linear_act(o.reshape(T, -1), self.proj_w, self.proj_b, residual=x)
        h = layer_norm(x, self.norm2_w, self.norm2_b, eps=self.eps)
        hidden = x.new_empty(T, -(-self.mlp // 8) * 8)[:, :self.mlp]
        linear_act(h, self.fc1_w, self.fc1_b, activation=self.activation, out=hidden)
        return linear_act(hidden, self.fc2_w, self.fc2_b, residual=x)
