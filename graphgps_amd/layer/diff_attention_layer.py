"""Differential self-attention over the graphs of a batch: ``GPSLayer``'s ``global_model_type='DiffTransformer'``.

Two softmax maps per head, the second subtracted with a learned weight, share one value; every head's output passes an RMS norm
before the output projection:

    q, k, v = x W_qkv;   o_h = (softmax(q1 k1^T / sqrt d) - lam_h softmax(q2 k2^T / sqrt d)) v_h
    y = concat_h((1 - lam0) rmsnorm(o_h)) W_out;   lam_h = exp(a1_h . b1_h) - exp(a2_h . b2_h) + lam0

``lam0 = 0.8 - 0.6 exp(-0.3 depth)``, ``depth`` = the layer's index in its stack (0 for the first).  The attention is
``ops.diff_segment_attention`` (csrc/diff_attn.hip), the head norm ``ops.sandwich_norm`` (csrc/sandwich.hip); both run on the
``ptr`` segments, nothing is padded.
"""
import math

import torch
import torch.nn as nn

from ..fused import linear
from ..ops import diff_segment_attention, sandwich_norm


class DiffSelfAttention(nn.Module):
    """``dim`` columns in ``heads`` heads of ``dim / heads`` value columns (half of it per score map: a multiple of 8, up to
    128); ``kv_heads`` of them have keys and values of their own."""

    def __init__(self, dim, heads, kv_heads=None, depth=0, eps=1e-5):
        super().__init__()
        kv_heads = heads if kv_heads is None else kv_heads
        if dim % heads or dim // heads % 16 or dim // heads > 256 or heads % kv_heads:
            raise ValueError(f"DiffSelfAttention: {dim} columns in {heads} heads over {kv_heads} key heads: a head needs a multiple "
                             f"of 16 columns, at most 256, and heads a multiple of key heads")
        self.heads, self.kv_heads, self.dim_map, self.eps = heads, kv_heads, dim // heads // 2, eps
        self.to_qkv = nn.Linear(dim, 2 * heads * self.dim_map + 4 * kv_heads * self.dim_map)
        self.to_out = nn.Linear(dim, dim)
        # one row each of a1, b1, a2, b2 per head
        self.lam_vectors = nn.Parameter(torch.randn(4, heads, self.dim_map) * 0.1)
        self.head_norm = nn.Parameter(torch.ones(2 * self.dim_map))
        self.set_depth(depth)

    def set_depth(self, depth):
        self.depth = int(depth)
        self.lam0 = 0.8 - 0.6 * math.exp(-0.3 * self.depth)

    def lam(self):
        a1, b1, a2, b2 = self.lam_vectors
        return torch.exp((a1 * b1).sum(-1)) - torch.exp((a2 * b2).sum(-1)) + self.lam0

    def forward_segments(self, x, gi):
        """[N, dim] node features + graph index -> [N, dim]."""
        qkv = linear(x, self.to_qkv.weight, self.to_qkv.bias)
        o = diff_segment_attention(qkv, self.lam(), gi, self.heads, self.kv_heads)
        o, _ = sandwich_norm(None, o, post_weight=self.head_norm, branch_scale=1.0 - self.lam0, kind="rms", eps=self.eps)
        return linear(o.view(x.shape[0], -1), self.to_out.weight, self.to_out.bias)

    def forward(self, x, mask=None, **kwargs):
        raise NotImplementedError("DiffSelfAttention works on ptr segments: call forward_segments(x, graph_index) (GPSLayer does)")

    def extra_repr(self):
        return f'heads={self.heads}, kv_heads={self.kv_heads}, dim_map={self.dim_map}, depth={self.depth}'
