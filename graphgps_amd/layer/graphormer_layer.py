"""GraphormerLayer on the varlen attention kernel with its additive-bias operand.

Drop-in for ``/root/reference/graphgps/layer/graphormer_layer.py:5-49`` (same constructor, same
parameter names: ``attention.*`` of a ``torch.nn.MultiheadAttention``, ``input_norm.*``, ``mlp.{0,1,4}.*``).
The reference pads with ``to_dense_batch``, runs the dense MHA with ``attn_mask=data.attn_bias`` and a key
padding mask and un-pads with a boolean index (:41-46); here the packed in-projection output goes straight
to ``csrc/seg_attention.hip`` with the dense ``[B*H, nmax, nmax]`` bias read in place.  LayerNorm, GELU and
the two d x d MLP GEMMs are library ops.

``sandwich=True`` (``graphormer.sandwich``; not in the reference) also normalises what each half adds to the stream and scales it
with a learned gate per channel, ``x <- x + gate o LayerNorm(half(LayerNorm(x)))``: the norm behind a half, its gate, the
residual addition and the norm in front of the next half are one pass over the rows (``ops.sandwich_norm``).
"""
import torch

from ..fused import linear
from ..ops import graph_index_of, sandwich_norm, segment_attention


class GraphormerLayer(torch.nn.Module):
    def __init__(self, embed_dim: int, num_heads: int, dropout: float,
                 attention_dropout: float, mlp_dropout: float, sandwich: bool = False):
        super().__init__()
        self.ctor_kwargs = dict(embed_dim=embed_dim, num_heads=num_heads, dropout=dropout,
                                attention_dropout=attention_dropout, mlp_dropout=mlp_dropout)
        # parameter container (names / init of the reference's module); its dense forward is never called
        self.attention = torch.nn.MultiheadAttention(embed_dim, num_heads, attention_dropout,
                                                     batch_first=True)
        self.num_heads = num_heads
        self.attention_dropout = attention_dropout
        self.input_norm = torch.nn.LayerNorm(embed_dim)
        self.dropout = torch.nn.Dropout(dropout)
        self.mlp = torch.nn.Sequential(
            torch.nn.LayerNorm(embed_dim),
            torch.nn.Linear(embed_dim, embed_dim),
            torch.nn.GELU(),
            torch.nn.Dropout(mlp_dropout),
            torch.nn.Linear(embed_dim, embed_dim),
            torch.nn.Dropout(dropout),
        )
        self.sandwich = bool(sandwich)
        if self.sandwich:
            self.ctor_kwargs["sandwich"] = True
            self.attention_post_norm = torch.nn.LayerNorm(embed_dim)
            self.mlp_post_norm = torch.nn.LayerNorm(embed_dim)
            self.attention_gate = torch.nn.Parameter(torch.ones(embed_dim))
            self.mlp_gate = torch.nn.Parameter(torch.ones(embed_dim))

    def forward(self, data):
        gi = graph_index_of(data)
        att = self.attention
        if self.sandwich:
            return self._forward_sandwich(data, gi)
        x = self.input_norm(data.x)                                              # reference :40
        qkv = linear(x, att.in_proj_weight, att.in_proj_bias)
        p = self.attention_dropout if self.training else 0.0
        o = segment_attention(qkv, gi, self.num_heads, p, bias=getattr(data, "attn_bias", None))  # :43-46
        x = linear(o, att.out_proj.weight, att.out_proj.bias)
        x = self.dropout(x) + data.x                                             # :47
        data.x = self.mlp(x) + x                                                 # :48
        return data

    def _forward_sandwich(self, data, gi):
        att, mlp = self.attention, self.mlp
        first, post_a, pre_m, post_m = self.input_norm, self.attention_post_norm, mlp[0], self.mlp_post_norm
        x, _ = sandwich_norm(None, data.x, post_weight=first.weight, post_bias=first.bias, kind="layer", eps=first.eps)
        qkv = linear(x, att.in_proj_weight, att.in_proj_bias)
        p = self.attention_dropout if self.training else 0.0
        o = segment_attention(qkv, gi, self.num_heads, p, bias=getattr(data, "attn_bias", None))
        o = self.dropout(linear(o, att.out_proj.weight, att.out_proj.bias))
        x, z = sandwich_norm(data.x, o, post_weight=post_a.weight, post_bias=post_a.bias, pre_weight=pre_m.weight,
                             pre_bias=pre_m.bias, gate=self.attention_gate, kind="layer", eps=first.eps)
        data.x, _ = sandwich_norm(x, mlp[1:](z), post_weight=post_m.weight, post_bias=post_m.bias, gate=self.mlp_gate, kind="layer",
                                  eps=first.eps)
        return data
