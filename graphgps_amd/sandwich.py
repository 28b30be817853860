"""The residual stream of a block in one pass over its rows (csrc/sandwich.hip).

    y = residual_scale * x + branch_scale * gate * norm(a; post)          z = norm(y; pre)

``x`` is the stream, ``a`` what a block adds to it, ``y`` the new stream and ``z`` the next block's input.  Reached as
``graphgps_amd.ops.sandwich_norm``; ``layer.GraphormerLayer`` (its ``sandwich`` form) and ``layer.DiffSelfAttention`` (its head
norm) call it.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

from . import lib as _lib
from .diff_attention import DTYPES, where
from .lib import SandwichNorm, check, current_stream, on_device, ptr

KINDS = {"rms": 0, "layer": 1}                    # GPS_NORM_RMS, GPS_NORM_LAYER


def _fail(msg: str):
    raise _lib.GpsHipError(msg)


def _rows(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """``[..., D]`` -> ``[N, D]``, contiguous within a row."""
    if t is None:
        return None
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    return t if t.shape[-1] == 1 or t.stride(1) == 1 else t.contiguous()


def _block(x, a, w, gate, full: bool, stats, kind, alpha, beta, eps) -> SandwichNorm:
    return SandwichNorm(a=a.data_ptr(), x=ptr(x), gate_full=ptr(gate) if full else None, gate=None if full else ptr(gate),
                        a_rs=a.stride(0), x_rs=x.stride(0) if x is not None else 0, g_rs=gate.stride(0) if full else 0,
                        post_weight=ptr(w[0]), post_bias=ptr(w[1]), pre_weight=ptr(w[2]), pre_bias=ptr(w[3]), N=a.shape[0],
                        D=a.shape[1], kind=kind, dtype=DTYPES[a.dtype], alpha=alpha, beta=beta, eps=eps, stats=ptr(stats))


class _Sandwich(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, a, post_weight, post_bias, pre_weight, pre_bias, gate, alpha, beta, kind, eps, train):
        dev = a.device
        x2, a2 = _rows(x), _rows(a)
        full = gate is not None and gate.dim() > 1
        g2 = _rows(gate) if full else (None if gate is None else gate.contiguous())
        w = [None if t is None else t.contiguous() for t in (post_weight, post_bias, pre_weight, pre_bias)]
        n, d = a2.shape
        y = torch.empty_like(a, memory_format=torch.contiguous_format)
        z = torch.empty_like(y) if pre_weight is not None else None
        stats = torch.empty(4, n, dtype=torch.float32, device=dev) if train and (post_weight is not None or pre_weight is not None) else None
        b = _block(x2, a2, w, g2, full, stats, kind, alpha, beta, eps)
        b.y, b.z = y.data_ptr(), ptr(z)
        with on_device(dev):
            check(_lib.load().gps_sandwich_norm_fwd(ctypes.addressof(b), current_stream(dev)), "gps_sandwich_norm_fwd")
        if train:
            ctx.set_materialize_grads(False)
            ctx.save_for_backward(x2, a2, *w, g2, stats)
            ctx.block, ctx.at, ctx.shape, ctx.full = b, where(x2, a2, *w, g2, stats), a.shape, full
        return y, z

    @staticmethod
    def backward(ctx, dy, dz):
        if torch.is_grad_enabled():
            _fail("sandwich_norm is differentiable once: its backward has no gradient of its own")
        if dy is None and dz is None:
            return (None,) * 12
        saved = x, a, w1, b1, w2, b2, gate, stats = ctx.saved_tensors
        dev, L, need, full = a.device, _lib.load(), ctx.needs_input_grad, ctx.full
        dy, dz = _rows(dy), _rows(dz)
        for t in (dy, dz):
            if t is not None and t.dtype != a.dtype:
                _fail(f"sandwich_norm: gradient of type {t.dtype} for an output of type {a.dtype}")
        b = SandwichNorm.from_buffer_copy(ctx.block)
        if where(*saved) != ctx.at:
            b = _block(x, a, (w1, b1, w2, b2), gate, full, stats, b.kind, b.alpha, b.beta, b.eps)
        n, d = b.N, b.D
        dx = torch.empty_like(x, memory_format=torch.contiguous_format) if need[0] else None
        da = torch.empty_like(a, memory_format=torch.contiguous_format)
        dw = [torch.empty_like(t) if need[i] else None for i, t in ((2, w1), (3, b1), (4, w2), (5, b2))]
        dg = torch.empty_like(gate, memory_format=torch.contiguous_format) if need[6] else None
        b.ws_floats = L.gps_sandwich_workspace_floats(n, d)
        ws = torch.empty(b.ws_floats, dtype=torch.float32, device=dev)
        b.ws, b.dx, b.da = ws.data_ptr(), ptr(dx), da.data_ptr()
        if dy is not None:
            b.dy, b.dy_rs = dy.data_ptr(), dy.stride(0)
        if dz is not None:
            b.dz, b.dz_rs = dz.data_ptr(), dz.stride(0)
        b.dpost_weight, b.dpost_bias, b.dpre_weight, b.dpre_bias = [ptr(t) for t in dw]
        if full:
            b.dgate_full = ptr(dg)
        else:
            b.dgate = ptr(dg)
        with on_device(dev):
            check(L.gps_sandwich_norm_bwd(ctypes.addressof(b), current_stream(dev)), "gps_sandwich_norm_bwd")
        if len(ctx.shape) != 2:
            dx, da = (None if t is None else t.view(ctx.shape) for t in (dx, da))
            dg = dg.view(ctx.shape) if full and dg is not None else dg
        return (dx, da, *dw, dg, None, None, None, None, None)


def sandwich_norm(x: Optional[torch.Tensor], a: torch.Tensor, *, post_weight: Optional[torch.Tensor] = None,
                  post_bias: Optional[torch.Tensor] = None, pre_weight: Optional[torch.Tensor] = None,
                  pre_bias: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None, residual_scale: float = 1.0,
                  branch_scale: float = 1.0, kind: str = "rms", eps: float = 1e-5) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """``y = residual_scale x + branch_scale gate norm(a)`` and ``z = norm(y)`` -> ``(y, z)``.

    ``a`` and ``x [..., D]`` share a type (float32, bfloat16, float16) and shape; ``x = None`` leaves the stream out.
    ``post_weight`` / ``pre_weight`` (float32 ``[D]``) turn the norm of ``a`` / of ``y`` on (without ``pre_weight``, ``z`` is None),
    their biases are optional.  ``kind``: ``"rms"`` or ``"layer"``, over the last dimension, for both.  ``gate``: float32 ``[D]``
    (a learned scale per channel) or of ``a``'s type and shape.  ``D <= 8192``; ``a`` has two dimensions or more.

    One read of every operand forward and backward, fp32 inside, each output rounded once (``z`` is the norm of ``y`` before its
    rounding).  Differentiable once in all tensors; gradients do not change from run to run."""
    if kind not in KINDS:
        _fail(f"sandwich_norm: kind {kind!r} is neither 'rms' nor 'layer'")
    if a.dim() < 2 or a.dtype not in DTYPES:
        _fail(f"sandwich_norm: a must be float32, bfloat16 or float16 [..., D], got {a.dtype} {tuple(a.shape)}")
    d = a.shape[-1]
    if not 0 < d <= 8192:
        _fail(f"sandwich_norm: rows of {d} columns have no kernel (1 .. 8192)")
    if x is not None and (x.shape != a.shape or x.dtype != a.dtype):
        _fail(f"sandwich_norm: x is {x.dtype} {tuple(x.shape)}, a is {a.dtype} {tuple(a.shape)}")
    for name, t in (("post_weight", post_weight), ("post_bias", post_bias), ("pre_weight", pre_weight), ("pre_bias", pre_bias)):
        if t is not None and (tuple(t.shape) != (d,) or t.dtype != torch.float32):
            _fail(f"sandwich_norm: {name} must be float32 [{d}], got {t.dtype} {tuple(t.shape)}")
    if post_bias is not None and post_weight is None or pre_bias is not None and pre_weight is None:
        _fail("sandwich_norm: a bias without its norm's weight")
    if gate is not None and not (tuple(gate.shape) == (d,) and gate.dtype == torch.float32
                                 or gate.shape == a.shape and gate.dtype == a.dtype):
        _fail(f"sandwich_norm: gate must be float32 [{d}] or {a.dtype} {tuple(a.shape)}, got {gate.dtype} {tuple(gate.shape)}")
    tensors = (x, a, post_weight, post_bias, pre_weight, pre_bias, gate)
    for t in tensors:
        if t is not None and not t.is_cuda:
            _fail("graphgps_amd ops run on an MI355X only (got a CPU tensor); there is no CPU fallback in the product path")
        if t is not None and t.device != a.device:
            _fail(f"tensors on different devices: {a.device} vs {t.device}")
    train = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)
    return _Sandwich.apply(*tensors, float(residual_scale), float(branch_scale), KINDS[kind], float(eps), train)
