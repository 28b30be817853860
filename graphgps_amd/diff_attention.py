"""Differential attention over ragged segments (csrc/diff_attn.hip, diff_attn_bwd.hip).

    o = (softmax(s q1 k1^T) - lam softmax(s q2 k2^T)) v          per segment and head

Two score maps per head, each over ``d`` columns of ``q`` and ``k``, share a value of ``2 d`` columns; ``lam`` (one learned
weight per head) sets how much of the second map is taken off the first.  Reached as ``graphgps_amd.ops.diff_attention``
(separate ``q`` / ``k`` / ``v``, separate query and key segments) and ``ops.diff_segment_attention`` (a packed projection over
the graphs of a batch, next to ``ops.segment_attention``); ``layer.diff_attention_layer.DiffSelfAttention`` is the module.

Like every operator of this package the calls only enqueue kernels on the current stream of the tensors' device: no
synchronisation, no host read-back, no fallback.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

from . import lib as _lib
from .lib import DiffAttn, check, current_stream, on_device, ptr

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}      # GPS_F32, GPS_BF16, GPS_F16


def _fail(msg: str):
    raise _lib.GpsHipError(msg)


def _chunked(t: torch.Tensor) -> torch.Tensor:
    """``t`` as the kernels read it: contiguous last dimension, 16-byte aligned chunks of eight elements, row and map strides whose
    multiples fit 32 bits."""
    st = t.stride()
    if st[-1] == 1 and t.data_ptr() % 16 == 0 and all(s % 8 == 0 for s in st[:-1]) and st[0] <= 1 << 22 and (len(st) < 4 or st[2] <= 1 << 28):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _check_ptr(p: torch.Tensor, name: str, dev) -> torch.Tensor:
    if not torch.is_tensor(p) or p.dim() != 1 or p.numel() < 1 or p.dtype not in (torch.int32, torch.int64):
        _fail(f"diff_attention: {name} must be int32 [segments + 1], got {getattr(p, 'dtype', type(p))} "
              f"{tuple(getattr(p, 'shape', ()))}")
    if p.device != dev:
        _fail(f"diff_attention: {name} is on {p.device}, q on {dev}")
    return _keepable(p.to(torch.int32).contiguous())


def _keepable(t: torch.Tensor) -> torch.Tensor:
    """autograd saves no tensor that was made under inference mode (a batch's index may have been): a copy then."""
    return t.clone() if t.is_inference() and not torch.is_inference_mode_enabled() else t


def _check_inputs(q, k, v, lam, key_mask) -> Tuple[int, int, int]:
    if q.dim() != 4 or q.shape[2] != 2 or k.dim() != 4 or k.shape[2] != 2 or v.dim() != 3:
        _fail(f"diff_attention: expected q [Nq, H, 2, d], k [Nk, Hk, 2, d], v [Nk, Hk, 2d], got {tuple(q.shape)}, "
              f"{tuple(k.shape)}, {tuple(v.shape)}")
    H, Hk, d = q.shape[1], k.shape[1], q.shape[3]
    if q.dtype not in DTYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        _fail(f"diff_attention: q, k, v must share one of float32, bfloat16, float16; got {q.dtype}, {k.dtype}, {v.dtype}")
    if k.shape[3] != d or tuple(v.shape) != (k.shape[0], Hk, 2 * d):
        _fail(f"diff_attention: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)} do not fit together")
    if Hk == 0 or H == 0 or H % Hk:
        _fail(f"diff_attention: {H} heads over {Hk} key heads")
    if d % 8 or not 0 < d <= 128:
        _fail(f"diff_attention: head width {d} has no kernel (multiples of 8 up to 128)")
    if tuple(lam.shape) != (H,) or lam.dtype not in (torch.float32, q.dtype):
        _fail(f"diff_attention: lam must be float32 or {q.dtype} [{H}], got {lam.dtype} {tuple(lam.shape)}")
    if key_mask is not None and (tuple(key_mask.shape) != (k.shape[0],) or key_mask.dtype not in (torch.bool, torch.uint8)):
        _fail(f"diff_attention: key_mask must be bool [{k.shape[0]}], got {key_mask.dtype} {tuple(key_mask.shape)}")
    for t in (q, k, v, lam, key_mask):
        if t is not None and not t.is_cuda:
            _fail("graphgps_amd ops run on an MI355X only (got a CPU tensor); there is no CPU fallback in the product path")
        if t is not None and t.device != q.device:
            _fail(f"tensors on different devices: {q.device} vs {t.device}")
    return H, Hk, d


class _Call:
    """What forward and backward of one call share."""

    def __init__(self, q, k, v, lam, q_ptr, k_ptr, causal, key_mask, scale, max_q, max_k):
        if scale is not None and not 0.0 < float(scale) < float("inf"):
            _fail(f"diff_attention: scale {scale} is not positive")
        H, Hk, d = _check_inputs(q, k, v, lam, key_mask)
        dev = q.device
        q_ptr = _check_ptr(q_ptr, "q_ptr", dev)
        k_ptr = q_ptr if k_ptr is None else _check_ptr(k_ptr, "k_ptr", dev)
        if q_ptr.numel() != k_ptr.numel():
            _fail(f"diff_attention: {q_ptr.numel() - 1} query segments, {k_ptr.numel() - 1} key segments")
        if max_q < 0 or max_k < 0:
            _fail(f"diff_attention: max_q={max_q}, max_k={max_k}")
        self.H, self.Hk, self.d, self.causal = H, Hk, d, bool(causal)
        self.scale = float(d) ** -0.5 if scale is None else float(scale)
        self.max_q, self.max_k = int(max_q), int(max_k)
        self.q_ptr, self.k_ptr = q_ptr, k_ptr
        self.keep = None if key_mask is None else _keepable(key_mask.contiguous().view(torch.uint8))

    def segments(self):
        """What the kernels read beside the operands.  The backward reads it too, so it is saved like an operand: a change in place in
        between raises there."""
        return self.q_ptr, self.k_ptr, self.keep

    def block(self, q, k, v, lam, o, kept, q_ptr, k_ptr, keep) -> DiffAttn:
        n = q.shape[0]
        a = DiffAttn(q=ptr(q), k=ptr(k), v=ptr(v), lam=ptr(lam), o=ptr(o), q_ptr=ptr(q_ptr), k_ptr=ptr(k_ptr), keep=ptr(keep),
                     Nq=n, Nk=k.shape[0], B=q_ptr.numel() - 1, H=self.H, Hk=self.Hk, d=self.d, causal=int(self.causal),
                     lam_f32=int(lam.dtype == torch.float32), dtype=DTYPES[q.dtype], max_q=self.max_q, max_k=self.max_k,
                     scale=self.scale)
        a.q_rs, a.q_hs, a.q_ms = q.stride()[:3]
        a.k_rs, a.k_hs, a.k_ms = k.stride()[:3]
        a.v_rs, a.v_hs = v.stride()[:2]
        if kept is not None and n:
            at, size = kept.data_ptr(), n * self.H * 2 * self.d
            a.o2, a.lse = at, at + 4 * size
            if q.dtype != torch.float32:                     # behind both, on 16 bytes
                a.o_rest = at + (4 * (size + 2 * n * self.H) + 15) // 16 * 16
        return a

    def forward(self, q, k, v, lam, train: bool):
        """-> (o, kept): ``kept`` is one fp32 buffer, the second map's share [Nq, H, 2d], then the log-sums [2, H, Nq], and for 16-bit
        types what ``o`` lost when it was rounded [Nq, H, 2d]."""
        dev, n, L = q.device, q.shape[0], _lib.load()
        o = torch.empty(n, self.H, 2 * self.d, dtype=q.dtype, device=dev)
        kept = None
        if train:
            rest = 0 if q.dtype == torch.float32 else n * self.H * self.d + 3
            kept = torch.empty(n * self.H * (2 * self.d + 2) + rest, dtype=torch.float32, device=dev)
        self.args = a = self.block(q, k, v, lam, o, kept, *self.segments())
        a.ws_floats = L.gps_diff_attn_fwd_workspace_floats(ctypes.addressof(a))
        ws = torch.empty(a.ws_floats, dtype=torch.float32, device=dev) if a.ws_floats else None
        a.ws = ptr(ws)
        with on_device(dev):
            check(L.gps_diff_attn_fwd(ctypes.addressof(a), current_stream(dev)), "gps_diff_attn_fwd")
        return o, kept

    def backward(self, a: DiffAttn, lam, do, dq, dk, dv):
        """``a``: the inputs' argument block, which is the backward's from here on."""
        if torch.is_grad_enabled():
            _fail("diff_attention is differentiable once: its backward has no gradient of its own")
        L, dev = _lib.load(), dq.device
        if do.dtype != dq.dtype:
            _fail(f"diff_attention: gradient of type {do.dtype} for an output of type {dq.dtype}")
        do = _chunked(do)
        dlam = torch.empty_like(lam)
        a.ws_floats = L.gps_diff_attn_bwd_workspace_floats(a.Nq, a.H, a.B)
        ws = torch.empty(a.ws_floats, dtype=torch.float32, device=dev)
        a.dout, a.dq, a.dk, a.dv, a.dlam, a.ws = [t.data_ptr() for t in (do, dq, dk, dv, dlam, ws)]
        a.do_rs, a.do_hs, _ = do.stride()
        a.dq_rs, a.dq_hs, a.dq_ms, _ = dq.stride()
        a.dk_rs, a.dk_hs, a.dk_ms, _ = dk.stride()
        a.dv_rs, a.dv_hs, _ = dv.stride()
        with on_device(dev):
            check(L.gps_diff_attn_bwd(ctypes.addressof(a), current_stream(dev)), "gps_diff_attn_bwd")
        return dlam


def where(*tensors):
    """What an argument block holds of tensors: while it is the same, so is the block.  Hooks on saved tensors (activation checkpoints,
    offloading) may hand a backward other memory than its forward had."""
    return [None if t is None else (t.data_ptr(), t.stride()) for t in tensors]


class _DiffAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lam, call: _Call, train: bool):
        q, k, v, lam = _chunked(q), _chunked(k), _chunked(v), lam.contiguous()
        o, kept = call.forward(q, k, v, lam, train)
        if train:
            saved = (q, k, v, lam, o, kept, *call.segments())
            ctx.save_for_backward(*saved)
            ctx.call, ctx.at = call, where(*saved)
        return o

    @staticmethod
    def backward(ctx, do):
        saved = q, k, v, lam, *_ = ctx.saved_tensors
        dq, dk, dv = [torch.empty_like(t, memory_format=torch.contiguous_format) for t in (q, k, v)]
        c = ctx.call
        a = DiffAttn.from_buffer_copy(c.args) if where(*saved) == ctx.at else c.block(*saved)
        dlam = c.backward(a, lam, do, dq, dk, dv)
        return dq, dk, dv, dlam, None, None


def _split(qkv: torch.Tensor, H: int, Hk: int, d: int):
    """Views of a packed projection's rows: q [n, H, 2, d] | k [n, Hk, 2, d] | v [n, Hk, 2d]."""
    n, (s, e), at = qkv.shape[0], qkv.stride(), qkv.storage_offset()
    return (qkv.as_strided((n, H, 2, d), (s, 2 * d * e, d * e, e), at),
            qkv.as_strided((n, Hk, 2, d), (s, 2 * d * e, d * e, e), at + 2 * H * d * e),
            qkv.as_strided((n, Hk, 2 * d), (s, 2 * d * e, e), at + 2 * (H + Hk) * d * e))


class _DiffSegmentAttention(torch.autograd.Function):
    """The packed form: the gradient comes back packed, written in place by the kernels."""

    @staticmethod
    def forward(ctx, qkv, lam, call: _Call, train: bool):
        qkv, lam = _chunked(qkv), lam.contiguous()
        o, kept = call.forward(*_split(qkv, call.H, call.Hk, call.d), lam, train)
        if train:
            saved = (qkv, lam, o, kept, *call.segments())
            ctx.save_for_backward(*saved)
            ctx.call, ctx.at = call, where(*saved)
        return o

    @staticmethod
    def backward(ctx, do):
        saved = qkv, lam, *rest = ctx.saved_tensors
        c = ctx.call
        d_qkv = torch.empty_like(qkv, memory_format=torch.contiguous_format)
        a = DiffAttn.from_buffer_copy(c.args) if where(*saved) == ctx.at else c.block(*_split(qkv, c.H, c.Hk, c.d), lam, *rest)
        dlam = c.backward(a, lam, do, *_split(d_qkv, c.H, c.Hk, c.d))
        return d_qkv, dlam, None, None


def diff_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lam: torch.Tensor, q_ptr: torch.Tensor,
                   k_ptr: Optional[torch.Tensor] = None, *, causal: bool = False, key_mask: Optional[torch.Tensor] = None,
                   scale: Optional[float] = None, max_q: int = 0, max_k: int = 0) -> torch.Tensor:
    """``(softmax(scale q1 k1^T) - lam softmax(scale q2 k2^T)) v`` per segment and head -> ``[Nq, H, 2d]``.

    ``q [Nq, H, 2, d]``, ``k [Nk, Hk, 2, d]``, ``v [Nk, Hk, 2d]`` of one type (float32, bfloat16, float16), any strides; ``H`` a
    multiple of ``Hk`` (head ``h`` reads key head ``h // (H / Hk)``); ``d`` a multiple of 8 up to 128.  ``lam [H]`` is float32 or
    of that type.  Segment ``s`` owns the query rows ``q_ptr[s] : q_ptr[s + 1]`` and the key rows ``k_ptr[s] : k_ptr[s + 1]``
    (int32, on the device, non-decreasing from 0; ``k_ptr = None``: the same).  Rows behind the last segment and rows that see no key
    give 0, and take no gradient.

    ``causal``: the query at index i of a segment with n queries and m keys sees the keys up to index ``i + m - n``; a key a
    query does not see has to be finite, as in any product with a zero weight.  ``key_mask [Nk]``: False drops a key for all
    queries; its rows of ``k`` and ``v`` may hold anything.  ``scale`` (positive) defaults to ``d ** -0.5``.  ``max_q`` / ``max_k``: the
    longest segment where the host knows it; they choose the launch shape only, and one query per segment
    (``max_q = 1``) over long key segments is split along the keys.

    Differentiable once in ``q``, ``k``, ``v`` and ``lam``; results do not change from run to run.  The backward reads the offsets
    and the mask again: one that was changed in place in between raises, like any saved tensor."""
    call = _Call(q, k, v, lam, q_ptr, k_ptr, causal, key_mask, scale, max_q, max_k)
    train = torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v, lam))
    return _DiffAttention.apply(q, k, v, lam, call, train)


def diff_segment_attention(qkv: torch.Tensor, lam: torch.Tensor, gi, num_heads: int, kv_heads: Optional[int] = None, *,
                           causal: bool = False, key_mask: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
    """Self-attention of :func:`diff_attention` over the graphs of a batch, off a packed projection -> ``[N, H, 2d]``.

    ``qkv [N, 2 H d + 4 Hk d]`` holds ``q [H, 2, d] | k [Hk, 2, d] | v [Hk, 2d]`` per row; ``gi`` is the batch's ``GraphIndex``
    (its ``ptr``, and its ``nmax_host`` for the launch shape)."""
    H = int(num_heads)
    Hk = H if kv_heads is None else int(kv_heads)
    if qkv.dim() != 2 or H <= 0 or Hk <= 0 or qkv.shape[1] % (2 * H + 4 * Hk):
        _fail(f"diff_segment_attention: qkv {tuple(qkv.shape)} does not hold {H} heads over {Hk} key heads")
    if qkv.shape[0] != gi.N:
        _fail(f"diff_segment_attention: qkv {tuple(qkv.shape)} vs N={gi.N}")
    d = qkv.shape[1] // (2 * H + 4 * Hk)
    n = int(gi.nmax_host)
    q, k, v = _split(qkv.detach(), H, Hk, d)
    call = _Call(q, k, v, lam, gi.ptr, None, causal, key_mask, scale, n, n)
    train = torch.is_grad_enabled() and (qkv.requires_grad or lam.requires_grad)
    return _DiffSegmentAttention.apply(qkv, lam, call, train)
