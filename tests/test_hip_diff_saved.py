"""What the backward of differential attention reads beside its operands: segment offsets and the key mask.  They are saved like
operands, so a change in place between a forward and its backward raises instead of giving another call's gradients."""
import pytest
import torch

from test_hip_diff_attention import F32, compare, make

pytestmark = pytest.mark.gpu


def inputs():
    lens = [40, 70, 9]
    q, k, v, lam, qp, kp, do = make(lens, lens, 4, 2, 32, F32, seed=21)
    keep = (torch.rand(k.shape[0], generator=torch.Generator().manual_seed(22)) < 0.7).cuda()
    return [t.requires_grad_(True) for t in (q, k, v, lam)], qp, kp, keep, do


@pytest.mark.parametrize("mask_dtype", [torch.bool, torch.uint8], ids=["bool", "uint8"])
@pytest.mark.parametrize("what", ["key_mask", "q_ptr", "k_ptr", "both_ptr"])
def test_a_refilled_buffer_raises(what, mask_dtype):
    from graphgps_amd import ops
    leaves, qp, kp, keep, do = inputs()
    keep = keep.to(mask_dtype)
    o = ops.diff_attention(*leaves, qp, None if what == "both_ptr" else kp, key_mask=keep)
    {"key_mask": keep, "q_ptr": qp, "k_ptr": kp, "both_ptr": qp}[what].zero_()      # the next micro-batch, in the same buffer
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(o, leaves, do)


@pytest.mark.parametrize("what", ["key_mask", "ptr"])
def test_a_refilled_buffer_raises_packed(what):
    from graphgps_amd import ops
    (q, k, v, lam), qp, _, keep, do = inputs()
    n = q.shape[0]
    gi = ops.build_graph_index(torch.zeros(2, 0, dtype=torch.int64, device="cuda"), n, 3, ptr_vec=qp)
    qkv = torch.cat([t.detach().reshape(n, -1) for t in (q, k, v)], 1).requires_grad_(True)
    o = ops.diff_segment_attention(qkv, lam, gi, 4, 2, key_mask=keep)
    (keep if what == "key_mask" else gi.ptr).zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(o, [qkv, lam], do)


def test_untouched_and_copied_buffers_are_fine():
    """int64 offsets are converted, a sliced mask is copied: what the caller does with theirs afterwards is the caller's."""
    from graphgps_amd import ops
    leaves, qp, kp, keep, do = inputs()
    wide = torch.stack([keep, ~keep], 1)
    q64, k64 = qp.long(), kp.long()
    o = ops.diff_attention(*leaves, q64, k64, key_mask=wide[:, 0])
    for t in (q64, k64, wide):
        t.zero_()
    got = [o.detach(), *torch.autograd.grad(o, leaves, do)]
    compare(got, (*leaves, qp, kp), do, F32, keep=keep)


def test_offsets_made_under_inference_mode():
    """A batch that was evaluated first may carry them."""
    from graphgps_amd import ops
    leaves, qp, kp, keep, do = inputs()
    with torch.inference_mode():
        qi, ki, mi = qp.clone(), kp.clone(), keep.clone()
        ops.diff_attention(*[t.detach() for t in leaves], qi, ki, key_mask=mi)
    o = ops.diff_attention(*leaves, qi, ki, key_mask=mi)
    compare([o.detach(), *torch.autograd.grad(o, leaves, do)], (*leaves, qp, kp), do, F32, keep=keep)
