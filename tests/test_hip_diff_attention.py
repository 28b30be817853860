"""Differential attention (ops.diff_attention / diff_segment_attention) against its definition in 64 bits.

Tolerances.  Let ``h`` be half a step of the type relative to a value (2^-24, 2^-8, 2^-11).  A weight is exp2 of a score: the score's
fp32 contraction of d terms is off by at most (d + 4) 2^-24 times its sum of magnitudes, and that absolute error of the exponent is
the weight's relative error ``w``.  Weights (and their gradients) are rounded once to the type before the second product, which
sums n terms in fp32; the result is rounded once more.  So an output is off by at most
``(w + 2 h + (n + 16) 2^-24) * mass``, ``mass`` = the same sum over magnitudes, and a gradient that goes through
dS = P (dP - D) by that with mass P (|dO| |V|^T + sum |dO| |O|), counted twice (dP and the saved output each bring one)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def reference(q, k, v, lam, q_ptr, k_ptr, causal=False, keep=None, scale=None, do=None):
    """Outputs, gradients and the masses of both, in float64 on the CPU, segment by segment."""
    q, k, v, lam = (t.detach().double().cpu() for t in (q, k, v, lam))
    do = None if do is None else do.detach().double().cpu()
    keep = torch.ones(k.shape[0], dtype=torch.bool) if keep is None else keep.detach().cpu().bool()
    k, v = (torch.where(keep.view(-1, 1, *[1] * (t.dim() - 2)), t, torch.zeros_like(t)) for t in (k, v))
    H, Hk, d = q.shape[1], k.shape[1], q.shape[3]
    s = d ** -0.5 if scale is None else scale
    r = {n: torch.zeros_like(t) for n, t in (("q", q), ("k", k), ("v", v), ("lam", lam))}
    mass = {n: torch.zeros_like(t) for n, t in r.items()}
    o = torch.zeros(q.shape[0], H, 2 * d, dtype=torch.float64)
    mass["o"], worst, longest = torch.zeros_like(o), 0.0, 1
    for b in range(len(q_ptr) - 1):
        q0, q1, k0, k1 = int(q_ptr[b]), int(q_ptr[b + 1]), int(k_ptr[b]), int(k_ptr[b + 1])
        if q1 <= q0 or k1 <= k0:
            continue
        longest = max(longest, k1 - k0, q1 - q0)
        see = keep[k0:k1].expand(q1 - q0, -1).clone()
        if causal:
            see &= torch.ones_like(see).tril((k1 - k0) - (q1 - q0))
        for h in range(H):
            hk = h // (H // Hk)
            V, P = v[k0:k1, hk], []
            for i in range(2):
                z = (q[q0:q1, h, i] @ k[k0:k1, hk, i].T) * s
                worst = max(worst, float((q[q0:q1, h, i].abs() @ k[k0:k1, hk, i].abs().T).max()) * abs(s))
                P.append(torch.nan_to_num(torch.softmax(z.masked_fill(~see, -math.inf), -1), nan=0.0))
            O = [p @ V for p in P]
            la = lam[h].abs()
            o[q0:q1, h] = O[0] - lam[h] * O[1]
            mass["o"][q0:q1, h] = (P[0] + la * P[1]) @ V.abs()
            if do is None:
                continue
            c = torch.where(see.any(1, keepdim=True), do[q0:q1, h], torch.zeros_like(do[q0:q1, h]))
            r["lam"][h] -= (c * O[1]).sum()
            mass["lam"][h] += (c.abs() * (P[1] @ V.abs())).sum()
            r["v"][k0:k1, hk] += (P[0] - lam[h] * P[1]).T @ c
            mass["v"][k0:k1, hk] += (P[0] + la * P[1]).T @ c.abs()
            dp, dpm = c @ V.T, c.abs() @ V.abs().T
            om = (c.abs() * mass["o"][q0:q1, h]).sum(-1, keepdim=True)
            for i, f in ((0, 1.0), (1, -lam[h])):
                ds = f * s * P[i] * (dp - (c * O[i]).sum(-1, keepdim=True))
                dsm = abs(f) * abs(s) * P[i] * (dpm + om + (c.abs() * (P[i] @ V.abs())).sum(-1, keepdim=True))
                r["q"][q0:q1, h, i] += ds @ k[k0:k1, hk, i]
                r["k"][k0:k1, hk, i] += ds.T @ q[q0:q1, h, i]
                mass["q"][q0:q1, h, i] += dsm @ k[k0:k1, hk, i].abs()
                mass["k"][k0:k1, hk, i] += dsm.T @ q[q0:q1, h, i].abs()
    r["o"] = o
    w = 2.0 ** -24 * (d + 4) * max(worst, 1.0) * 1.5
    return r, mass, w, longest


def close(got, want, mass, rel, what):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.isfinite(got).all(), f"{what}: not finite"
    off = (got - want).abs() - rel * mass - 1e-30
    assert float(off.max()) <= 0 if off.numel() else True, (
        f"{what}: off by {float((got - want).abs().max()):.3e}, {float(((got - want).abs() / (rel * mass + 1e-30)).max()):.2f} x the bound")


def make(q_lens, k_lens, H, Hk, d, dtype, seed=0, tail=0, std=1.0):
    g = torch.Generator().manual_seed(seed)
    nq, nk = sum(q_lens) + tail, sum(k_lens) + tail

    def randn(*shape):
        return (torch.randn(*shape, generator=g) * std).to(dtype).cuda()
    q, k, v = randn(nq, H, 2, d), randn(nk, Hk, 2, d), randn(nk, Hk, 2 * d)
    lam = (0.1 + 0.8 * torch.rand(H, generator=g)).cuda()
    ptrs = [torch.tensor([sum(x[:i]) for i in range(len(x) + 1)], dtype=torch.int32, device="cuda") for x in (q_lens, k_lens)]
    return q, k, v, lam, ptrs[0], ptrs[1], randn(nq, H, 2 * d)


def run(q, k, v, lam, q_ptr, k_ptr, do, **kw):
    from graphgps_amd import ops
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v, lam)]
    o = ops.diff_attention(*leaves, q_ptr, k_ptr, **kw)
    return [o.detach(), *torch.autograd.grad(o, leaves, do)]


def compare(got, args, do, dtype, lam_dtype=F32, **kw):
    want, mass, w, n = reference(*args, do=do, **kw)
    rel = w + 2 * HALF[dtype] + (n + 16) * 2.0 ** -24
    close(got[0], want["o"], mass["o"], rel, "o")
    for name, t, f in (("q", got[1], 2), ("k", got[2], 2), ("v", got[3], 1), ("lam", got[4], 1)):
        group = args[0].shape[1] // args[1].shape[1] if name in "kv" else 1
        close(t, want[name], mass[name], f * rel + group * n * 2.0 ** -24 + (HALF[lam_dtype] if name == "lam" else 0.0), "d" + name)


LENS = {"mixed": [30, 1, 0, 47, 64, 17], "long": [517, 130], "ones": [1, 1, 1], "block": [128, 64], "molecules": [29, 31, 8, 33, 51, 16, 2]}


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("d", [8, 24, 32, 40, 64, 96, 128])
@pytest.mark.parametrize("lens", ["mixed", "long"])
def test_forward_and_gradients(dtype, d, lens):
    H, Hk = (4, 2) if d % 16 == 0 else (3, 3)
    q, k, v, lam, qp, kp, do = make(LENS[lens], LENS[lens], H, Hk, d, dtype)
    compare(run(q, k, v, lam, qp, kp, do), (q, k, v, lam, qp, kp), do, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("hint", [0, 16, 64, 600])
@pytest.mark.parametrize("lens", sorted(LENS))
def test_launch_shapes_agree(dtype, hint, lens):
    """The hints choose a launch shape; a wrong one costs time, not results."""
    q, k, v, lam, qp, kp, do = make(LENS[lens], LENS[lens], 4, 1, 24, dtype, seed=1)
    compare(run(q, k, v, lam, qp, kp, do, max_q=hint, max_k=hint), (q, k, v, lam, qp, kp), do, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("lens,hint", [("mixed", 1), ("long", 2), ("molecules", 3)])
def test_more_queries_than_the_few_that_were_said(dtype, lens, hint):
    q, k, v, lam, qp, kp, do = make(LENS[lens], LENS[lens], 4, 2, 40, dtype, seed=16)
    keep = (torch.rand(k.shape[0], generator=torch.Generator().manual_seed(17)) < 0.8).cuda()
    got = run(q, k, v, lam, qp, kp, do, max_q=hint, causal=True, key_mask=keep)
    compare(got, (q, k, v, lam, qp, kp), do, dtype, causal=True, keep=keep)


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("q_lens,k_lens", [([40, 3, 0, 70], [40, 9, 5, 200]), ([33, 100, 4], [7, 100, 0]), ([1, 1], [300, 1])])
@pytest.mark.parametrize("causal", [False, True])
def test_separate_segments_and_causal(dtype, q_lens, k_lens, causal):
    """Query and key segments of different lengths: under `causal`, queries in front of the first key see nothing."""
    q, k, v, lam, qp, kp, do = make(q_lens, k_lens, 6, 2, 32, dtype, seed=2)
    got = run(q, k, v, lam, qp, kp, do, causal=causal, max_q=max(q_lens), max_k=max(k_lens))
    compare(got, (q, k, v, lam, qp, kp), do, dtype, causal=causal)


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("d", [32, 128])
def test_dropped_keys_hold_anything(dtype, causal, d):
    lens = [70, 5, 129, 1]
    q, k, v, lam, qp, kp, do = make(lens, lens, 4, 2, d, dtype, seed=3, tail=5)
    keep = torch.rand(k.shape[0], generator=torch.Generator().manual_seed(4)) < 0.6
    keep[70:75] = False                       # nothing left in the second segment
    keep = keep.cuda()
    clean = (k.clone(), v.clone())
    k[~keep], v[~keep] = float("nan"), float("inf")
    k[-3:], v[-3:], q[-3:], do[-3:] = float("nan"), float("-inf"), float("nan"), float("nan")     # behind the last segment
    do[72] = float("nan")                     # the gradient of a row that saw nothing
    got = run(q, k, v, lam, qp, kp, do, causal=causal, key_mask=keep)
    n = sum(lens)
    args = (q[:n], clean[0][:n], clean[1][:n], lam, qp, kp)
    compare([t[:n] if t.dim() > 1 else t for t in got], args, do[:n], dtype, causal=causal, keep=keep[:n])
    for t in got[:4]:
        assert (t[n:] == 0).all(), "rows behind the last segment"
    assert (got[0][70:75] == 0).all() and (got[1][70:75] == 0).all()
    assert (got[2][:n][~keep[:n]] == 0).all() and (got[3][:n][~keep[:n]] == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("q_len", [1, 3])
@pytest.mark.parametrize("H,Hk", [(8, 2), (3, 3), (16, 1), (32, 1)])
@pytest.mark.parametrize("d", [32, 64, 128])
def test_few_queries_over_many_keys(dtype, q_len, H, Hk, d):
    """The single-token form: the hints say so, the keys are split and joined."""
    from graphgps_amd import ops
    k_lens = [2500, 0, 1, 700, 64, 33]
    q, k, v, lam, qp, kp, _ = make([q_len] * 6, k_lens, H, Hk, d, dtype, seed=5)
    keep = (torch.rand(k.shape[0], generator=torch.Generator().manual_seed(6)) < 0.9).cuda()
    for kw in ({}, {"key_mask": keep}, {"causal": True}):
        with torch.no_grad():
            got = ops.diff_attention(q, k, v, lam, qp, kp, max_q=q_len, max_k=2500, **kw)
        want, mass, w, n = reference(q, k, v, lam, qp, kp, causal=kw.get("causal", False), keep=kw.get("key_mask"))
        close(got, want["o"], mass["o"], w + 2 * HALF[dtype] + (n + 16) * 2.0 ** -24, str(sorted(kw)))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
def test_training_with_few_queries(dtype):
    k_lens = [2500, 0, 1, 700]
    q, k, v, lam, qp, kp, do = make([1] * 4, k_lens, 4, 2, 32, dtype, seed=7)
    compare(run(q, k, v, lam, qp, kp, do, max_q=1, max_k=2500), (q, k, v, lam, qp, kp), do, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("kv_heads", [None, 2])
def test_packed_projection(dtype, kv_heads):
    from graphgps_amd import ops
    lens, H, d = LENS["molecules"], 4, 24
    Hk = kv_heads or H
    q, k, v, lam, qp, _, do = make(lens, lens, H, Hk, d, dtype, seed=8)
    n = q.shape[0]
    gi = ops.build_graph_index(torch.zeros(2, 0, dtype=torch.int64, device="cuda"), n, len(lens), ptr_vec=qp)
    gi.nmax_host = max(lens)
    qkv = torch.cat([t.reshape(n, -1) for t in (q, k, v)], 1).requires_grad_(True)
    lam = lam.requires_grad_(True)
    o = ops.diff_segment_attention(qkv, lam, gi, H, kv_heads)
    g, gl = torch.autograd.grad(o, [qkv, lam], do)
    gq, gk, gv = g.split([2 * H * d, 2 * Hk * d, 2 * Hk * d], 1)
    compare([o, gq.reshape(q.shape), gk.reshape(k.shape), gv.reshape(v.shape), gl], (q, k, v, lam, qp, qp), do, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
def test_strides_alignment_and_broadcast_gradients(dtype):
    """Transposed heads, a slice that starts off a 16-byte boundary, an expanded output gradient, lam in the inputs' type, int64
    offsets."""
    lens = [37, 90]
    q, k, v, lam, qp, kp, do = make(lens, lens, 4, 2, 32, dtype, seed=9)
    wide = torch.zeros(q.shape[0], 4, 2, 33, dtype=dtype, device="cuda")
    wide[..., 1:] = q
    q_odd = wide[..., 1:]                                                  # odd strides and start
    k_t = k.transpose(0, 1).contiguous().transpose(0, 1)                   # [Hk, Nk] order in memory
    v_t = v.transpose(1, 2).contiguous().transpose(1, 2)                   # last dimension not contiguous
    do = do[:1, :1].expand(do.shape)
    lam = lam.to(dtype)
    got = run(q_odd, k_t, v_t, lam, qp.long(), kp.long(), do)
    assert got[4].dtype == dtype
    compare(got, (q, k, v, lam, qp, kp), do, dtype, lam_dtype=dtype)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
def test_large_scores_and_scale(dtype):
    """Scores of several hundred: all the weight on single keys, no overflow."""
    lens = [50, 20]
    q, k, v, lam, qp, kp, do = make(lens, lens, 2, 2, 32, dtype, seed=10, std=6.0)
    compare(run(q, k, v, lam, qp, kp, do, scale=0.5), (q, k, v, lam, qp, kp), do, dtype, scale=0.5)


def test_non_finite_inputs_spread_like_in_the_formula():
    lens = [20, 20]
    q, k, v, lam, qp, kp, do = make(lens, lens, 2, 2, 32, F32, seed=11)
    q[3, 0, 0, 0] = float("nan")
    from graphgps_amd import ops
    o = ops.diff_attention(q, k, v, lam, qp, kp)
    bad = torch.isnan(o).any(-1)
    assert bad[3, 0] and int(bad.sum()) == 1


def test_gradient_against_differences():
    from graphgps_amd import ops
    lens = [20, 9, 33]
    q, k, v, lam, qp, kp, do = make(lens, lens, 4, 2, 24, F32, seed=12)
    leaves = [q, k, v, lam]
    got = run(q, k, v, lam, qp, kp, do)
    g = torch.Generator().manual_seed(13)
    for i in range(4):
        e = torch.randn(leaves[i].shape, generator=g).cuda()
        h = 1e-2
        f = [float((ops.diff_attention(*[t + s * h * e if j == i else t for j, t in enumerate(leaves)], qp, kp).double() * do.double()).sum())
             for s in (1, -1)]
        slope, want = (f[0] - f[1]) / (2 * h), float((got[1 + i].double() * e.double()).sum())
        # truncation h^2 / 6 f''' with derivatives of the order of the sums themselves, rounding 2^-24 * 1e4 terms / h
        assert abs(slope - want) <= 2e-3 * float((got[1 + i].double() * e.double()).abs().sum()) + 1e-2


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
def test_same_bits_every_time_and_on_another_stream(dtype):
    q, k, v, lam, qp, kp, do = make([300, 40], [300, 40], 4, 2, 64, dtype, seed=14)
    first = run(q, k, v, lam, qp, kp, do)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = run(q, k, v, lam, qp, kp, do)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, second):
        assert torch.equal(a, b)


@pytest.mark.parametrize("max_q", [0, 1])
def test_captured_and_replayed(max_q):
    from graphgps_amd import ops
    lens_q, lens_k = ([40, 50], [40, 50]) if max_q == 0 else ([1, 1], [3000, 500])
    q, k, v, lam, qp, kp, do = make(lens_q, lens_k, 4, 2, 32, F32, seed=15)
    leaves = [t.requires_grad_(True) for t in (q, k, v, lam)]

    def step():
        o = ops.diff_attention(*leaves, qp, kp, max_q=max_q)
        return [o, *torch.autograd.grad(o, leaves, do)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        with torch.no_grad():
            q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(20 + i)))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        eager = step()
        torch.cuda.synchronize()
        for a, b in zip(got, eager):
            assert torch.equal(a, b.detach())
        del eager


def test_empty_calls():
    q, k, v, lam, qp, kp, do = make([0, 0], [0, 0], 2, 2, 16, F32)
    got = run(q, k, v, lam, qp, kp, do)
    assert got[0].shape == (0, 2, 32) and (got[4] == 0).all()
    q, k, v, lam, qp, kp, do = make([0, 0], [5, 6], 2, 2, 16, F32)
    got = run(q, k, v, lam, qp, kp, do)
    assert all((t == 0).all() for t in got)
    q, k, v, lam, qp, kp, do = make([5, 6], [0, 0], 2, 2, 16, F32)
    got = run(q, k, v, lam, qp, kp, do, max_q=6)
    assert all((t == 0).all() for t in got)


def test_no_second_derivative():
    from graphgps_amd import ops
    from graphgps_amd.lib import GpsHipError
    q, k, v, lam, qp, kp, do = make([5], [5], 2, 2, 16, F32)
    o = ops.diff_attention(q.requires_grad_(True), k, v, lam, qp, kp)
    with pytest.raises(GpsHipError, match="once"):
        torch.autograd.grad(o, q, do, create_graph=True)


@pytest.mark.parametrize("how", ["checkpoint", "offload"])
@pytest.mark.parametrize("max_q", [0, 2])
def test_saved_tensors_that_come_back_elsewhere(how, max_q):
    """Activation checkpoints compute them anew and offloading copies them (contiguous): the gradients stay the same bits."""
    from graphgps_amd import ops
    q, k, v, lam, qp, kp, do = make([2, 1, 2], [200, 90, 131], 4, 2, 40, F32, seed=5)
    want = run(q, k, v, lam, qp, kp, do, max_q=max_q)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v, lam)]

    def call(q, k, v, lam):
        # inputs that live in the graph only: sliced out of wider rows, so their strides are not those of a copy
        q, v = torch.cat([q * 1.0, q], 1)[:, :4], torch.cat([v * 1.0, v], 1)[:, :2]
        return ops.diff_attention(q, k * 1.0, v, lam * 1.0, qp, kp, max_q=max_q)
    if how == "checkpoint":
        from torch.utils.checkpoint import checkpoint
        o = checkpoint(call, *leaves, use_reentrant=False)
    else:
        with torch.autograd.graph.save_on_cpu():
            o = call(*leaves)
    junk = [torch.full((1 << 20,), float("nan"), device="cuda") for _ in range(8)]   # takes what the forward freed
    got = [o.detach(), *torch.autograd.grad(o, leaves, do)]
    del junk
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("how", ["checkpoint", "offload"])
def test_packed_projection_that_comes_back_elsewhere(how):
    from graphgps_amd import ops
    lens, H, d = LENS["molecules"], 4, 24
    q, k, v, lam, qp, _, do = make(lens, lens, H, H, d, BF16, seed=8)
    n = q.shape[0]
    gi = ops.build_graph_index(torch.zeros(2, 0, dtype=torch.int64, device="cuda"), n, len(lens), ptr_vec=qp)
    gi.nmax_host = max(lens)
    qkv, lam = torch.cat([t.reshape(n, -1) for t in (q, k, v)], 1).requires_grad_(True), lam.requires_grad_(True)
    want = torch.autograd.grad(ops.diff_segment_attention(qkv, lam, gi, H), [qkv, lam], do)

    def call(qkv, lam):
        return ops.diff_segment_attention(torch.cat([qkv, qkv], 1)[:, :qkv.shape[1]], lam * 1.0, gi, H)
    if how == "checkpoint":
        from torch.utils.checkpoint import checkpoint
        o = checkpoint(call, qkv, lam, use_reentrant=False)
    else:
        with torch.autograd.graph.save_on_cpu():
            o = call(qkv, lam)
    junk = [torch.full((1 << 20,), float("nan"), device="cuda") for _ in range(8)]
    got = torch.autograd.grad(o, [qkv, lam], do)
    del junk
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("max_q", [0, 1])
def test_a_row_with_one_key_has_no_gradient_of_its_scores(dtype, max_q):
    """One key: both maps' weights are 1 whatever the scores, so dS = dP - dO . O1 = 0.  What may be left of it: the weight that the
    values meet is 1 - lam in 16 bits, half a step off and the same for all columns; what O lost, to 16 bits; the sums' fp32.  (An O
    that is rounded in that difference would leave half a step of every column.)"""
    n, H, d = 200, 4, 32
    q, k, v, lam, qp, kp, do = make([1] * n, [1] * n, H, H, d, dtype, seed=9)
    _, dq, dk, _, _ = run(q, k, v, lam, qp, kp, do, max_q=max_q, max_k=100 * max_q)
    v, do, l = v.double().cpu(), do.double().cpu(), lam.double().cpu()[None]
    half, size, dot = HALF[dtype], (v * do).abs().sum(-1), (v * do).sum(-1).abs()
    lost = half * (1 - l) * dot + half ** 2 * 1.01 * (1 - l) * size + (2.0 ** -25 * do.abs().sum(-1) if dtype == F16 else 0.0)
    ds = (lost + 2.0 ** -24 * (2 * d + 16) * (2 + l) * size) * (1 + 2 * half)
    for got, other in ((dq, k), (dk, q)):
        got, other = got.double().cpu().abs(), other.double().cpu().abs()
        bound = ds[:, :, None, None] * d ** -0.5 * other * (1 + 2 * half) + 2.0 ** -25
        assert (got <= bound).all(), float((got / bound).max())
