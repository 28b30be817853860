"""Differential attention where scores change along a segment: what a block of keys weighs when it is met and what it weighs in the
end differ by orders of magnitude.  Bounds are those of test_hip_diff_attention.py: every rounding to the inputs' type is relative to
a term of the result (or smaller), so they hold whatever the order of the keys.

float16 adds what its range adds: it has no values between 0 and 2^-24 and steps of 2^-24 up to 2^-14, so that a rounding there is off
by up to 2^-25 whatever the value.  Weights far below their row's largest, met here and hardly in iid scores, are in that range: an
output gets 2^-25 of its own, dv 2^-25 |dO| from the rounding of each W, dk and dq 2^-25 s |q| and 2^-25 s |k| from that of each dS
(times max(1, |lam|) <= 1 here), counted with the largest |dO|, |q| and |k| over the rows of a segment and the heads of a group."""
import math

import pytest
import torch

from test_hip_diff_attention import BF16, F16, F32, HALF, close, make, reference, run

pytestmark = pytest.mark.gpu

TYPES = pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["fp32", "bf16", "fp16"])
LN2 = math.log(2.0)


def scores(kind, n):
    """Scores of the two maps along n keys, in nats."""
    i = torch.arange(n, dtype=torch.float32)
    flat, late = torch.zeros(n), torch.where(i < 32, 0.0, 1.0)
    if kind == "low_start":              # the second map's first block is lower
        return flat, 3.0 * late
    if kind == "high_start":             # the first map's is higher
        return -3.0 * late, flat
    if kind == "tree":                   # 64 keys of one kind in front
        return flat, torch.where(i < 64, 0.0, 5.5 * LN2)
    if kind == "sink":                   # one key among far lower ones, then many that stay within reach of it
        return flat, torch.where(i == 0, 0.0, torch.where(i < 32, -20.0 * LN2, 5.5 * LN2))
    if kind == "last_block":             # the first map dips at both ends, the second jumps at the end
        ends = (i < 32) | (i >= n - n % 32 - 32)
        return torch.where(ends, -5.8 * LN2, 0.0), torch.where(i == n - 3, 20.0, 0.0)
    if kind == "two_peaks":              # flat against a peak that rises in two steps
        s = flat.clone()
        s[int(0.72 * n)], s[int(0.88 * n)] = 30.0 * LN2, 35.8 * LN2
        return flat, s
    if kind == "drift":                  # both maps change steadily, in opposite directions
        return 2.0 - 4.0 * i / n, 4.0 * i / n
    if kind == "far_drift":              # the same by far more than one key's weight
        return 30.0 - 60.0 * i / n, 60.0 * i / n
    raise ValueError(kind)


KINDS = ["low_start", "high_start", "tree", "sink", "last_block", "two_peaks", "drift", "far_drift"]


def drifting(kind, q_lens, k_lens, H, Hk, d, dtype, seed=0):
    """Inputs whose scores are `scores(kind)` plus a little of everything else; values with a mean."""
    q, k, v, lam, qp, kp, do = make(q_lens, k_lens, H, Hk, d, dtype, seed=seed)
    q *= 0.2
    q[..., 0] = 1.0
    for b, n in enumerate(k_lens):
        s = scores(kind, n)
        for m in range(2):
            k[int(kp[b]):int(kp[b + 1]), :, m, 0] = s[m][:, None].to(dtype).cuda()
    return q, k, v + 0.5, lam, qp, kp, do


def compare(got, args, do, dtype, **kw):
    q, k = args[0], args[1]
    want, mass, w, n = reference(*args, do=do, **kw)
    rel = w + 2 * HALF[dtype] + (n + 16) * 2.0 ** -24
    group = q.shape[1] // k.shape[1]
    step = 2.0 ** -25 if dtype == F16 else 0.0
    most = {m: float(t.double().abs().max()) for m, t in (("do", do), ("q", q), ("k", k))}
    floor = {"o": step, "q": step * (1 + n * most["k"]), "k": step * (1 + group * n * most["q"]), "v": step * (1 + group * n * most["do"]), "lam": 0.0}
    for name, t, f in (("o", got[0], 1), ("q", got[1], 2), ("k", got[2], 2), ("v", got[3], 1), ("lam", got[4], 1)):
        r = rel if name == "o" else f * rel + (group if name in "kv" else 1) * n * 2.0 ** -24 + (HALF[F32] if name == "lam" else 0.0)
        off = (t.double().cpu() - want[name]).abs()
        allowed = r * mass[name] + floor[name] + 1e-30
        assert torch.isfinite(off).all(), f"{name}: not finite"
        assert (off <= allowed).all(), f"{name}: off by {float(off.max()):.3e}, {float((off / allowed).max()):.2f} x the bound"


@TYPES
@pytest.mark.parametrize("d", [24, 64, 128])
@pytest.mark.parametrize("kind", KINDS)
def test_forward_and_gradients(kind, d, dtype):
    q_lens, k_lens = [20, 7], [2500, 125]
    q, k, v, lam, qp, kp, do = drifting(kind, q_lens, k_lens, 4, 2, d, dtype)
    got = run(q, k, v, lam, qp, kp, do, scale=1.0)
    compare(got, (q, k, v, lam, qp, kp), do, dtype, scale=1.0)


@TYPES
@pytest.mark.parametrize("kind", KINDS)
def test_causal(kind, dtype):
    """Every row of a segment ends at another place of the drift; some keys are dropped."""
    lens = [310, 70]
    q, k, v, lam, qp, kp, do = drifting(kind, lens, lens, 3, 3, 40, dtype, seed=1)
    keep = (torch.rand(k.shape[0], generator=torch.Generator().manual_seed(2)) < 0.9).cuda()
    got = run(q, k, v, lam, qp, kp, do, scale=1.0, causal=True, key_mask=keep)
    compare(got, (q, k, v, lam, qp, kp), do, dtype, scale=1.0, causal=True, keep=keep)


@TYPES
@pytest.mark.parametrize("d", [24, 64, 128])
@pytest.mark.parametrize("kind", KINDS)
def test_few_queries(kind, d, dtype):
    q, k, v, lam, qp, kp, _ = drifting(kind, [1, 2], [2500, 125], 4, 2, d, dtype, seed=3)
    from graphgps_amd import ops
    with torch.no_grad():
        got = ops.diff_attention(q, k, v, lam, qp, kp, scale=1.0, max_q=2, max_k=2500)
    want, mass, w, n = reference(q, k, v, lam, qp, kp, scale=1.0)
    close(got, want["o"], mass["o"], w + 2 * HALF[dtype] + (n + 16) * 2.0 ** -24, kind)


@TYPES
@pytest.mark.parametrize("max_q", [0, 2])
@pytest.mark.parametrize("kind", ["drift", "far_drift", "sink"])
def test_large_values_that_end_with_little_weight(kind, max_q, dtype):
    """What a key's value leaves in the result goes by its weight at the end, not by the one it had when it was met."""
    q, k, v, lam, qp, kp, do = drifting(kind, [2, 1], [1500, 300], 2, 2, 32, dtype, seed=4)
    v[:, :, ::2] = 0.01 * v[:, :, ::2]
    for at in (0, 1500):
        v[at:at + 32] *= 300.0
    got = run(q, k, v, lam, qp, kp, do, scale=1.0, max_q=max_q)
    compare(got, (q, k, v, lam, qp, kp), do, dtype, scale=1.0)


@TYPES
@pytest.mark.parametrize("n", [64, 900])
@pytest.mark.parametrize("max_q", [0, 1])
def test_map_that_hands_over(max_q, n, dtype):
    """The first map rests on key 0.  The second one starts among the keys behind it, whose values are large, and moves to later keys
    with all its weight: nothing of those values may be left."""
    q, k, v, lam, qp, kp, do = make([2], [n], 2, 1, 32, dtype, seed=6)
    i = torch.arange(n)
    q *= 0.05
    q[..., 0] = 1.0
    for m, s in enumerate((torch.where(i == 0, 0.0, -20.0), torch.where(i < 32, 0.0, 20.0))):
        k[:, :, m, 0] = s[:, None].to(dtype).cuda()
    v[0] *= 0.01
    v[1:32] *= 300.0
    got = run(q, k, v, lam, qp, kp, do, scale=1.0, max_q=max_q)
    compare(got, (q, k, v, lam, qp, kp), do, dtype, scale=1.0)


@TYPES
@pytest.mark.parametrize("max_q", [0, 1])
def test_long_row_with_a_share_far_below_its_peak(max_q, dtype):
    """A peak of the first map and 2^20 keys at 2^-25.6 of it, 2 % of the row together: weights that float16 does not hold as they
    are.  The bound counts fp32 sums as they are made: 16-bit products come 32 keys to an addition, fp32 products (whose weights
    need no help: the type is there to see that they stay as they were) one by one, n additions of half a step of a sum that does not
    exceed the mass.  float16 adds what may round to zero:
    2^-25 of a peak at 2^9 for each key, and in the split form 2^-25 of the peak for the at most 1,024 keys of its unit."""
    from graphgps_amd import ops
    n = 1 << 20
    g = torch.Generator().manual_seed(7)
    q, k = torch.zeros(1, 1, 2, 8), torch.zeros(n, 1, 2, 8)
    q[..., 0] = 1.0
    k[1:, :, 0, 0] = -25.6 * LN2
    v = torch.rand(n, 1, 16, generator=g) + 0.5
    q, k, v = (t.to(dtype).cuda() for t in (q, k, v))
    lam, qp, kp = torch.tensor([0.5]).cuda(), torch.tensor([0, 1], dtype=torch.int32).cuda(), torch.tensor([0, n], dtype=torch.int32).cuda()
    with torch.no_grad():
        got = ops.diff_attention(q, k, v, lam, qp, kp, scale=1.0, max_q=max_q)
    want, mass, w, _ = reference(q, k, v, lam, qp, kp, scale=1.0)
    lost = 0.0 if dtype != F16 else n * 2.0 ** -34 if max_q == 0 else 1024 * 2.0 ** -25
    close(got, want["o"], mass["o"], w + 2 * HALF[dtype] + (n + 16 if dtype == F32 else n // 32 + 64) * 2.0 ** -24 + lost, "o")
