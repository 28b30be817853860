"""Differential attention's gradients in float16, where output gradients are small (a loss without a scale) or large.

Bounds.  The relative part is test_hip_diff_attention.py's.  float16 has steps of 2^-24 below 2^-14, so a rounding there is off by up to
2^-25 whatever the value.  A result gets that once.  The kernel rounds W times 2^a and dS times 2^b: a = 13, or less where
2^a (1 + |lam|) would pass 2^15, so 2^-a <= max(2^-13, (1 + |lam|) 2^-14); b starts at 13 and falls only where a dS of the same key or
query would pass 2^15, to where that one is at least 2^12, so 2^-b <= max(2^-13, 2^-12 max|dS|).  With max|dS| <= 2 max(1, |lam|) max|dP|
(a weight is at most 1 and D is a mean of dP) and max|dP| <= max_row(|dO|_2) max_row(|v|_2), what the n (times the heads of a group)
roundings of a sum can bring is n 2^-25 2^-a max|dO| for dv, n 2^-25 2^-b s max|q| for dk and the same with |k| (and max(1, |lam|), which
dq's second map is multiplied with at the end) for dq."""
import pytest
import torch

from test_hip_diff_attention import F16, F32, HALF, make, reference, run

pytestmark = pytest.mark.gpu


def compare(got, args, do, **kw):
    q, k, v, lam = args[:4]
    want, mass, w, n = reference(*args, do=do, **kw)
    group, s = q.shape[1] // k.shape[1], kw.get("scale") or q.shape[3] ** -0.5
    rel = w + 2 * HALF[F16] + (n + 16) * 2.0 ** -24
    most = lambda t: float(t.double().abs().max())                                     # noqa: E731
    row = lambda t: float(t.double().norm(dim=-1).max())                               # noqa: E731
    big = max(1.0, most(lam))
    ds = 2.0 ** -25 * max(2.0 ** -13, 2.0 ** -12 * 2 * big * row(do) * row(v))
    floor = {"q": n * ds * s * most(k) * big, "k": n * group * ds * s * most(q),
             "v": n * group * 2.0 ** -25 * max(2.0 ** -13, (1 + most(lam)) * 2.0 ** -14) * most(do)}
    for name, t, f in (("q", got[1], 2), ("k", got[2], 2), ("v", got[3], 1)):
        off = (t.double().cpu() - want[name]).abs()
        allowed = (f * rel + (group if name in "kv" else 1) * n * 2.0 ** -24) * mass[name] + 2.0 ** -25 + floor[name]
        assert torch.isfinite(off).all(), f"d{name}: not finite"
        assert (off <= allowed).all(), f"d{name}: off by {float(off.max()):.3e}, {float((off / allowed).max()):.2f} x the bound"
    off = (got[4].double().cpu() - want["lam"]).abs()
    assert (off <= (rel + n * 2.0 ** -24 + HALF[F32]) * mass["lam"] + n * 2.0 ** -24 * n * 2.0 ** -25).all(), "dlam"


@pytest.mark.parametrize("d", [24, 64, 128])
@pytest.mark.parametrize("size", [1e-6, 1e-4, 1.0, 300.0])
@pytest.mark.parametrize("causal", [False, True])
def test_output_gradients_of_any_size(d, size, causal):
    lens = [500, 130, 3]
    q, k, v, lam, qp, kp, do = make(lens, lens, 4, 2, d, F16, seed=30)
    do = (do.float() * size).half()
    keep = (torch.rand(k.shape[0], generator=torch.Generator().manual_seed(31)) < 0.9).cuda() if causal else None
    got = run(q, k, v, lam, qp, kp, do, causal=causal, key_mask=keep)
    compare(got, (q, k, v, lam, qp, kp), do, causal=causal, keep=keep)


@pytest.mark.parametrize("d", [32, 64])
@pytest.mark.parametrize("rows", ["few_large", "last_large"])
def test_sizes_that_differ_from_row_to_row(d, rows):
    """The power of two falls on the way: small gradients before a large one, large ones among small ones."""
    lens = [300, 70]
    q, k, v, lam, qp, kp, do = make(lens, lens, 4, 2, d, F16, seed=32, std=1.5)
    size = torch.full((sum(lens),), 1e-4)
    if rows == "few_large":
        size[::37] = 100.0
    else:
        size[290:300], size[360:370] = 1000.0, 1000.0
    do = (do.float() * size[:, None, None].cuda()).half()
    got = run(q, k, v, lam, qp, kp, do)
    compare(got, (q, k, v, lam, qp, kp), do)


@pytest.mark.parametrize("d", [32, 64])
def test_weights_of_the_second_map_above_one(d):
    """Heads of a group with lam of very different sizes share a key's sums."""
    lens = [200, 33]
    q, k, v, lam, qp, kp, do = make(lens, lens, 4, 1, d, F16, seed=33)
    lam = torch.tensor([0.1, -40.0, 3.0, 300.0]).cuda()
    do = (do.float() * 0.01).half()
    got = run(q, k, v, lam, qp, kp, do)
    compare(got, (q, k, v, lam, qp, kp), do)


def test_long_rows():
    """Weights of 2^-14 and less, under small gradients: no single dS is a float16 number."""
    q, k, v, lam, qp, kp, do = make([64], [20000], 2, 1, 32, F16, seed=34)
    do = (do.float() * 1e-4).half()
    got = run(q, k, v, lam, qp, kp, do)
    compare(got, (q, k, v, lam, qp, kp), do)
