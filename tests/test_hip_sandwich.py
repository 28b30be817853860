"""ops.sandwich_norm against its definition in 64 bits.

Tolerances: everything inside is fp32, each output is rounded once to its type: half a step (2^-24, 2^-8, 2^-11) relative to the
value, plus fp32 arithmetic.  A sum over a row of D terms or over N rows is off by at most its number of sequential additions
(here: bounded by 64) times 2^-24 of its sum of magnitudes; a normalised row multiplies that by its few dozen operations.  Written
as 2^-24 * 256 of the largest magnitude met in the row (forward, row gradients) or of the column's sum of magnitudes (column
gradients); where the deviation of a row is small against its values (rstd large), the centred value loses |x| rstd 2^-24 each time."""
import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
NAMES = ("x", "a", "post_weight", "post_bias", "pre_weight", "pre_bias", "gate")


def norm(t, w, b, kind, eps):
    if w is None:
        return t
    if kind == "layer":
        t = t - t.mean(-1, keepdim=True)
    t = t / torch.sqrt(t.square().mean(-1, keepdim=True) + eps) * w
    return t if b is None else t + b


def reference(t, kind, alpha, beta, eps, dy, dz):
    f = {n: None if v is None else v.detach().double().cpu().requires_grad_(True) for n, v in t.items()}
    n = norm(f["a"], f["post_weight"], f["post_bias"], kind, eps)
    y = beta * (n if f["gate"] is None else n * f["gate"])
    y = y if f["x"] is None else y + alpha * f["x"]
    z = norm(y, f["pre_weight"], f["pre_bias"], kind, eps) if f["pre_weight"] is not None else None
    outs, couts = [y], [dy.double().cpu() if dy is not None else torch.zeros_like(y)]
    if z is not None and dz is not None:
        outs.append(z)
        couts.append(dz.double().cpu())
    leaves = [v for v in f.values() if v is not None]
    grads = dict(zip([n for n, v in f.items() if v is not None], torch.autograd.grad(outs, leaves, couts, allow_unused=True)))
    return y.detach(), None if z is None else z.detach(), grads


def make(n, d, dtype, kind, gate, post=True, pre=True, stream=True, seed=0, mean=0.0):
    g = torch.Generator().manual_seed(seed)

    def randn(*s):
        return torch.randn(*s, generator=g)
    bias = kind == "layer"
    t = dict(x=(randn(n, d) * 1.5 + mean).to(dtype) if stream else None, a=(randn(n, d) + mean).to(dtype),
             post_weight=1 + 0.2 * randn(d) if post else None, post_bias=0.1 * randn(d) if post and bias else None,
             pre_weight=1 + 0.2 * randn(d) if pre else None, pre_bias=0.1 * randn(d) if pre and bias else None,
             gate={"none": None, "channel": 0.5 + 0.2 * randn(d), "full": randn(n, d).to(dtype)}[gate])
    t = {k: None if v is None else v.cuda() for k, v in t.items()}
    return t, randn(n, d).to(dtype).cuda(), randn(n, d).to(dtype).cuda()


def run(t, kind, alpha, beta, eps, dy, dz):
    from graphgps_amd import ops
    leaves = {n: None if v is None else v.detach().requires_grad_(True) for n, v in t.items()}
    y, z = ops.sandwich_norm(leaves["x"], leaves["a"], residual_scale=alpha, branch_scale=beta, kind=kind, eps=eps,
                             **{n: leaves[n] for n in NAMES[2:]})
    outs = [(o, c) for o, c in ((y, dy), (z, dz)) if o is not None and c is not None]
    some = [v for v in leaves.values() if v is not None]
    grads = torch.autograd.grad([o for o, _ in outs], some, [c for _, c in outs], allow_unused=True)
    return y.detach(), None if z is None else z.detach(), dict(zip([n for n, v in leaves.items() if v is not None], grads))


def check(t, kind, gate, dy, dz, alpha=0.75, beta=0.5, eps=1e-5, got=None, harder=1.0):
    dtype = t["a"].dtype
    y, z, grads = got or run(t, kind, alpha, beta, eps, dy, dz)
    ry, rz, rg = reference(t, kind, alpha, beta, eps, dy, dz)
    fine = 256 * 2.0 ** -24 * harder

    def close(a, b, per_row, what):
        if b is None:
            assert a is None or (a == 0).all(), what
            return
        a, b = a.detach().double().cpu(), b.detach().double()
        assert a.shape == b.shape, (what, a.shape, b.shape)
        scale = b.abs().amax(-1, keepdim=True) if per_row else b.abs().amax()
        tol = 1.01 * HALF[dtype if per_row else F32] * b.abs() + fine * torch.clamp(scale, min=1.0 if not per_row else 1e-3)
        assert ((a - b).abs() <= tol).all(), f"{what}: off by {float((a - b).abs().max()):.2e}, {float(((a - b).abs() / tol).max()):.2f} x the bound"
    if y.numel() == 0:
        return
    close(y, ry, True, "y")
    if z is not None:
        close(z, rz, True, "z")
    assert grads.keys() == rg.keys()
    for n, r in rg.items():
        close(grads[n], r, n in ("x", "a") or (n == "gate" and gate == "full"), "d" + n)


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("d", [1, 5, 16, 48, 64, 100, 128, 257, 384, 512, 1024, 1111, 2048, 4096, 8192])
def test_widths(dtype, kind, d):
    n = 1 + 4000 // d if d < 1000 else 5
    t, dy, dz = make(n, d, dtype, kind, "channel", seed=d)
    if d == 1 and kind == "layer":       # one column: the centred row is zero, its gradient rounding noise over sqrt(eps)
        t["post_weight"] = t["post_bias"] = t["pre_weight"] = t["pre_bias"] = None
    if d == 1 and kind == "rms":         # x / |x|: the same for gradients
        t["post_weight"] = t["pre_weight"] = None
    check(t, kind, "channel", dy, dz if t["pre_weight"] is not None else None)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("gate", ["none", "channel", "full"])
@pytest.mark.parametrize("post,pre,stream", [(True, True, True), (True, False, True), (False, True, True), (False, False, True),
                                             (True, False, False), (True, True, False)])
def test_forms(dtype, kind, gate, post, pre, stream):
    t, dy, dz = make(77, 48, dtype, kind, gate, post, pre, stream, seed=1)
    check(t, kind, gate, dy, dz if pre else None)
    if pre:
        check(t, kind, gate, None, dz)           # only one of the outputs is used
        check(t, kind, gate, dy, None)


@pytest.mark.parametrize("n", [0, 1, 3, 4097, 70001])
@pytest.mark.parametrize("dtype", [F32, F16], ids=["fp32", "fp16"])
def test_row_counts(n, dtype):
    t, dy, dz = make(n, 64, dtype, "layer", "full", seed=2)
    got = run(t, "layer", 0.75, 0.5, 1e-5, dy, dz)
    if n == 0:
        assert all((g == 0).all() for g in got[2].values())
    check(t, "layer", "full", dy, dz, got=got, harder=4.0)      # 70,001 rows: up to 70 sequential additions and four tree levels more


def test_strides_and_alignment():
    """Row slices of a wider matrix, rows that start off a 16-byte boundary, transposed operands, expanded gradients, leading
    dimensions."""
    t, dy, dz = make(33, 40, F32, "rms", "full", seed=3)
    u = dict(t)
    wide = torch.zeros(33, 97, device="cuda")
    wide[:, 3:43], wide[:, 50:90] = t["x"], t["a"]
    u["x"], u["a"] = wide[:, 3:43], wide[:, 50:90]
    u["gate"] = t["gate"].t().contiguous().t()
    check(t, "rms", "full", dy, dz, got=run(u, "rms", 0.75, 0.5, 1e-5, dy, dz))
    row = dy[:1].expand(33, 40)
    check(t, "rms", "full", row, dz, got=run(t, "rms", 0.75, 0.5, 1e-5, row, dz))
    from graphgps_amd import ops
    y, z = ops.sandwich_norm(t["x"].view(3, 11, 40), t["a"].view(3, 11, 40), post_weight=t["post_weight"], pre_weight=t["pre_weight"])
    y2, z2 = ops.sandwich_norm(t["x"], t["a"], post_weight=t["post_weight"], pre_weight=t["pre_weight"])
    assert y.shape == (3, 11, 40) and torch.equal(y.view(33, 40), y2) and torch.equal(z.view(33, 40), z2)


@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_constant_and_shifted_rows(kind):
    t, dy, dz = make(9, 64, F32, kind, "none", post=False, seed=4, mean=50.0)
    check(t, kind, "none", dy, dz, harder=64.0)       # centred values lose |x| rstd = about 50 steps
    t["x"].zero_(), t["a"].zero_()                    # rows without deviation: rstd = 1 / sqrt(eps)
    y, z, _ = run(t, kind, 0.75, 0.5, 1e-5, dy, dz)
    assert (y == 0).all() and torch.isfinite(z).all()


def test_gradient_against_differences():
    from graphgps_amd import ops
    t, dy, dz = make(12, 20, F32, "layer", "channel", seed=5)
    _, _, grads = run(t, "layer", 0.75, 0.5, 1e-5, dy, dz)

    def f(u):
        y, z = ops.sandwich_norm(u["x"], u["a"], residual_scale=0.75, branch_scale=0.5, kind="layer", **{n: u[n] for n in NAMES[2:]})
        return float((y.double() * dy.double()).sum() + (z.double() * dz.double()).sum())
    g = torch.Generator().manual_seed(6)
    for n in NAMES:
        e, h = torch.randn(t[n].shape, generator=g).cuda(), 1e-2
        slope = (f({**t, n: t[n] + h * e}) - f({**t, n: t[n] - h * e})) / (2 * h)
        want = (grads[n].double() * e.double())
        assert abs(slope - float(want.sum())) <= 2e-3 * float(want.abs().sum()) + 1e-2, n


@pytest.mark.parametrize("d", [48, 2048])
def test_same_bits_every_time_captured_and_on_another_stream(d):
    t, dy, dz = make(501, d, BF16, "rms", "full", seed=7)
    first = run(t, "rms", 0.75, 0.5, 1e-5, dy, dz)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = run(t, "rms", 0.75, 0.5, 1e-5, dy, dz)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(first[1], second[1]) and all(torch.equal(first[2][n], second[2][n]) for n in first[2])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(t, "rms", 0.75, 0.5, 1e-5, dy, dz)
    for i in range(3):
        t["a"].copy_(torch.randn(t["a"].shape, generator=torch.Generator().manual_seed(i)))
        graph.replay()
        torch.cuda.synchronize()
        got = (out[1].clone(), {n: g.clone() for n, g in out[2].items()})
        want = run(t, "rms", 0.75, 0.5, 1e-5, dy, dz)
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[1]) and all(torch.equal(got[1][n], want[2][n]) for n in want[2])


def test_no_second_derivative():
    from graphgps_amd import ops
    from graphgps_amd.lib import GpsHipError
    t, dy, _ = make(5, 16, F32, "rms", "none")
    y, _ = ops.sandwich_norm(t["x"].requires_grad_(True), t["a"])
    with pytest.raises(GpsHipError, match="once"):
        torch.autograd.grad(y, t["x"], dy, create_graph=True)


@pytest.mark.parametrize("how", ["checkpoint", "offload"])
@pytest.mark.parametrize("gate", ["channel", "full"])
def test_saved_tensors_that_come_back_elsewhere(how, gate):
    """Activation checkpoints compute them anew and offloading copies them (contiguous): the gradients stay the same bits."""
    from graphgps_amd import ops
    t, dy, dz = make(301, 96, F32, "layer", gate, seed=4)
    want = run(t, "layer", 0.75, 0.5, 1e-5, dy, dz)[2]
    leaves = {n: v.detach().requires_grad_(True) for n, v in t.items()}

    def call(x, a, *rest):
        wide = torch.cat([a * 1.0, a], 1)[:, :a.shape[1]]      # rows whose stride a copy does not keep
        return ops.sandwich_norm(x * 1.0, wide, residual_scale=0.75, branch_scale=0.5, kind="layer",
                                 **{n: v * 1.0 for n, v in zip(NAMES[2:], rest)})
    args = [leaves[n] for n in NAMES]
    if how == "checkpoint":
        from torch.utils.checkpoint import checkpoint
        y, z = checkpoint(call, *args, use_reentrant=False)
    else:
        with torch.autograd.graph.save_on_cpu():
            y, z = call(*args)
    junk = [torch.full((1 << 20,), float("nan"), device="cuda") for _ in range(8)]
    got = torch.autograd.grad([y, z], args, [dy, dz])
    del junk
    for n, g in zip(NAMES, got):
        assert torch.equal(g, want[n]), n


def test_more_rows_than_one_grid_dimension_holds():
    """2^24 workgroups of 256 threads are 2^32 threads: one row per workgroup at this width, so the grid needs a second dimension."""
    from graphgps_amd import ops
    n, d = (1 << 24) + 3, 257
    a = torch.zeros(n, d, dtype=F16, device="cuda")
    some = torch.cat([torch.arange(5), (1 << 20) + torch.arange(-2, 3), torch.arange(n - 5, n)]).cuda()
    a[some] = torch.randn(len(some), d, generator=torch.Generator().manual_seed(1)).to(F16).cuda()
    w = torch.ones(d, device="cuda")
    y, _ = ops.sandwich_norm(None, a, post_weight=w)
    want, _ = ops.sandwich_norm(None, a[some], post_weight=w)
    assert torch.equal(y[some], want) and int(torch.count_nonzero(want)) > 0
