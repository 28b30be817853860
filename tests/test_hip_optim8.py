"""FlatAdamW8bit (csrc/optim8.hip): the step against a model of it in float32 arithmetic (codes equal), the moving averages'
means, and the update against AdamW in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
M32 = 0xFFFFFFFF


def mix(x):
    x = x & M32
    x = ((x ^ (x >> 16)) * 0x7FEB352D) & M32
    x = ((x ^ (x >> 15)) * 0x846CA68B) & M32
    return x ^ (x >> 16)


def decode(code, exp, signed, block=256):
    """One parameter's codes and block exponents -> float32 values (CPU)."""
    c = code.to(torch.int32)
    size = c & 127 if signed else c
    units = torch.where(size < 8, size.float(), ((size + 1032) << 20).view(torch.float32))
    unit = (exp.to(torch.int32) << 23).view(torch.float32).repeat_interleave(block)[:len(c)]
    x = units * unit
    return torch.where((c & 128) != 0, -x, x) if signed else x


def encode(x, r16, octaves, block=256):
    n = len(x)
    pad = -n % block
    y = torch.nn.functional.pad(x, (0, pad)).view(-1, block)
    r = torch.nn.functional.pad(r16, (0, pad)).view(-1, block)
    top = y.abs().amax(-1)
    frac, e = torch.frexp(top)
    k = (e + (frac > 0.9375) - octaves).clamp(min=-126)
    u = y.abs() * ((127 - k) << 23).to(torch.int32).view(torch.float32)[:, None]
    small = torch.floor(u + r.float() * 2.0 ** -16).long()
    large = ((u.view(torch.int32).long() + (r << 4)) >> 20) - 1032
    c = torch.where(u < 8, small, large)
    if octaves == 34:
        c = torch.where((c == 0) & (u > 0), 1, c)
    else:
        c = c | ((y < 0) & (c > 0)).long() << 7
    return c.view(-1)[:n].to(torch.uint8), torch.where(top == 0, 0, k + 127).to(torch.uint8)


def model_step(p, g, m, v, step, index, norm, lr, b1, b2, eps, wd, most, seed):
    """All float32 on the CPU, one rounding per operation; `m`, `v`: (codes, exponents)."""
    f = lambda x: torch.tensor(x, dtype=torch.float64).float()   # noqa: E731
    clip = torch.clamp(f(most) / (norm + f(1e-6)), max=1.0) if most else f(1.0)
    g = g * clip
    M, V = decode(*m, True), decode(*v, False)
    M = M + f(1 - b1) * (g - M)
    V = f(b2) * V + f(1 - b2) * g * g
    p = p * f(1 - lr * wd) - f(lr / (1 - b1 ** step)) * (M / (V.sqrt() * f(1 / math.sqrt(1 - b2 ** step)) + f(eps)))
    key = int(mix(torch.tensor(((step * 0x9E3779B9) & M32) + seed)))
    bits = mix(index + key)
    return p, encode(M, bits & 0xFFFF, 18), encode(V, bits >> 16, 34), M, V


def make(sizes, seed=0):
    g = torch.Generator().manual_seed(seed)
    params = [torch.nn.Parameter(torch.randn(*s, generator=g).cuda()) for s in sizes]
    return params, g


SIZES = [(300,), (1,), (17, 33), (4096,), (4097,), (3, 5000), (256,), (255,), (12289,)]


@pytest.mark.parametrize("max_norm", [None, 1.0])
@pytest.mark.parametrize("stacked", [False, True])
def test_codes_equal_the_model(max_norm, stacked):
    from graphgps_amd.optim import FlatAdamW8bit
    params, g = make(SIZES)
    if stacked:         # parameters of one storage at odd offsets keep them: unaligned blocks
        flat = torch.cat([p.detach().reshape(-1) for p in params])
        at = 0
        for p in params:
            p.data = flat[at:at + p.numel()].view(p.shape)
            at += p.numel()
    opt = FlatAdamW8bit(params, lr=3e-3, weight_decay=0.02, max_grad_norm=max_norm, seed=7)
    a = opt.arena
    model = [(p.detach().cpu().reshape(-1), (torch.zeros(p.numel(), dtype=torch.uint8), torch.zeros(-(-p.numel() // 256), dtype=torch.uint8)),
              (torch.zeros(p.numel(), dtype=torch.uint8), torch.zeros(-(-p.numel() // 256), dtype=torch.uint8))) for p in params]
    steps = [0] * len(params)
    for it in range(5):
        for i, p in enumerate(params):
            p.grad = None
            if it == 2 and i in (1, 3):       # no gradient this step: nothing moves
                continue
            scale = torch.exp(3 * torch.randn(p.shape, generator=g))
            p.grad = (torch.randn(p.shape, generator=g) * scale * 10.0 ** -(it + i % 3)).cuda()
            if i == 6:
                p.grad.zero_()
        opt.step()
        norm = opt.total_norm.float().cpu()
        want_norm = math.sqrt(sum(float(p.grad.double().square().sum()) for p in params if p.grad is not None))
        assert abs(float(norm) - want_norm) <= 1e-6 * want_norm
        for i, (p, (b, nb)) in enumerate(zip(params, opt._block_ranges())):
            if p.grad is not None:
                steps[i] += 1
                o = a.offsets[i]
                pm, m, v, _, _ = model_step(model[i][0], p.grad.cpu().reshape(-1), model[i][1], model[i][2], steps[i],
                                            torch.arange(o, o + p.numel()), norm, 3e-3, 0.9, 0.999, 1e-8, 0.02, max_norm, 7)
                model[i] = (pm, m, v)
            o, k = a.offsets[i], p.numel()
            got = p.detach().cpu().reshape(-1)
            # the model's own result, but for the order of p's last additions: two half steps
            assert (got - model[i][0]).abs().max() <= 2.0 ** -23 * max(1.0, float(model[i][0].abs().max())), (it, i)
            model[i] = (got, *model[i][1:])
            for name, (code, exp) in (("exp_avg", model[i][1]), ("exp_avg_sq", model[i][2])):
                assert torch.equal(getattr(opt, name + "_exp")[b:b + nb].cpu(), exp), (it, i, name)
                assert torch.equal(getattr(opt, name)[o:o + k].cpu(), code), (it, i, name)
    for dtype in (torch.bfloat16, torch.float32):
        mo, vo = opt.moments(dtype)
        covered = torch.zeros(mo.numel(), dtype=torch.bool)
        for i, p in enumerate(params):
            o, k = a.offsets[i], p.numel()
            covered[o:o + k] = True
            assert torch.equal(mo[o:o + k].float().cpu(), decode(*model[i][1], True))
            assert torch.equal(vo[o:o + k].float().cpu(), decode(*model[i][2], False))
        assert (mo.cpu()[~covered] == 0).all() and (vo.cpu()[~covered] == 0).all()


def test_one_step_is_adamw_from_the_same_moments():
    """The update uses the moments before they are rounded: a first step (zero moments) is AdamW's, to fp32 rounding."""
    from graphgps_amd.optim import FlatAdamW8bit
    params, g = make(SIZES, 1)
    ref = [p.detach().double().cpu().requires_grad_(True) for p in params]
    o_ref = torch.optim.AdamW(ref, lr=1e-2, weight_decay=0.1)
    opt = FlatAdamW8bit(params, lr=1e-2, weight_decay=0.1)
    for p, r in zip(params, ref):
        r.grad = torch.randn(p.shape, generator=g).double()
        p.grad = r.grad.float().cuda()
    opt.step(), o_ref.step()
    for p, r in zip(params, ref):
        # p and the update each lose a few half steps; updates are lr-sized
        assert ((p.detach().double().cpu() - r.detach()).abs() <= 4 * 2.0 ** -24 * (r.detach().abs() + 1e-2) + 1e-9).all()


def test_moving_averages_keep_their_mean():
    """A constant gradient: exp_avg_sq grows by 1 / 1000 of the way per step, far below half a code.  Rounding to nearest would
    stay where it is; here the mean over 8,192 equal elements follows b2's average.  One rounding has a deviation of at most half a
    step, 1 / 16 of the value; over 400 steps of the average at most sqrt(400) of them add up (fewer: they decay): 1.25 values per
    element, 0.0138 for the mean; four deviations."""
    from graphgps_amd.optim import FlatAdamW8bit
    p = torch.nn.Parameter(torch.zeros(8192, device="cuda"))
    opt = FlatAdamW8bit([p], lr=0.0, weight_decay=0.0, seed=3)
    for _ in range(400):
        p.grad = torch.full((8192,), 0.5, device="cuda")
        opt.step()
    m, v = opt.moments(torch.float32)
    want = 0.25 * (1 - 0.999 ** 400)
    assert abs(float(v.mean()) / want - 1) < 4 * 0.0138
    assert abs(float(m.mean()) / 0.5 - 1) < 4 * 0.0138
    opt2 = FlatAdamW8bit([torch.nn.Parameter(torch.zeros(8192, device="cuda"))], lr=0.0, seed=4)
    assert opt2.seed == 4 and (opt2.exp_avg == 0).all()


def test_extremes():
    """Zero, subnormal, largest and non-finite gradients."""
    from graphgps_amd.optim import FlatAdamW8bit
    p = torch.nn.Parameter(torch.ones(1024, device="cuda"))
    opt = FlatAdamW8bit([p], lr=1e-3, weight_decay=0.0)
    g = torch.zeros(1024)
    g[256:512] = 1e-30
    g[300] = 1e-41
    g[512:768] = 1e18
    g[768:] = 1.0
    g[800] = float("inf")
    p.grad = g.cuda()
    opt.step()
    m, v = (t.float().cpu() for t in opt.moments())
    assert (m[:256] == 0).all() and (p.detach()[:256] == 1).all()
    assert torch.isfinite(m[:768]).all() and torch.isfinite(v[:768]).all() and torch.isfinite(p.detach()[:768]).all()
    assert (v[512:768] > 0).all() and torch.isnan(m[768:]).all()
    assert torch.isfinite(p.detach().cpu()[768:800]).all() and not torch.isfinite(p.detach().cpu()[800])


@pytest.mark.parametrize("from_fp32", [False, True])
def test_checkpoints(from_fp32):
    from graphgps_amd.optim import FlatAdamW, FlatAdamW8bit
    params, g = make(SIZES, 2)
    first = (FlatAdamW if from_fp32 else FlatAdamW8bit)(params, lr=1e-3)
    grads = [[torch.randn(p.shape, generator=g).cuda() for p in params] for _ in range(4)]

    def steps(opt, ps, which):
        for w in which:
            for p, gr in zip(ps, grads[w]):
                p.grad = gr.clone()
            opt.step()
    steps(first, params, (0, 1))
    sd = first.state_dict()
    again = [torch.nn.Parameter(p.detach().clone()) for p in params]
    second = FlatAdamW8bit(again, lr=5.0)
    second.load_state_dict(sd)
    assert second.param_groups[0]["lr"] == 1e-3 and float(second.step_count) == 2
    if not from_fp32:
        steps(first, params, (2, 3))
        steps(second, again, (2, 3))
        for a, b in zip(params, again):
            assert torch.equal(a, b)
        for n in ("exp_avg", "exp_avg_sq"):
            for i, p in enumerate(params):
                x, y = (o.state_dict()["state"][i][n] for o in (first, second))
                assert torch.equal(x, y)
        return
    for i, p in enumerate(params):
        o, k = second.arena.offsets[i], p.numel()
        for t, n in zip(second.moments(torch.float32), ("exp_avg", "exp_avg_sq")):
            want = sd["state"][i][n].reshape(-1)
            # half a step of three mantissa bits; below 8 units half a unit, a unit being 2^-17 (2^-33) of the block's largest or less
            # (values of exp_avg_sq under half a unit become one)
            unit = float(want.abs().max()) * (2.0 ** -17 if n == "exp_avg" else 2.0 ** -33)
            assert ((t[o:o + k] - want).abs() <= want.abs() * 2.0 ** -4 + unit).all()


def test_parameters_that_move_and_captured_steps():
    """The arena follows moved parameters; a captured step replays with fresh random bits and equals the eager one."""
    from graphgps_amd.optim import FlatAdamW8bit
    params, g = make(SIZES, 3)
    twin = [torch.nn.Parameter(p.detach().clone()) for p in params]
    a, b = FlatAdamW8bit(params, lr=1e-3, max_grad_norm=1.0), FlatAdamW8bit(twin, lr=1e-3, max_grad_norm=1.0)
    gr = [torch.randn(p.shape, generator=g).cuda() for p in params]

    def set_grads(ps):
        for p, x in zip(ps, gr):
            p.grad = x.clone()
    for ps, o in ((params, a), (twin, b)):
        set_grads(ps)
        o.step()
    graph = torch.cuda.CUDAGraph()
    a.pack_grads()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        a.step()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        set_grads(twin)
        b.step()
        torch.cuda.synchronize()
        for x, y in zip(params, twin):
            assert torch.equal(x, y)
        assert torch.equal(a.exp_avg, b.exp_avg) and torch.equal(a.exp_avg_sq_exp, b.exp_avg_sq_exp)
    codes = {i: v["exp_avg"] for i, v in b.state_dict()["state"].items()}
    twin[2].data = twin[2].data.clone()               # moved out of the arena: the state follows
    set_grads(twin)
    b.pack_grads()
    for i, v in b.state_dict()["state"].items():
        assert torch.equal(v["exp_avg"], codes[i])
    b.step()
    set_grads(params)
    a.step()
    torch.cuda.synchronize()
    for x, y in zip(params, twin):
        # the arena offsets differ now, so the codes do; the update itself uses the unrounded moments
        assert (x - y).abs().max() <= 2.0 ** -22 * float(x.abs().max())


def test_parameters_without_elements():
    """More parameters than chunks: the empty ones have no chunk, and nothing of theirs is touched."""
    from graphgps_amd.optim import FlatAdamW8bit
    g = torch.Generator().manual_seed(3)
    start, grads = torch.randn(700, generator=g), torch.randn(3, 700, generator=g)
    out = []
    for empties in (0, 5000):
        params = [torch.nn.Parameter(torch.zeros(0, 4, device="cuda")) for _ in range(empties)] + [torch.nn.Parameter(start.cuda())]
        opt = FlatAdamW8bit(params, lr=1e-2, max_grad_norm=1.0)
        for gr in grads:
            for p in params:
                p.grad = torch.zeros_like(p)
            params[-1].grad = gr.cuda()
            opt.step()
        state = opt.state_dict()["state"]
        assert list(state) == [empties] and float(state[empties]["step"]) == 3
        out.append((params[-1].detach(), state[empties]))
        again = FlatAdamW8bit(params)
        again.load_state_dict(opt.state_dict())
        for a, b in zip(again.moments(), opt.moments()):
            assert torch.equal(a, b)
    (p0, s0), (p1, s1) = out
    assert torch.equal(p0, p1) and all(torch.equal(s0[k], s1[k]) for k in ("exp_avg_sq_exp", "exp_avg_exp"))
