"""A captured 8-bit step and the seed of its random bits: a checkpoint loaded into the optimizer reaches the graph."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def make(seed):
    from graphgps_amd.optim import FlatAdamW8bit
    g = torch.Generator().manual_seed(3)
    params = [torch.nn.Parameter(torch.randn(*s, generator=g).cuda()) for s in ((300,), (17, 33), (4097,))]
    return params, FlatAdamW8bit(params, lr=1e-3, max_grad_norm=1.0, seed=seed), [torch.randn(p.shape, generator=g).cuda() for p in params]


def step(params, opt, grads):
    for p, x in zip(params, grads):
        p.grad = x.clone()
    opt.step()


@pytest.mark.parametrize("seed", [11, (1 << 32) - 2])
def test_a_captured_step_follows_a_loaded_seed(seed):
    params, captured, grads = make(seed=1)
    twins, eager, _ = make(seed=seed)
    step(params, captured, grads)
    step(twins, eager, grads)
    captured.pack_grads()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured.step()
    captured.load_state_dict(eager.state_dict())
    assert captured.seed == seed
    with torch.no_grad():
        for p, t in zip(params, twins):
            p.copy_(t)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        step(twins, eager, grads)
        torch.cuda.synchronize()
        for name in ("exp_avg", "exp_avg_sq", "exp_avg_exp", "exp_avg_sq_exp"):
            assert torch.equal(getattr(captured, name), getattr(eager, name)), name
        for p, t in zip(params, twins):
            assert torch.equal(p, t)


def test_seeds_differ_and_repeat():
    codes = []
    for seed in (1, 2, 1):
        params, opt, grads = make(seed)
        step(params, opt, grads)
        codes.append(opt.exp_avg.clone())
    assert torch.equal(codes[0], codes[2]) and not torch.equal(codes[0], codes[1])
