"""FlatAdamW8bit.load_state_dict: a state that does not fit is refused before anything of the optimizer has changed."""
import copy

import pytest
import torch


def make(seed=5):
    from graphgps_amd.optim import FlatAdamW8bit
    g = torch.Generator().manual_seed(1)
    params = [torch.nn.Parameter(torch.randn(*s, generator=g)) for s in ((300,), (17, 33), (5,))]
    opt = FlatAdamW8bit(params, lr=1e-3, max_grad_norm=1.0, seed=seed)
    return opt, g


def state_of(opt, g, fp32=False):
    """A state as a run of three steps might leave it."""
    state = {}
    for i, p in enumerate(opt.arena.params):
        st = dict(step=torch.tensor(3.0))
        for name in ("exp_avg", "exp_avg_sq"):
            if fp32:
                st[name] = torch.rand(p.shape, generator=g)
            else:
                st[name] = torch.randint(0, 128, p.shape, generator=g, dtype=torch.uint8)
                st[name + "_exp"] = torch.randint(90, 120, (-(-p.numel() // 256),), generator=g, dtype=torch.uint8)
        state[i] = st
    return dict(state=state, param_groups=[dict(lr=0.5, betas=(0.8, 0.9), eps=1e-6, weight_decay=0.3, max_grad_norm=2.0, params=[0, 1, 2])], seed=9)


def snapshot(opt):
    names = ("exp_avg", "exp_avg_sq", "exp_avg_exp", "exp_avg_sq_exp", "param_step", "hyper")
    group = {k: v for k, v in opt.param_groups[0].items() if k != "params"}
    return [getattr(opt, n).clone() for n in names], copy.deepcopy(group), opt.seed


def spoil(sd, how):
    if how == "last moment has another size":
        sd["state"][2]["exp_avg_sq"] = sd["state"][2]["exp_avg_sq"][:3]
    elif how == "last block count":
        sd["state"][2]["exp_avg_exp"] = torch.zeros(2, dtype=torch.uint8)
    elif how == "block exponents of another type":
        sd["state"][2]["exp_avg_exp"] = torch.zeros(1)
    elif how == "no second moment":
        del sd["state"][1]["exp_avg_sq"]
    elif how == "no exponents":
        del sd["state"][1]["exp_avg_exp"]
    elif how == "seed":
        sd["seed"] = 1 << 32
    elif how == "no group":
        sd["param_groups"] = []
    return sd


@pytest.mark.parametrize("how", ["last moment has another size", "last block count", "block exponents of another type", "no second moment",
                                 "no exponents", "seed", "no group"])
def test_a_refused_state_leaves_the_optimizer_as_it_was(how):
    opt, g = make()
    opt.load_state_dict(dict(state_of(opt, g), seed=5))
    before = snapshot(opt)
    with pytest.raises((ValueError, KeyError, IndexError)):
        opt.load_state_dict(spoil(state_of(opt, g), how))
    after = snapshot(opt)
    assert all(torch.equal(a, b) for a, b in zip(before[0], after[0])) and before[1:] == after[1:]


@pytest.mark.parametrize("fp32", [False, True])
def test_a_state_that_fits_is_taken_whole(fp32):
    opt, g = make()
    sd = state_of(opt, g, fp32)
    sd["state"].pop(1)                                   # a parameter that has not seen a gradient
    opt.load_state_dict(sd)
    got = opt.state_dict()
    assert sorted(got["state"]) == [0, 2] and opt.seed == 9 and opt.param_groups[0]["lr"] == 0.5 and float(opt.step_count) == 3
    if not fp32:
        for i in (0, 2):
            for k, v in sd["state"][i].items():
                assert torch.equal(got["state"][i][k], v), (i, k)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_moments_of_cpu_parameters_are_refused(dtype):
    """Its kernel would take their host pointers."""
    from graphgps_amd.lib import GpsHipError
    opt, g = make()
    opt.load_state_dict(state_of(opt, g))
    with pytest.raises(GpsHipError, match="on the CPU"):
        opt.moments(dtype)
