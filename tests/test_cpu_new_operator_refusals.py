"""What differential attention, the residual-stream norm and the 8-bit optimizer refuse, at the Python and at the C entries.
Refusals need no GPU: nothing is launched."""
import ctypes

import pytest
import torch

from graphgps_amd import lib, ops
from graphgps_amd.lib import DiffAttn, GpsHipError, SandwichNorm


def diff_args(nq=6, nk=6, H=4, Hk=2, d=16, dtype=torch.float32):
    p = torch.tensor([0, nq], dtype=torch.int32)
    return [torch.zeros(nq, H, 2, d, dtype=dtype), torch.zeros(nk, Hk, 2, d, dtype=dtype), torch.zeros(nk, Hk, 2 * d, dtype=dtype),
            torch.zeros(H), p, torch.tensor([0, nk], dtype=torch.int32)]


@pytest.mark.parametrize("change,text", [
    ({0: torch.zeros(6, 4, 16)}, "expected q"),
    ({0: torch.zeros(6, 4, 3, 16)}, "expected q"),
    ({1: torch.zeros(6, 2, 2, 8)}, "do not fit"),
    ({2: torch.zeros(6, 2, 16)}, "do not fit"),
    ({2: torch.zeros(5, 2, 32)}, "do not fit"),
    ({1: torch.zeros(6, 3, 2, 16), 2: torch.zeros(6, 3, 32)}, "4 heads over 3"),
    ({0: torch.zeros(6, 4, 2, 16, dtype=torch.float64)}, "must share"),
    ({1: torch.zeros(6, 2, 2, 16, dtype=torch.bfloat16)}, "must share"),
    ({3: torch.zeros(3)}, "lam must be"),
    ({3: torch.zeros(4, dtype=torch.float16)}, "lam must be"),
])
def test_diff_attention_refuses(change, text):
    a = diff_args()
    for i, t in change.items():
        a[i] = t
    with pytest.raises(GpsHipError, match=text):
        ops.diff_attention(*a)


@pytest.mark.parametrize("d", [4, 12, 136])
def test_diff_attention_refuses_head_widths(d):
    with pytest.raises(GpsHipError, match="no kernel"):
        ops.diff_attention(*diff_args(d=d))


def test_diff_attention_refuses_masks_and_cpu_tensors():
    with pytest.raises(GpsHipError, match="key_mask"):
        ops.diff_attention(*diff_args(), key_mask=torch.ones(5, dtype=torch.bool))
    with pytest.raises(GpsHipError, match="key_mask"):
        ops.diff_attention(*diff_args(), key_mask=torch.ones(6))
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(GpsHipError, match="scale"):
            ops.diff_attention(*diff_args(), scale=scale)
    with pytest.raises(GpsHipError, match="no CPU fallback"):
        ops.diff_attention(*diff_args())


def c_block(**kw):
    keep = torch.zeros(4096)
    at = keep.data_ptr() + -keep.data_ptr() % 16
    a = DiffAttn(q=at, k=at, v=at, lam=at, q_ptr=at, k_ptr=at, o=at, Nq=4, Nk=4, B=1, H=2, Hk=2, d=16, q_rs=64, q_hs=32, q_ms=16,
                 k_rs=64, k_hs=32, k_ms=16, v_rs=64, v_hs=32, scale=1.0)
    for n, v in kw.items():
        setattr(a, n, at + v if n in ("q", "k", "v", "o") and isinstance(v, int) and v else v)
    return a, keep


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=3), "dtype"), (dict(H=3), "H=3"), (dict(Hk=0), "Hk=0"), (dict(d=20), "d=20"), (dict(d=256), "d=256"), (dict(d=0), "d=0"),
    (dict(Nq=-1), "Nq=-1"), (dict(Nk=1 << 31), "Nk="), (dict(max_q=-1), "max_q"), (dict(q_ptr=None), "null"), (dict(lam=None), "null"),
    (dict(q=None), "null"), (dict(v=None), "null"), (dict(q=4), "aligned"), (dict(k_rs=63), "strides"), (dict(lse=16), "together"),
    (dict(B=-1), "B=-1"), (dict(scale=0.0), "scale")])
def test_diff_attention_c_entry_refuses(kw, text):
    L = lib.load()
    for fn in (L.gps_diff_attn_fwd, L.gps_diff_attn_bwd):
        a, _ = c_block(**kw)
        assert fn(ctypes.addressof(a), None) == -1 and text in L.gps_last_error().decode()
    assert L.gps_diff_attn_fwd(None, None) == -1


def test_diff_attention_backward_c_entry_refuses():
    L = lib.load()
    a, keep = c_block()
    at = a.q
    assert L.gps_diff_attn_bwd(ctypes.addressof(a), None) == -1 and "null" in L.gps_last_error().decode()
    for n in ("o2", "lse", "dout", "dq", "dk", "dv", "dlam"):
        setattr(a, n, at)
    assert L.gps_diff_attn_bwd(ctypes.addressof(a), None) == -1 and "workspace" in L.gps_last_error().decode()
    a.ws, a.ws_floats = at, L.gps_diff_attn_bwd_workspace_floats(4, 2, 1) - 1
    assert L.gps_diff_attn_bwd(ctypes.addressof(a), None) == -1 and "workspace" in L.gps_last_error().decode()
    a.ws_floats, a.dk_rs = 1 << 20, 12
    assert L.gps_diff_attn_bwd(ctypes.addressof(a), None) == -1 and "multiples" in L.gps_last_error().decode()
    assert L.gps_diff_attn_bwd_workspace_floats(-1, 2, 1) == 0


@pytest.mark.parametrize("kw,text", [
    (dict(kind="batch"), "neither"), (dict(a=torch.zeros(8)), r"\[\.\.\., D\]"), (dict(a=torch.zeros(2, 8, dtype=torch.float64)), "must be"),
    (dict(a=torch.zeros(2, 8193)), "no kernel"), (dict(a=torch.zeros(2, 0)), "no kernel"), (dict(x=torch.zeros(3, 8)), "x is"),
    (dict(x=torch.zeros(2, 8, dtype=torch.bfloat16)), "x is"), (dict(post_weight=torch.zeros(7)), "post_weight"),
    (dict(pre_weight=torch.zeros(8, dtype=torch.bfloat16)), "pre_weight"), (dict(post_bias=torch.zeros(8)), "without"),
    (dict(pre_bias=torch.zeros(8)), "without"), (dict(gate=torch.zeros(2, 1)), "gate"), (dict(gate=torch.zeros(8, dtype=torch.float16)), "gate"),
    (dict(), "no CPU fallback")])
def test_sandwich_norm_refuses(kw, text):
    kw = dict(dict(x=torch.zeros(2, 8), a=torch.zeros(2, 8)), **kw)
    with pytest.raises(GpsHipError, match=text):
        ops.sandwich_norm(kw.pop("x"), kw.pop("a"), **kw)


@pytest.mark.parametrize("kw,text", [(dict(dtype=5), "dtype"), (dict(kind=2), "kind"), (dict(N=-1), "N=-1"), (dict(D=0), "D=0"),
                                     (dict(D=9000), "D=9000"), (dict(a=None), "null"), (dict(gate=16, gate_full=16), "two gates")])
def test_sandwich_norm_c_entry_refuses(kw, text):
    L = lib.load()
    for fn in (L.gps_sandwich_norm_fwd, L.gps_sandwich_norm_bwd):
        b = SandwichNorm(a=16, y=16, N=4, D=8)
        for n, v in kw.items():
            setattr(b, n, v)
        assert fn(ctypes.addressof(b), None) == -1 and text in L.gps_last_error().decode()
    b = SandwichNorm(a=16, y=16, N=4, D=8, pre_weight=16)
    assert L.gps_sandwich_norm_fwd(ctypes.addressof(b), None) == -1          # z is missing
    b = SandwichNorm(a=16, da=16, N=4, D=8, pre_weight=16, ws=16, ws_floats=1 << 20)
    assert L.gps_sandwich_norm_bwd(ctypes.addressof(b), None) == -1 and "statistics" in L.gps_last_error().decode()
    b = SandwichNorm(a=16, da=16, N=4, D=8, ws=16, ws_floats=3)
    assert L.gps_sandwich_norm_bwd(ctypes.addressof(b), None) == -1 and "workspace" in L.gps_last_error().decode()


def test_optimizer_refuses():
    from graphgps_amd.optim import FlatAdamW8bit
    p = torch.nn.Parameter(torch.zeros(8))
    with pytest.raises(ValueError, match="seed"):
        FlatAdamW8bit([p], seed=-1)
    opt = FlatAdamW8bit([p])
    p.grad = torch.ones(8)
    with pytest.raises(GpsHipError, match="no CPU path"):
        opt.step()
    with pytest.raises(GpsHipError, match="neither"):
        opt.moments(torch.float16)
    flat = torch.zeros(16)
    shared = [torch.nn.Parameter(flat[:10]), torch.nn.Parameter(flat[4:])]
    with pytest.raises(ValueError, match="share"):
        FlatAdamW8bit(shared)
    with pytest.raises(ValueError, match="blocks"):
        opt.load_state_dict({"param_groups": [{"lr": 1.0}], "state": {0: dict(step=1.0, exp_avg=torch.zeros(8, dtype=torch.uint8),
                                                                              exp_avg_exp=torch.zeros(2, dtype=torch.uint8))}})
    L = lib.load()
    none = [None] * 6
    assert L.gps_adamw8_step(*none, None, None, None, None, 1, None, None, 0, None, None) == -1
    assert L.gps_adamw8_step(*none, None, None, None, None, -1, None, None, 0, None, None) == -1
    assert L.gps_adamw8_values(None, None, None, None, None, None, 1, None, None, 0, 0, None, None, None) == -1
    assert L.gps_adamw8_values(None, None, None, None, None, None, 0, None, None, 0, 2, None, None, None) == -1


def test_stored_moments_round_to_nearest():
    from graphgps_amd.optim import encode_moment
    x = torch.tensor([0.0, 1.0, -1.0, 1.0625, 1.0624, 240.0, -0.001, 3e-3] + [0.0] * 292)
    code, exp = encode_moment(x, 18)
    assert code.numel() == 300 and exp.numel() == 2 and int(exp[1]) == 0
    c = code.int()
    size = c & 127
    val = torch.where(size < 8, size.float(), ((size + 1032) << 20).view(torch.float32)) * 2.0 ** (int(exp[0]) - 127)
    val = torch.where(c >= 128, -val, val)
    assert float(val[5]) == 240.0 and float(val[1]) == 1.0 and float(val[2]) == -1.0 and float(val[3]) in (1.0, 1.125)
    assert ((val - x).abs() <= x.abs() / 16 + 2.0 ** (int(exp[0]) - 127) / 2).all()
    code, exp = encode_moment(torch.tensor([1e-12, 1.0, 0.0]), 34)
    assert int(code[0]) == 1 and int(code[2]) == 0                 # what is not zero does not become zero
    code, exp = encode_moment(torch.tensor([1.0, float("nan")]), 18)
    assert int(exp[0]) == 255 and (code == 0).all()


def test_layers_and_config():
    import math
    import os
    import graphgps_amd as g
    from graphgps_amd.layer.diff_attention_layer import DiffSelfAttention
    from graphgps_amd.layer.gps_layer import GPSLayer
    from graphgps_amd.layer.graphormer_layer import GraphormerLayer
    from graphgps_amd.optim import FlatAdamW8bit
    m = g.create_model(os.path.join(g.CONFIG_DIR, "zinc_gps_diff.yaml"), ["gt.layers", 3], 1, 1)
    assert [layer.self_attn.depth for layer in m.layers] == [0, 1, 2]
    assert abs(m.layers[2].self_attn.lam0 - (0.8 - 0.6 * math.exp(-0.6))) < 1e-12
    opt = g.register.optimizer_dict[g.cfg.optim.optimizer](m.parameters(), 1e-3, 0.01)
    assert isinstance(opt, FlatAdamW8bit) and opt.state_dict()["state"] == {}
    with pytest.raises(NotImplementedError, match="attn_dropout"):
        GPSLayer(64, "None", "DiffTransformer", 4, attn_dropout=0.1)
    for bad in ((64, 5, None), (40, 4, None), (64, 4, 3), (1024, 2, None)):
        with pytest.raises(ValueError, match="heads"):
            DiffSelfAttention(*bad)
    plain, sandwich = GraphormerLayer(80, 8, 0.0, 0.0, 0.0), GraphormerLayer(80, 8, 0.0, 0.0, 0.0, sandwich=True)
    assert set(sandwich.state_dict()) - set(plain.state_dict()) == {"attention_gate", "mlp_gate", "attention_post_norm.weight",
                                                                    "attention_post_norm.bias", "mlp_post_norm.weight",
                                                                    "mlp_post_norm.bias"}


def test_fp32_optimizer_refuses_8_bit_state():
    from graphgps_amd.optim import FlatAdamW
    p = torch.nn.Parameter(torch.zeros(5))
    opt = FlatAdamW([p])
    sd = opt.state_dict()
    sd["state"][0] = dict(step=torch.tensor(1.0), exp_avg=torch.zeros(5, dtype=torch.uint8), exp_avg_sq=torch.zeros(5, dtype=torch.uint8))
    with pytest.raises(ValueError, match="8-bit moments"):
        opt.load_state_dict(sd)
