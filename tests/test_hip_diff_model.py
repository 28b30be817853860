"""Differential attention, the residual-stream norm and the 8-bit AdamW as models use them: DiffSelfAttention, GraphormerLayer's
sandwich form, a small stack trained for a step against 64 bits, and GPSModel's training step, eager, captured and resumed.

Tolerances: fp32 through a handful of products and norms over widths of at most 64 and segments of at most 64 rows: every stage is off by
a few dozen half steps (2^-24) of its largest value, a stack of two by their sum: 1e-5 of the largest value, the project's bar."""
import math
import os

import pytest
import torch

from conftest import assert_close
from helpers import segment_attention_ref

pytestmark = pytest.mark.gpu


def batch_index(lens):
    from graphgps_amd import ops
    ptr = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device="cuda")
    gi = ops.build_graph_index(torch.zeros(2, 0, dtype=torch.int64, device="cuda"), sum(lens), len(lens), ptr_vec=ptr)
    gi.nmax_host = max(lens)
    return gi


def diff_attention_plain(m, w, x, lens):
    """DiffSelfAttention `m` with parameters `w` (any type), graph by graph."""
    H, Hk, d = m.heads, m.kv_heads, m.dim_map
    qkv = x @ w["to_qkv.weight"].T + w["to_qkv.bias"]
    q, k, v = qkv.split([2 * H * d, 2 * Hk * d, 2 * Hk * d], 1)
    a1, b1, a2, b2 = w["lam_vectors"]
    lam = torch.exp((a1 * b1).sum(-1)) - torch.exp((a2 * b2).sum(-1)) + m.lam0
    out, at = [], 0
    for n in lens:
        Q = q[at:at + n].reshape(n, Hk, H // Hk, 2, d)
        K, V = k[at:at + n].reshape(n, Hk, 2, d), v[at:at + n].reshape(n, Hk, 2 * d)
        s = torch.softmax(torch.einsum("ihgmd,jhmd->hgmij", Q, K) / math.sqrt(d), -1)
        p = s[:, :, 0] - lam.view(Hk, H // Hk, 1, 1) * s[:, :, 1]
        out.append(torch.einsum("hgij,jhe->ihge", p, V).reshape(n, H, 2 * d))
        at += n
    o = torch.cat(out)
    o = o / torch.sqrt(o.square().mean(-1, keepdim=True) + m.eps) * w["head_norm"] * (1 - m.lam0)
    return o.reshape(x.shape[0], -1) @ w["to_out.weight"].T + w["to_out.bias"]


@pytest.mark.parametrize("dim,heads,kv_heads,depth", [(64, 4, None, 0), (64, 4, 2, 3), (96, 2, 1, 1)])
def test_module_against_64_bits(dim, heads, kv_heads, depth):
    from graphgps_amd.layer.diff_attention_layer import DiffSelfAttention
    torch.manual_seed(0)
    lens = [23, 1, 40, 64, 9]
    m = DiffSelfAttention(dim, heads, kv_heads, depth).cuda()
    x = torch.randn(sum(lens), dim, device="cuda", requires_grad=True)
    g = torch.randn(sum(lens), dim, device="cuda")
    y = m.forward_segments(x, batch_index(lens))
    grads = torch.autograd.grad(y, [x, *m.parameters()], g)
    w = {n: p.detach().double().cpu().requires_grad_(True) for n, p in m.named_parameters()}
    xr = x.detach().double().cpu().requires_grad_(True)
    yr = diff_attention_plain(m, w, xr, lens)
    ref = torch.autograd.grad(yr, [xr, *w.values()], g.double().cpu())
    assert_close(y, yr, 1e-5, "y", rel_to_max=True)
    for n, a, b in zip(["x", *w], grads, ref):
        assert_close(a, b, 1e-5, f"d{n}", rel_to_max=True)


@pytest.mark.parametrize("dropout", [0.0])
def test_graphormer_sandwich_against_64_bits(dropout):
    from graphgps_amd.data import Batch
    from graphgps_amd.layer.graphormer_layer import GraphormerLayer
    torch.manual_seed(1)
    lens = [12, 30, 5]
    layer = GraphormerLayer(80, 8, dropout, 0.0, 0.0, sandwich=True).cuda()
    for p in (layer.attention_gate, layer.mlp_gate, layer.attention_post_norm.weight, layer.mlp_post_norm.weight):
        p.data += 0.2 * torch.randn_like(p)
    n = sum(lens)
    x = torch.randn(n, 80, device="cuda", requires_grad=True)
    ptr = torch.tensor([0, 12, 42, 47], device="cuda")
    b = Batch(x=x, edge_index=torch.zeros(2, 0, dtype=torch.int64, device="cuda"), ptr=ptr, num_graphs=3)
    y = layer(b).x
    g = torch.randn_like(y)
    got = torch.autograd.grad(y, [x, *layer.parameters()], g)
    w = {k: p.detach().double().cpu().requires_grad_(True) for k, p in layer.named_parameters()}
    xr = x.detach().double().cpu().requires_grad_(True)
    F = torch.nn.functional

    def ln(t, k):
        return F.layer_norm(t, (80,), w[k + ".weight"], w[k + ".bias"])
    qkv = ln(xr, "input_norm") @ w["attention.in_proj_weight"].T + w["attention.in_proj_bias"]
    o = segment_attention_ref(qkv, ptr.cpu(), 8) @ w["attention.out_proj.weight"].T + w["attention.out_proj.bias"]
    h = xr + w["attention_gate"] * ln(o, "attention_post_norm")
    m = F.gelu(ln(h, "mlp.0") @ w["mlp.1.weight"].T + w["mlp.1.bias"]) @ w["mlp.4.weight"].T + w["mlp.4.bias"]
    yr = h + w["mlp_gate"] * ln(m, "mlp_post_norm")
    ref = torch.autograd.grad(yr, [xr, *w.values()], g.double().cpu())
    assert_close(y, yr, 1e-5, "y", rel_to_max=True)
    for k, a, r in zip(["x", *w], got, ref):
        assert_close(a, r, 1e-5, f"d{k}", rel_to_max=True)


def test_a_stack_and_its_step_against_64_bits():
    """Two blocks x <- x + gate o norm(attention(norm(x))) and one clipped AdamW step from zero moments."""
    from graphgps_amd import ops
    from graphgps_amd.layer.diff_attention_layer import DiffSelfAttention
    from graphgps_amd.optim import FlatAdamW8bit
    torch.manual_seed(2)
    lens, D = [31, 17, 1, 50], 64
    gi = batch_index(lens)

    class Block(torch.nn.Module):
        def __init__(self, depth):
            super().__init__()
            self.att = DiffSelfAttention(D, 2, depth=depth)
            self.post = torch.nn.Parameter(1 + 0.1 * torch.randn(D))
            self.pre = torch.nn.Parameter(1 + 0.1 * torch.randn(D))
            self.gate = torch.nn.Parameter(0.5 + 0.1 * torch.randn(D))
    model = torch.nn.ModuleList([Block(0), Block(1)]).cuda()
    x = torch.randn(sum(lens), D, device="cuda")
    target = torch.randn(sum(lens), D, device="cuda")
    start = {k: p.detach().double().cpu() for k, p in model.named_parameters()}

    def run(x, block, att, norm):
        y, z = x, x
        for i in range(2):
            y, z = norm(y, att(i, z), block(i))
        return (z * target.to(z)).mean()
    opt = FlatAdamW8bit(model.parameters(), lr=1e-2, weight_decay=0.1, max_grad_norm=0.01)
    loss = run(x, lambda i: model[i], lambda i, z: model[i].att.forward_segments(z, gi),
               lambda y, a, b: ops.sandwich_norm(y, a, post_weight=b.post, pre_weight=b.pre, gate=b.gate, kind="rms"))
    loss.backward()
    grads = {k: p.grad.clone() for k, p in model.named_parameters()}
    opt.step()

    w = {k: p.clone().requires_grad_(True) for k, p in start.items()}

    def rms(t, g):
        return t / torch.sqrt(t.square().mean(-1, keepdim=True) + 1e-5) * g

    def sub(i, p):
        return {k[len(f"{i}.{p}"):]: v for k, v in w.items() if k.startswith(f"{i}.{p}")}

    def norm64(y, a, b):
        y = y + b["gate"] * rms(a, b["post"])
        return y, rms(y, b["pre"])
    ref = run(x.double().cpu(), lambda i: {n: w[f"{i}.{n}"] for n in ("gate", "post", "pre")},
              lambda i, z: diff_attention_plain(model[i].att, sub(i, "att."), z, lens), norm64)
    ref.backward()
    assert abs(float(loss) - float(ref)) <= 1e-5 * max(1.0, abs(float(ref)))
    big = max(float(v.grad.abs().max()) for v in w.values())
    for k in w:
        assert float((grads[k].double().cpu() - w[k].grad).abs().max()) <= 1e-5 * big, k
    o_ref = torch.optim.AdamW(w.values(), lr=1e-2, weight_decay=0.1)
    torch.nn.utils.clip_grad_norm_(w.values(), 0.01)
    o_ref.step()
    for k, p in model.named_parameters():
        # a first step moves every element by lr g / (|g| + eps'): where |g| is near the gradient's own error it may be anything in
        # +- lr, elsewhere it is lr times the sign
        sure = w[k].grad.abs() > 1e-3 * float(w[k].grad.abs().max())
        d = (p.detach().double().cpu() - w[k].detach()).abs()
        assert float(d.max()) <= 2.1e-2 and (not bool(sure.any()) or float(d[sure].max()) <= 1e-2 * 2e-2), (k, float(d[sure].max()))


def zinc_diff(layers=2):
    import graphgps_amd as g
    torch.manual_seed(0)
    m = g.create_model(os.path.join(g.CONFIG_DIR, "zinc_gps_diff.yaml"), ["gt.layers", layers], 1, 1).cuda().train()
    opt = g.register.optimizer_dict[g.cfg.optim.optimizer](m.parameters(), g.cfg.optim.base_lr, g.cfg.optim.weight_decay,
                                                           max_grad_norm=1.0)
    return m, opt


def test_gps_model_trains_eagerly_and_captured_alike():
    from graphgps_amd.loss.losses import compute_loss
    from graphgps_amd.optim import FlatAdamW8bit
    from graphgps_amd.synthetic import model_batch
    from graphgps_amd.train import TrainStep
    b = model_batch("zinc", 16, seed=7).to("cuda")
    runs = []
    for captured in (False, True):
        model, opt = zinc_diff()
        assert isinstance(opt, FlatAdamW8bit)
        ts = TrainStep(model, opt, loss_fn=compute_loss)
        if captured:
            snap = {k: v.detach().clone() for k, v in model.state_dict().items()}
            ts.capture(b.clone, warmup=2)
            with torch.no_grad():          # the warm-up steps trained the model: rewind
                for k, v in model.state_dict().items():
                    v.copy_(snap[k])
                for t in (opt.exp_avg, opt.exp_avg_sq, opt.exp_avg_exp, opt.exp_avg_sq_exp, opt.param_step):
                    t.zero_()
                opt.hyper[6].zero_()
        losses = [float(ts(b.clone())) for _ in range(4)]
        runs.append((losses, torch.cat([p.detach().reshape(-1) for p in model.parameters()]).cpu()))
        assert all(math.isfinite(x) for x in losses)
    for a, c in zip(runs[0][0], runs[1][0]):
        assert abs(a - c) <= 1e-6 * max(abs(a), 1.0), runs
    # the arenas may be laid out differently (the random bits go by offset): parameters agree to the noise of four 8-bit steps
    assert float((runs[0][1] - runs[1][1]).abs().max()) <= 4 * 2e-3


def test_gps_model_resumes_from_its_checkpoint():
    from graphgps_amd.loss.losses import compute_loss
    from graphgps_amd.synthetic import model_batch
    from graphgps_amd.train import TrainStep
    bs = [model_batch("zinc", 8, seed=20 + i).to("cuda") for i in range(4)]
    model, opt = zinc_diff(1)
    ts = TrainStep(model, opt, loss_fn=compute_loss)
    for b in bs[:2]:
        ts(b.clone())
    saved = {k: v.detach().clone() for k, v in model.state_dict().items()}, opt.state_dict()
    want = [float(ts(b.clone())) for b in bs[2:]]
    again, opt2 = zinc_diff(1)
    again.load_state_dict(saved[0])
    opt2.load_state_dict(saved[1])
    ts2 = TrainStep(again, opt2, loss_fn=compute_loss)
    got = [float(ts2(b.clone())) for b in bs[2:]]
    assert abs(want[0] - got[0]) <= 1e-6 * max(1.0, abs(want[0]))
    assert abs(want[1] - got[1]) <= 1e-5 * max(1.0, abs(want[1]))
    model.eval()
    with torch.no_grad():
        pred, _ = model(bs[0].clone())
    assert torch.isfinite(pred).all()


def test_graphormer_model_with_sandwich_runs():
    import graphgps_amd as g
    from graphgps_amd.loss.losses import compute_loss
    from graphgps_amd.synthetic import model_batch
    model = g.create_model(os.path.join(g.CONFIG_DIR, "zinc_graphormer.yaml"),
                           ["graphormer.sandwich", True, "graphormer.num_layers", 2, "dataset.node_encoder_name", "TypeDictNode",
                            "posenc_GraphormerBias.enable", False, "graphormer.use_graph_token", False, "model.graph_pooling", "mean",
                            "gnn.head", "san_graph"], 1, 1).cuda().train()
    pred, true = model(model_batch("zinc", 8, seed=3).to("cuda"))
    loss, _ = compute_loss(pred, true)
    loss.backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for n, p in model.named_parameters() if "layers" in n)
