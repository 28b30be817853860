"""Workloads of three operators, in a plain form and as the framework's own calls, for timing and comparing them.

``diff``: differential attention over ragged segments, ``o = (softmax(s q1 k1^T) - lam softmax(s q2 k2^T)) v`` per head.
``norm``: the residual stream of a block, ``y = alpha x + beta gate * norm(a)`` and ``z = norm(y)`` in one pass.
``adamw``: clip + AdamW over a parameter arena with both moments held in 8 bits (stochastic rounding, blocks of 256).
"""
import math
import random

import torch

own = False

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_BLOCK = 256


# ---------------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one training step's attention over a batch of molecules (256 graphs of ~30 nodes, width 384)
        dict(name="molecules_train", op="diff", form="train", dtype="fp32", segments=256, mean=30, spread=0.25, one_query=False,
             heads=8, kv_heads=8, dim=24, causal=False, masked=False, packed=True, lens=1),
        # the same for syntax trees of ~125 nodes, width 256
        dict(name="trees_train", op="diff", form="train", dtype="bf16", segments=32, mean=125, spread=0.6, one_query=False,
             heads=4, kv_heads=4, dim=32, causal=False, masked=False, packed=True, lens=2),
        # training on two large graphs, shared key heads
        dict(name="large_graphs_train", op="diff", form="train", dtype="bf16", segments=2, mean=4097, spread=0.2, one_query=False,
             heads=8, kv_heads=4, dim=64, causal=False, masked=False, packed=False, lens=3),
        # inference over ordered sequences with dropped keys, wide heads
        dict(name="ordered_infer", op="diff", form="infer", dtype="fp16", segments=4, mean=2501, spread=0.3, one_query=False,
             heads=6, kv_heads=2, dim=128, causal=True, masked=True, packed=False, lens=4),
        # one read-out query for each tree: few rows, where latency counts
        dict(name="readout_infer", op="diff", form="infer", dtype="fp32", segments=32, mean=125, spread=0.6, one_query=True,
             heads=4, kv_heads=4, dim=32, causal=False, masked=False, packed=False, lens=5),
        # one new token for each of eight long cached sequences
        dict(name="long_cache_infer", op="diff", form="infer", dtype="bf16", segments=8, mean=33001, spread=0.4, one_query=True,
             heads=8, kv_heads=2, dim=64, causal=False, masked=False, packed=False, lens=6),
        # a few node rows of a small model at inference
        dict(name="few_rows_infer", op="norm", form="infer", dtype="fp32", rows=737, width=64, kind="layer", gate="none"),
        # the stream of the molecule model in training
        dict(name="stream_train", op="norm", form="train", dtype="fp32", rows=7681, width=384, kind="layer", gate="channel"),
        # many rows in 16 bits with a gate for every element
        dict(name="wide_stream_train", op="norm", form="train", dtype="bf16", rows=50001, width=2048, kind="rms", gate="full"),
        # parameters of a small model, a medium one (19 M), a large one
        dict(name="small_model_step", op="adamw", tensors=40, params=600_011, seed_of_sizes=1),
        dict(name="medium_model_step", op="adamw", tensors=60, params=19_400_003, seed_of_sizes=2),
        dict(name="large_model_step", op="adamw", tensors=48, params=200_000_033, seed_of_sizes=3),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["diff", "diff", "diff", "norm", "norm", "adamw"])
    if op == "norm":
        width = rng.choice([16, 48, 64, 80, 100, 256, 384, 514, 768, 1024, 1111, 2048])
        return dict(op="norm", form=rng.choice(["infer", "train", "train"]), dtype=rng.choice(sorted(_TYPES)),
                    rows=_log(rng, 1, 90_000_000 // width // 2), width=width, kind=rng.choice(["rms", "layer"]),
                    gate=rng.choice(["none", "channel", "full"]))
    if op == "adamw":
        return dict(op="adamw", tensors=rng.randint(1, 60), params=_log(rng, 1000, 100_000_000), seed_of_sizes=rng.randrange(1 << 30))
    kv_heads = rng.choice([1, 2, 3, 4])
    heads = kv_heads * rng.choice([4, 8] if kv_heads == 1 else [2, 4] if kv_heads < 4 else [1, 2])
    dim = rng.choice([8, 16, 24, 32, 40, 64, 96, 128])
    one_query = rng.random() < 0.3
    form = "infer" if one_query else rng.choice(["train", "train", "infer"])
    segments = _log(rng, 1, 300)
    most = 264_000 // segments if one_query else int(math.sqrt(20e6 / segments * 8 / heads * 64 / max(dim, 64)))
    least = 8 if form == "train" else 1      # a softmax over one key has no gradient but rounding noise
    return dict(op="diff", form=form, dtype=rng.choice(sorted(_TYPES)), segments=segments, mean=max(least, min(_log(rng, least, 40_000), most)),
                spread=rng.choice([0.0, 0.2, 0.5]), one_query=one_query, heads=heads, kv_heads=kv_heads, dim=dim,
                causal=rng.random() < 0.3, masked=rng.random() < 0.3, packed=not one_query and rng.random() < 0.5, lens=rng.randrange(1 << 30))


def _lengths(case):
    """Key rows of each segment: spread around the mean, no longer than 2.5 times it."""
    r = random.Random(case["lens"])
    return [max(1, min(int(2.5 * case["mean"]), round(case["mean"] * math.exp(r.gauss(0.0, case["spread"]))))) for _ in range(case["segments"])]


def _sizes(case):
    """Element counts of the parameter tensors: a few large ones, many small ones, together about `params`; the last one ends
    with its block."""
    r = random.Random(case["seed_of_sizes"])
    w = [math.exp(r.gauss(0.0, 2.0)) for _ in range(case["tensors"])]
    sizes = [max(1, int(case["params"] * x / sum(w))) for x in w]
    return sizes[:-1] + [-(-sizes[-1] // _BLOCK) * _BLOCK]


def work(case):
    if case["op"] == "norm":
        n, d = case["rows"], case["width"]
        e, full = (4 if case["dtype"] == "fp32" else 2), case["gate"] == "full"
        b, f = 4 * n * d * e + (n * d * e if full else 0), 16.0 * n * d     # x, a -> y, z
        if case["form"] == "train":
            b, f = b + 4 * n * d * e + (n * d * e if full else 0), f + 40.0 * n * d  # dy, dz -> dx, da
        return {"bytes": float(b), "flops": f}
    if case["op"] == "adamw":
        n = sum(_sizes(case))
        return {"bytes": n * (12.0 + 4.0 + 4.0), "flops": 60.0 * n}      # p both ways, g; codes both ways; both moments as values
    ks = _lengths(case)
    qs = [1] * len(ks) if case["one_query"] else ks
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    e = 4 if case["dtype"] == "fp32" else 2
    pairs = float(sum(q * k if not case["causal"] else sum(max(0, k - q + i + 1) for i in range(q)) for q, k in zip(qs, ks)))
    qo, kv = sum(qs) * h * 2 * d, sum(ks) * hk * 4 * d
    b, f = e * (2 * qo + kv), pairs * h * 8 * d
    if case["form"] == "train":
        b, f = b + e * (2 * qo + kv), f + pairs * h * 16 * d             # o, do -> dq, dk, dv
    return {"bytes": float(b), "flops": f}


# --------------------------------------------------------------------------------------------------------- the inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed) * 1000003 + 17)

    def randn(*shape, dtype=torch.float32, std=1.0):
        return (torch.randn(*shape, generator=g, device=dev) * std).to(dtype)

    s = dict(case)
    if case["op"] == "norm":
        n, d, t, train = case["rows"], case["width"], _TYPES[case["dtype"]], case["form"] == "train"
        s["x"], s["a"] = randn(n, d, dtype=t, std=1.5), randn(n, d, dtype=t, std=0.7)
        s["post_weight"], s["pre_weight"] = 1.0 + randn(d, std=0.2), 1.0 + randn(d, std=0.2)
        s["post_bias"] = randn(d, std=0.1) if case["kind"] == "layer" else None
        s["pre_bias"] = randn(d, std=0.1) if case["kind"] == "layer" else None
        s["gate"] = {"none": lambda: None, "channel": lambda: 0.5 + randn(d, std=0.2), "full": lambda: randn(n, d, dtype=t)}[case["gate"]]()
        s["leaves"] = ["x", "a"] + [k for k in ("post_weight", "post_bias", "pre_weight", "pre_bias", "gate") if s[k] is not None]
        if train:
            s["dy"], s["dz"] = randn(n, d, dtype=t), randn(n, d, dtype=t)
            for k in s["leaves"]:
                s[k].requires_grad_(True)
        return s
    if case["op"] == "adamw":
        sizes = _sizes(case)
        spans = [-(-n // _BLOCK) * _BLOCK for n in sizes]
        at, n = [sum(spans[:i]) for i in range(len(spans))], sum(spans)
        s["at"], s["sizes"], s["step"] = at, sizes, 100
        keep = torch.zeros(n, device=dev)
        for o, k in zip(at, sizes):
            keep[o:o + k] = 1.0
        s["p"], s["g"] = randn(n, std=0.05) * keep, randn(n, std=1e-3) * keep
        # gradient scales that differ from tensor to tensor and from element to element, as they do in a model
        s["g"] *= torch.exp(randn(n, std=1.0))
        s["hyper"] = dict(lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, max_grad_norm=1.0)
        half = torch.full((n // _BLOCK, _BLOCK), 32768, dtype=torch.int64, device=dev)
        s["m_code"], s["m_exp"] = _encode((s["g"] * 0.3 + randn(n, std=3e-4) * keep).view(-1, _BLOCK), half, 18)
        s["v_code"], s["v_exp"] = _encode((s["g"].square() * 0.5 + randn(n, std=3e-4).square() * keep).view(-1, _BLOCK), half, 34)
        if own:
            from graphgps_amd.optim import FlatAdamW8bit
            s["tensors"] = [torch.nn.Parameter(s["p"][o:o + k]) for o, k in zip(at, sizes)]
            s["opt"] = FlatAdamW8bit(s["tensors"], **s["hyper"])
            state = {}
            for i, (o, k) in enumerate(zip(at, sizes)):
                b = slice(o // _BLOCK, o // _BLOCK + -(-k // _BLOCK))
                state[i] = dict(step=torch.tensor(100.0), exp_avg=s["m_code"].view(-1)[o:o + k], exp_avg_exp=s["m_exp"][b],
                                exp_avg_sq=s["v_code"].view(-1)[o:o + k], exp_avg_sq_exp=s["v_exp"][b])
                s["tensors"][i].grad = s["g"][o:o + k]
            s["opt"].load_state_dict(dict(state=state, param_groups=[dict(s["hyper"], params=list(range(len(sizes))))]))
        return s
    ks = _lengths(case)
    qs = [1] * len(ks) if case["one_query"] else ks
    h, hk, d, t = case["heads"], case["kv_heads"], case["dim"], _TYPES[case["dtype"]]
    tail = 3 if case["masked"] and not case["packed"] else 0             # rows behind the last segment
    nq, nk = sum(qs) + tail, sum(ks) + tail
    if case["packed"]:
        s["qkv"] = randn(nk, 2 * h * d + 4 * hk * d, dtype=t)
        s["leaves"] = ["qkv", "lam"]
    else:
        s["q"], s["k"], s["v"] = randn(nq, h, 2, d, dtype=t), randn(nk, hk, 2, d, dtype=t), randn(nk, hk, 2 * d, dtype=t)
        s["leaves"] = ["q", "k", "v", "lam"]
    s["lam"] = (0.1 + 0.8 * torch.rand(h, generator=g, device=dev)).to(t)
    s["q_ptr"] = torch.tensor([sum(qs[:i]) for i in range(len(qs) + 1)], dtype=torch.int32, device=dev)
    s["k_ptr"] = torch.tensor([sum(ks[:i]) for i in range(len(ks) + 1)], dtype=torch.int32, device=dev)
    s["max_q"], s["max_k"], s["rows_q"], s["rows_k"], s["nq"] = max(qs), max(ks), sum(qs), sum(ks), nq
    s["keep"] = None
    if case["masked"]:
        s["keep"] = torch.rand(nk, generator=g, device=dev) < 0.8
        if len(ks) > 1:
            s["keep"][:ks[0]] = False                                    # nothing to attend to in the first segment
    if case["form"] == "train":
        s["do"] = randn(nq, h, 2 * d, dtype=t)
        for k in s["leaves"]:
            s[k].requires_grad_(True)
    if own and case["packed"]:
        from graphgps_amd.ops import build_graph_index
        s["index"] = build_graph_index(torch.zeros(2, 0, dtype=torch.int64, device=dev), nk, len(ks), ptr_vec=s["k_ptr"])
        s["index"].nmax_host = s["max_k"]
    return s


# ----------------------------------------------------------------------------------------------------- the plain forms
def _places(ptr, longest, rows):
    """Where each of the first `rows` rows goes in [segments * longest], which places hold one, and the lengths."""
    n = (ptr[1:] - ptr[:-1]).long()
    i = torch.arange(rows, device=ptr.device)
    segment = torch.repeat_interleave(torch.arange(len(n), device=ptr.device), n, output_size=rows)
    return segment * longest + i - ptr.long()[segment], torch.arange(longest, device=ptr.device)[None, :] < n[:, None], n


def _spread(t, to, segments, longest):
    out = torch.zeros(segments * longest, *t.shape[1:], dtype=t.dtype, device=t.device)
    return out.index_copy(0, to, t[:len(to)]).view(segments, longest, *t.shape[1:])


def _diff_plain(q, k, v, lam, s):
    """Dense over [segments, heads, queries, keys], padded to the longest segment; float32 or wider in, the same out."""
    h, hk, d = s["heads"], s["kv_heads"], s["dim"]
    mq, mk = s["max_q"], s["max_k"]
    to_q, ok_q, nq = _places(s["q_ptr"], mq, s["rows_q"])
    to_k, ok_k, nk = _places(s["k_ptr"], mk, s["rows_k"])
    if s["keep"] is not None:
        ok_k = ok_k & _spread(s["keep"], to_k, len(nk), mk)
    see = ok_q[:, :, None] & ok_k[:, None, :]
    if s["causal"]:
        i, j = torch.arange(mq, device=q.device), torch.arange(mk, device=q.device)
        see = see & (j[None, None, :] <= (i[None, :] + (nk - nq)[:, None])[:, :, None])
    see = see[:, None, None, None]                                       # over [segment, kv head, head of the group, map]
    qd = _spread(q, to_q, len(nq), mq).view(len(nq), mq, hk, h // hk, 2, d).permute(0, 2, 3, 4, 1, 5)
    kd = _spread(k, to_k, len(nk), mk).permute(0, 2, 3, 4, 1)[:, :, None].contiguous()         # [segment, kv head, 1, map, d, keys]
    vd = _spread(v, to_k, len(nk), mk).permute(0, 2, 1, 3)[:, :, None].contiguous()
    w = torch.matmul(qd, kd) * d ** -0.5
    w = w.masked_fill(~see, -math.inf)
    top = w.detach().amax(-1, keepdim=True)
    w = torch.exp(w - top.masked_fill(top == -math.inf, 0.0))
    total = w.sum(-1, keepdim=True)
    w = w / total.masked_fill(total == 0, 1.0)
    w = w[:, :, :, 0] - lam.view(1, hk, h // hk, 1, 1) * w[:, :, :, 1]
    o = torch.matmul(w, vd).permute(0, 3, 1, 2, 4).reshape(len(nq) * mq, h, 2 * d)
    o = o.index_select(0, to_q)
    return torch.cat([o, o.new_zeros(s["nq"] - len(to_q), h, 2 * d)]) if s["nq"] > len(to_q) else o


def _unpack(qkv, s):
    h, hk, d = s["heads"], s["kv_heads"], s["dim"]
    q, k, v = qkv.split([2 * h * d, 2 * hk * d, 2 * hk * d], 1)
    return q.reshape(-1, h, 2, d), k.reshape(-1, hk, 2, d), v.reshape(-1, hk, 2 * d)


def _norm_one(t, weight, bias, kind, eps):
    if kind == "layer":
        t = t - t.mean(-1, keepdim=True)
    t = t * torch.rsqrt(t.square().mean(-1, keepdim=True) + eps) * weight
    return t if bias is None else t + bias


def _norm_plain(f, s):
    n = _norm_one(f["a"], f["post_weight"], f.get("post_bias"), s["kind"], 1e-5)
    y = 0.75 * f["x"] + 0.5 * (n if s["gate"] is None else n * f["gate"])
    return y, _norm_one(y, f["pre_weight"], f.get("pre_bias"), s["kind"], 1e-5)


def _mix(x):
    x = x & 0xFFFFFFFF
    x = ((x ^ (x >> 16)) * 0x7FEB352D) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0x846CA68B) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _random_bits(n, step, device):
    """One 32-bit word for each element and step."""
    key = _mix(torch.tensor((step * 0x9E3779B9) & 0xFFFFFFFF, device=device))
    return _mix(torch.arange(n, device=device) + key)


def _encode(x, r16, octaves):
    """Blocks of 256 values -> codes with three bits of mantissa and one exponent for the block.

    The unit 2^k of a block is the smallest that keeps its largest value within 15 * 2^(octaves - 4) units.  A magnitude of y units
    is floor(y + r) below 8 units; above, its float's mantissa is cut to three bits after r * 2^-16 of a step has been added."""
    size = x.abs()
    a, e = torch.frexp(size.amax(-1))
    k = (e + (a > 0.9375) - octaves).clamp(min=-126)
    unit = ((127 - k) << 23).to(torch.int32).view(torch.float32)
    y = size * unit[:, None]
    small = torch.floor(y + r16.to(torch.float32) * 2.0 ** -16).to(torch.int64)
    large = ((y.view(torch.int32).to(torch.int64) + (r16 << 4)) >> 20) - 1032
    code = torch.where(y < 8, small, large)
    if octaves == 34:
        code = torch.where((code == 0) & (y > 0), torch.ones_like(code), code)
    else:
        code = code | ((x < 0) & (code > 0)).to(torch.int64) << 7
    none = size.amax(-1) == 0
    return code.to(torch.uint8), torch.where(none, torch.zeros_like(k), k + 127).to(torch.uint8)


def _decode(code, exponent, signed):
    c = code.to(torch.int32)
    size = c & 127 if signed else c
    units = torch.where(size < 8, size.to(torch.float32), ((size + 1032) << 20).view(torch.float32))
    x = units * (exponent.to(torch.int32) << 23).view(torch.float32)[:, None]
    return torch.where((c & 128) != 0, -x, x) if signed else x


def _adamw_plain(s):
    hy, (b1, b2) = s["hyper"], s["hyper"]["betas"]
    s["step"] += 1
    step = s["step"]
    norm = s["g"].double().square().sum().sqrt().float()
    g = s["g"] * torch.clamp(hy["max_grad_norm"] / (norm + 1e-6), max=1.0)
    m = _decode(s["m_code"], s["m_exp"], True).view(-1)
    v = _decode(s["v_code"], s["v_exp"], False).view(-1)
    m = m + (1 - b1) * (g - m)
    v = b2 * v + (1 - b2) * g * g
    s["p"] = s["p"] * (1 - hy["lr"] * hy["weight_decay"]) - hy["lr"] / (1 - b1 ** step) * (
        m / (v.sqrt() * (1 / math.sqrt(1 - b2 ** step)) + hy["eps"]))
    bits = _random_bits(m.numel(), step, m.device).view(-1, _BLOCK)
    s["m_code"], s["m_exp"] = _encode(m.view(-1, _BLOCK), bits & 0xFFFF, 18)
    s["v_code"], s["v_exp"] = _encode(v.view(-1, _BLOCK), bits >> 16, 34)
    # a value is four significant bits times a power of two: bfloat16 holds it exactly
    return [s["p"], _decode(s["m_code"], s["m_exp"], True).view(-1).bfloat16(), _decode(s["v_code"], s["v_exp"], False).view(-1).bfloat16()]


# ------------------------------------------------------------------------------------------------------------ one pass
def _run_plain(s):
    if s["op"] == "adamw":
        return _adamw_plain(s)
    train = s["form"] == "train"
    wide = {k: s[k].detach().float().requires_grad_(train) for k in s["leaves"]}
    if s["op"] == "norm":
        outs, couts = _norm_plain(wide, s), [s["dy"].float(), s["dz"].float()] if train else None
        types = [s["x"].dtype] * 2
    else:
        q, k, v = _unpack(wide["qkv"], s) if s["packed"] else (wide["q"], wide["k"], wide["v"])
        outs, couts = [_diff_plain(q, k, v, wide["lam"], s)], [s["do"].float()] if train else None
        types = [s["lam"].dtype]
    got = [o.detach().to(t) for o, t in zip(outs, types)]
    if train:
        grads = torch.autograd.grad(outs, [wide[k] for k in s["leaves"]], couts)
        got += [g.to(s[k].dtype) for k, g in zip(s["leaves"], grads)]
    return got


def _run_own(s):
    if s["op"] == "adamw":
        s["opt"].step()
        return [s["opt"].arena.flat_p, *s["opt"].moments()]
    from graphgps_amd import ops
    train = s["form"] == "train"
    if s["op"] == "norm":
        outs = ops.sandwich_norm(s["x"], s["a"], post_weight=s["post_weight"], post_bias=s["post_bias"], pre_weight=s["pre_weight"],
                                 pre_bias=s["pre_bias"], gate=s["gate"], residual_scale=0.75, branch_scale=0.5, kind=s["kind"], eps=1e-5)
        couts = [s["dy"], s["dz"]] if train else None
    elif s["packed"]:
        outs = [ops.diff_segment_attention(s["qkv"], s["lam"], s["index"], s["heads"], s["kv_heads"], causal=s["causal"], key_mask=s["keep"])]
        couts = [s["do"]] if train else None
    else:
        outs = [ops.diff_attention(s["q"], s["k"], s["v"], s["lam"], s["q_ptr"], s["k_ptr"], causal=s["causal"], key_mask=s["keep"],
                                   max_q=s["max_q"], max_k=s["max_k"])]
        couts = [s["do"]] if train else None
    got = list(outs)
    if train:
        got += torch.autograd.grad(outs, [s[k] for k in s["leaves"]], couts)
    return got


def run(state):
    return _run_own(state) if own else _run_plain(state)


# -------------------------------------------------------------------------------------------- the definition in 64 bits
def _diff_exact(s):
    """Segment by segment and head by head, with the gradients' formulas written out."""
    if s["packed"]:
        w, h, hk, d = s["qkv"].detach().double(), s["heads"], s["kv_heads"], s["dim"]
        q, k, v = w[:, :2 * h * d].reshape(-1, h, 2, d), w[:, 2 * h * d:2 * (h + hk) * d].reshape(-1, hk, 2, d), w[:, 2 * (h + hk) * d:].reshape(-1, hk, 2 * d)
    else:
        q, k, v = (s[x].detach().double() for x in "qkv")
    lam, train = s["lam"].detach().double(), s["form"] == "train"
    o = torch.zeros(s["nq"], s["heads"], 2 * s["dim"], dtype=torch.float64, device=q.device)
    dq, dk, dv, dl = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v), torch.zeros_like(lam)
    do = s["do"].double() if train else None
    qp, kp, scale, group = s["q_ptr"].tolist(), s["k_ptr"].tolist(), 1.0 / math.sqrt(s["dim"]), s["heads"] // s["kv_heads"]
    for b in range(len(kp) - 1):
        k0, k1 = kp[b], kp[b + 1]
        for h in range(s["heads"]):
            for q0 in range(qp[b], qp[b + 1], 2048):
                q1 = min(q0 + 2048, qp[b + 1])
                see = torch.ones(q1 - q0, k1 - k0, dtype=torch.bool, device=q.device)
                if s["keep"] is not None:
                    see &= s["keep"][k0:k1]
                if s["causal"]:
                    see = see.tril((q0 - qp[b]) + (k1 - k0) - (qp[b + 1] - qp[b]))
                vals, maps = v[k0:k1, h // group], []
                for i in range(2):
                    z = (q[q0:q1, h, i] @ k[k0:k1, h // group, i].T * scale).masked_fill(~see, -math.inf)
                    maps.append(torch.nan_to_num(torch.softmax(z, -1), nan=0.0) if k1 > k0 else z)
                heads = [p @ vals for p in maps]
                o[q0:q1, h] = heads[0] - lam[h] * heads[1]
                if train:
                    c = do[q0:q1, h]
                    dl[h] -= (c * heads[1]).sum()
                    dv[k0:k1, h // group] += (maps[0] - lam[h] * maps[1]).T @ c
                    dp = c @ vals.T
                    for i, f in ((0, 1.0), (1, -lam[h])):
                        ds = f * scale * maps[i] * (dp - (c * heads[i]).sum(-1, keepdim=True))
                        dq[q0:q1, h, i] += ds @ k[k0:k1, h // group, i]
                        dk[k0:k1, h // group, i] += ds.T @ q[q0:q1, h, i]
    if not train:
        return [o]
    if s["packed"]:
        return [o, torch.cat([x.reshape(x.shape[0], -1) for x in (dq, dk, dv)], 1), dl]
    return [o, dq, dk, dv, dl]


def _norm_exact(s):
    d, eps, layer = s["width"], 1e-5, s["kind"] == "layer"
    f = {k: s[k].detach().double() for k in s["leaves"]}

    def forward(t):
        c = t - t.mean(-1, keepdim=True) if layer else t
        r = 1.0 / torch.sqrt((c * c).sum(-1, keepdim=True) / d + eps)
        return c * r, r

    def back(g, hat, r):
        g = g - hat * (g * hat).mean(-1, keepdim=True)
        return r * (g - g.mean(-1, keepdim=True) if layer else g)

    ahat, ra = forward(f["a"])
    n = ahat * f["post_weight"] + (f["post_bias"] if layer else 0.0)
    gate = f.get("gate", torch.ones((), dtype=torch.float64, device=n.device))
    y = 0.75 * f["x"] + 0.5 * gate * n
    yhat, ry = forward(y)
    got = [y, yhat * f["pre_weight"] + (f["pre_bias"] if layer else 0.0)]
    if s["form"] == "train":
        dz = s["dz"].double()
        dy = s["dy"].double() + back(dz * f["pre_weight"], yhat, ry)
        dn = 0.5 * dy * gate
        by = {"x": 0.75 * dy, "a": back(dn * f["post_weight"], ahat, ra), "post_weight": (dn * ahat).sum(0), "post_bias": dn.sum(0),
              "pre_weight": (dz * yhat).sum(0), "pre_bias": dz.sum(0)}
        if "gate" in f:
            by["gate"] = 0.5 * dy * n if f["gate"].dim() == 2 else (0.5 * dy * n).sum(0)
        got += [by[k] for k in s["leaves"]]
    return got


def _adamw_exact(s):
    hy, t = s["hyper"], s["step"] + 1
    b1, b2 = hy["betas"]
    dev, n = s["p"].device, s["p"].numel()

    def values(code, exponent, octaves):
        c = code.double()
        sign = torch.ones_like(c)
        if octaves == 18:
            sign, c = torch.where(c >= 128, -1.0, 1.0), c % 128
        e = torch.clamp(torch.floor(c / 8) - 1, min=0)
        units = torch.where(c < 8, c, (8 + c % 8) * torch.exp2(e))
        return (sign * units * torch.exp2(exponent.double() - 127)[:, None]).view(-1)

    def rounded(x, bits, octaves):
        x = x.view(-1, _BLOCK)
        size, r = x.abs(), bits.view(-1, _BLOCK).double() / 65536
        top = size.amax(-1, keepdim=True)
        unit = torch.exp2(torch.ceil(torch.log2(torch.where(top > 0, top, torch.ones_like(top)) / 15)) - octaves + 4)
        unit = torch.where(unit * 15 * 2.0 ** (octaves - 5) >= top, unit / 2, unit)
        unit = torch.where(unit * 15 * 2.0 ** (octaves - 4) < top, unit * 2, unit).clamp(min=2.0 ** -126)
        y = size / unit
        step = torch.exp2(torch.clamp(torch.floor(torch.log2(torch.clamp(y, min=1.0))) - 3, min=0))
        z = torch.floor(y / step + r) * step
        if octaves == 34:
            z = torch.where((z == 0) & (y > 0), torch.ones_like(z), z)
        return (torch.sign(x) * z * unit).view(-1)

    g = s["g"].double()
    g = g * min(1.0, hy["max_grad_norm"] / (float((g * g).sum()) ** 0.5 + 1e-6))
    m = b1 * values(s["m_code"], s["m_exp"], 18) + (1 - b1) * g
    v = b2 * values(s["v_code"], s["v_exp"], 34) + (1 - b2) * g * g
    p = s["p"].double() * (1 - hy["lr"] * hy["weight_decay"])
    p -= hy["lr"] * (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + hy["eps"])

    def mix(x):
        x = ((x ^ (x >> 16)) * 0x7FEB352D) % (1 << 32)
        x = ((x ^ (x >> 15)) * 0x846CA68B) % (1 << 32)
        return x ^ (x >> 16)

    word = mix((torch.arange(n, device=dev) + int(mix(torch.tensor(t * 0x9E3779B9 % (1 << 32))))) % (1 << 32))
    return [p, rounded(m, word % 65536, 18), rounded(v, word // 65536, 34)]


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"diff": _diff_exact, "norm": _norm_exact, "adamw": _adamw_exact}[case["op"]](s)
