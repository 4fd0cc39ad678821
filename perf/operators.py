"""Cases, plain forms and exact values of the score-modified attention, layer norm and
8-bit AdamW operators.

These are the operators of one training step of a GPT variant: causal attention whose
scores are capped by a tanh and biased by distance (optionally under a document, padding
or prefix mask, with key/value heads shared by several query heads), layer norm instead of
RMS norm, and an AdamW update that keeps both moments in 8 bits.

`run` computes a case in its plain form (elementary torch operations in 32 bits) where
`own` is false and calls the framework's kernels where it is true; `exact` gives the same
values in 64 bits, from the definitions.
"""

import math
import os
import struct
import sys

import numpy as np
import torch

own = False

F32, BF16, I32 = torch.float32, torch.bfloat16, torch.int32
HEAD_DIM = 64
LN_EPS = 1e-5
BLOCK = 64        # elements that share one exponent of an 8-bit state
HISTORY = 4096    # rows of the optimizer's (loss, learning rate, gradient norm) log
ADAM = dict(learning_rate=1e-3, min_lr_ratio=0.1, warmup_steps=256, total_steps=HISTORY,
            beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.1, grad_scale=1.0)


# ------------------------------------------------------------------ cases
def listed():
    def attention(name, batch, heads, kv_heads, seq, mask, softcap, bias, train):
        return dict(name=name, op="attention", batch=batch, heads=heads, kv_heads=kv_heads, seq=seq,
                    mask=mask, softcap=softcap, bias=bias, train=train)

    def norm(name, rows, width, dtype, residual, train):
        return dict(name=name, op="layer_norm", rows=rows, width=width, dtype=dtype,
                    residual=residual, train=train)

    def adam(name, layers, width, vocab, clip):
        return dict(name=name, op="adamw8", layers=layers, width=width, vocab=vocab, clip=clip)

    return [
        # one short sequence on the smoke model's heads: launch latency
        attention("attention_short", 1, 4, 4, 33, "causal", 30.0, True, True),
        # the 125M model's heads on packed 1k documents, one micro-batch
        attention("attention_1k_documents", 8, 12, 12, 1024, "documents", 30.0, False, True),
        # the same heads with three query heads to a key/value head, a bidirectional prefix
        # and a length that ends inside a tile
        attention("attention_shared_prefix", 4, 12, 4, 1500, "prefix", 0.0, True, True),
        # the 8k context, capped and biased
        attention("attention_8k", 1, 12, 12, 8192, "causal", 50.0, True, True),
        # evaluation (forward only) of right-padded rows of an odd length
        attention("attention_eval_padded", 16, 12, 12, 777, "padded", 20.0, True, False),
        # a few rows of the smoke model's width: launch latency
        norm("norm_short", 33, 256, "bfloat16", False, True),
        # the 125M model's norm over its global batch, with the residual stream's gradient
        norm("norm_125m", 131072, 768, "bfloat16", True, True),
        # 32-bit activations of an odd width
        norm("norm_odd_fp32", 4097, 771, "float32", True, True),
        # evaluation of a wide model
        norm("norm_eval_wide", 8192, 4096, "bfloat16", False, False),
        # a tiny model's tensors: launch latency
        adam("adamw8_tiny", 2, 64, 512, 0.0),
        # every tensor of the 125M model, unclipped as its configuration says
        adam("adamw8_125m", 12, 768, 50304, 0.0),
        # the 60M base tier, clipped at a global gradient norm of 1
        adam("adamw8_60m_clipped", 12, 384, 50304, 1.0),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "layer_norm", "adamw8"])
    if op == "attention":
        kv = rng.choice([1, 2, 3, 4, 6])
        heads = kv * rng.choice([1, 1, 2, 4])
        seq = _log(rng, 1, 6000)
        if seq == 3072:
            seq += 1
        batch = max(1, min(_log(rng, 1, 16), int(4e8 / (heads * seq * seq + 1))))
        return dict(op=op, batch=batch, heads=heads, kv_heads=kv, seq=seq,
                    mask=rng.choice(["causal", "documents", "prefix", "padded"]),
                    softcap=rng.choice([0.0, 15.0, 30.0, 50.0]), bias=rng.random() < 0.6,
                    # a query that sees one key has a score gradient of zero, which every order
                    # of summing leaves as its own rounding noise: training has more keys
                    train=seq >= 16 and rng.random() < 0.75)
    if op == "layer_norm":
        width = _log(rng, 40, 6000)
        if rng.random() < 0.75:
            width = (width + 7) // 8 * 8
        if width == 3072:
            width += 8
        rows = _log(rng, 1, max(2, int(6e7 / width)))
        return dict(op=op, rows=rows, width=width, dtype=rng.choice(["bfloat16", "bfloat16", "float32"]),
                    residual=rng.random() < 0.5, train=rng.random() < 0.75)
    width = 64 * rng.choice([1, 2, 3, 5, 6, 8, 10])
    return dict(op=op, layers=rng.randint(1, 12), width=width, vocab=_log(rng, 200, 51000),
                clip=rng.choice([0.0, 1.0]))


# ------------------------------------------------------------------ shared by prepare and the forms
def _slopes(heads, device):
    """Geometric distance slopes, 2^(-8 (h + 1) / heads)."""
    return torch.pow(2.0, -8.0 * (torch.arange(heads, device=device, dtype=F32) + 1) / heads)


def _adam_tensors(case):
    """[(size, lr, eps, decay multipliers, decays)] of a small GPT's tensors."""
    d, v = case["width"], case["vocab"]
    mats = [(d * 3 * d), (d * d), (d * 4 * d), (4 * d * d)]
    vecs = [d, d, 3 * d, d, d, d, 4 * d, d]
    out = []
    for _ in range(case["layers"]):
        out += [(n, 0.5, 0.5, 2.0, 1) for n in mats] + [(n, 1.0, 0.5, 1.0, 0) for n in vecs]
    return out + [(d, 1.0, 1.0, 1.0, 0), (d, 1.0, 1.0, 1.0, 0), (v * d, 1.0, 0.5, 1.0, 1)]


def _padded(n):
    return (n + BLOCK - 1) // BLOCK * BLOCK


def _encode(x, dither, mantissa, flush):
    """Codes and block exponents of |x|: 4 exponent bits and `mantissa` bits under the
    block's largest exponent, the bits below rounded by adding `dither` (an integer below one
    unit of the last kept bit) and cutting. `flush`: what is too small becomes 0 (else the
    smallest code)."""
    shift = 23 - mantissa
    bits = x.abs().view(I32).view(-1, BLOCK)
    top = (bits.amax(1, keepdim=True) + ((1 << shift) - 1)) >> 23
    exponent = torch.where(top >= 255, 255, top.clamp(min=16))
    code = (bits + dither.view(-1, BLOCK) - ((exponent - 15) << 23)) >> shift
    low = torch.zeros_like(code) if flush else (bits > 0).to(I32)
    code = torch.maximum(code, low).clamp(max=(16 << mantissa) - 1)
    return code.view(-1), exponent.view(-1).to(torch.uint8)


def _decode(code, exponent, mantissa):
    e = exponent.to(I32).view(-1, 1)
    bits = (code.view(-1, BLOCK) << (23 - mantissa)) + ((e - 15) << 23)
    x = torch.where(code.view(-1, BLOCK) == 0, 0.0, bits.view(F32))
    return torch.where(e == 255, math.nan, x).view(-1)


def _decode_m(state):
    c = state["m"].to(I32)
    x = _decode(c & 127, state["m_exp"], 3)
    return torch.where(c >= 128, -x, x)


def _decode_r(state):
    return _decode(state["v"].to(I32), state["v_exp"], 4)


def _mix32(h):
    """The finalizer of MurmurHash3 (32 bits), on int64 tensors or ints."""
    mask = 0xFFFFFFFF
    h = ((h ^ (h >> 16)) * 0x85EBCA6B) & mask
    h = ((h ^ (h >> 13)) * 0xC2B2AE35) & mask
    return h ^ (h >> 16)


def _dither(n, seed, step):
    """32 random bits of every element at 1-based step `step` (an int64 tensor of one value)."""
    i = torch.arange(n, device=step.device)
    key = _mix32(_mix32(step & 0xFFFFFFFF) ^ (seed & 0xFFFFFFFF))
    return _mix32(((i & 0xFFFFFFFF) * 0x9E3779B1 + (i >> 32) * 0x85EBCA77 + key) & 0xFFFFFFFF)


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, dtype=F32, scale=1.0):
        return (torch.randn(*shape, generator=g, device=dev) * scale).to(dtype)

    if case["op"] == "attention":
        b, h, kv, t = case["batch"], case["heads"], case["kv_heads"], case["seq"]
        # one packed projection output [B, T, H + 2 KV, 64], as the model's QKV product writes
        packed = normal(b, t, h + 2 * kv, HEAD_DIM, dtype=BF16)
        packed[:, :, :h] *= 3.0  # trained models' scores spread wider than a unit normal
        s = dict(case=case, q=packed[:, :, :h], k=packed[:, :, h:h + kv], v=packed[:, :, h + kv:],
                 do=normal(b, t, h, HEAD_DIM, dtype=BF16), scale=HEAD_DIM ** -0.5,
                 slopes=_slopes(h, dev) if case["bias"] else None, segments=None, prefix=None)
        if case["mask"] == "documents":
            cut = torch.rand(b, t, generator=g, device=dev) < 1.0 / _mean_document(case)
            s["segments"] = torch.cumsum(cut, 1).to(I32)
        elif case["mask"] == "padded":  # the rows' ends carry no token (segment -1)
            keep = torch.randint((t + 1) // 2, t + 1, (b, 1), generator=g, device=dev)
            at = torch.arange(t, device=dev)[None]
            s["segments"] = torch.where(at < keep, 0, -1).to(I32)
        elif case["mask"] == "prefix":
            s["prefix"] = torch.randint(0, t // 2 + 1, (b,), generator=g, device=dev, dtype=I32)
        return s
    if case["op"] == "layer_norm":
        n, d = case["rows"], case["width"]
        dt = getattr(torch, case["dtype"])
        return dict(case=case, x=normal(n, d, dtype=dt, scale=1.5) + normal(n, 1, dtype=dt, scale=0.5),
                    scale=(1 + normal(d, scale=0.1)).to(dt), bias=normal(d, dtype=dt, scale=0.1),
                    dy=normal(n, d, dtype=dt), dres=normal(n, d, dtype=dt) if case["residual"] else None,
                    alpha=0.5)
    tensors = _adam_tensors(case)
    n = sum(_padded(t[0]) for t in tensors)
    offsets, at = [], 0
    for t in tensors:
        offsets.append(at)
        at += _padded(t[0])
    live = torch.zeros(n, device=dev, dtype=torch.bool)
    for o, t in zip(offsets, tensors):
        live[o:o + t[0]] = True
    grads = torch.where(live, normal(n) * torch.exp(normal(n)) * 1e-3, 0.0)
    params = torch.where(live, normal(n, scale=0.05), 0.0)
    m = torch.where(live, normal(n, scale=3e-4) * torch.exp(normal(n)), 0.0)
    r = torch.where(live, torch.exp(normal(n)) * 1e-3, 0.0)
    m_code, m_exp = _encode(m, torch.full_like(m, 1 << 19, dtype=I32), 3, True)
    v_code, v_exp = _encode(r, torch.full_like(r, 1 << 18, dtype=I32), 4, False)
    m_code += 128 * (m < 0).to(I32)
    table = b"".join(struct.pack("<qqfffi", o, *t) for o, t in zip(offsets, tensors))
    groups = torch.frombuffer(bytearray(table), dtype=torch.uint8).to(dev)
    sizes = torch.tensor([_padded(t[0]) for t in tensors], device=dev)
    mult = torch.tensor([t[1:4] for t in tensors], device=dev, dtype=F32)
    decays = torch.tensor([t[4] for t in tensors], device=dev, dtype=F32)
    return dict(case=case, n=n, params=params, grads=grads, m=m_code.to(torch.uint8), m_exp=m_exp,
                v=v_code.to(torch.uint8), v_exp=v_exp, mirror=params.to(BF16), groups=groups,
                n_groups=len(tensors), sizes=sizes, mult=mult, decays=decays, seed=seed & 0x7FFFFFFF,
                step=torch.full((1,), 20, device=dev, dtype=I32),
                loss=torch.full((1,), 3.5, device=dev), history=torch.zeros(HISTORY, 3, device=dev))


def _mean_document(case):
    return max(2.0, min(300.0, case["seq"] / 3))


# ------------------------------------------------------------------ one pass
def run(state):
    op = state["case"]["op"]
    if own:
        return {"attention": _own_attention, "layer_norm": _own_norm, "adamw8": _own_adam}[op](state)
    return {"attention": _plain_attention, "layer_norm": _plain_norm, "adamw8": _plain_adam}[op](state)


def _visible(s, t, device):
    """[B or 1, 1, T, T]: whether query i sees key j."""
    i = torch.arange(t, device=device)
    see = (i[None, :] <= i[:, None])[None]
    if s["prefix"] is not None:
        see = see | (i[None, None, :] < s["prefix"][:, None, None])
    if s["segments"] is not None:
        g = s["segments"]
        see = see & (g[:, :, None] == g[:, None, :]) & (g[:, :, None] >= 0)
    return see[:, None]


def _plain_attention(s):
    c = s["case"]
    b, t, h, _ = s["q"].shape
    kv = c["kv_heads"]
    cap, scale = c["softcap"], s["scale"]
    # shared key/value heads: one more axis of query heads, [B, KV, G, T, 64] against [B, KV, 1, T, 64]
    q = s["q"].float().transpose(1, 2).reshape(b, kv, h // kv, t, HEAD_DIM)
    k = s["k"].float().transpose(1, 2).unsqueeze(2)
    v = s["v"].float().transpose(1, 2).unsqueeze(2)
    x = (q @ k.transpose(-1, -2)) * scale
    if cap:
        th = torch.tanh(x / cap)
        x = cap * th
    if s["slopes"] is not None:
        i = torch.arange(t, device=x.device)
        x = x - s["slopes"].view(1, kv, h // kv, 1, 1) * (i[:, None] - i[None, :]).abs()
    see = _visible(s, t, x.device).unsqueeze(2)
    x = torch.where(see, x, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    o = p @ v

    def back(y):  # [B, KV, G, T, 64] -> [B, T, H, 64]
        return y.reshape(b, -1, t, HEAD_DIM).transpose(1, 2).to(BF16)

    if not c["train"]:
        return dict(o=back(o))
    do = s["do"].float().transpose(1, 2).reshape(b, kv, h // kv, t, HEAD_DIM)
    dv = (p.transpose(-1, -2) @ do).sum(2)
    ds = p * (do @ v.transpose(-1, -2) - (do * o).sum(-1, keepdim=True))
    if cap:
        ds = ds * (1 - th * th)
    ds = ds * scale
    return dict(o=back(o), dq=back(ds @ k), dk=back((ds.transpose(-1, -2) @ q).sum(2)), dv=back(dv))


def _plain_norm(s):
    c = s["case"]
    dt = s["x"].dtype
    x, w, bias = s["x"].float(), s["scale"].float(), s["bias"].float()
    d = x.shape[1]
    mean = x.sum(1, keepdim=True) / d
    xc = x - mean
    rstd = 1 / torch.sqrt((xc * xc).sum(1, keepdim=True) / d + LN_EPS)
    hat = xc * rstd
    y = (hat * w + bias).to(dt)
    if not c["train"]:
        return dict(y=y)
    dy = s["dy"].float()
    dn = dy * w
    dx = rstd * (dn - dn.sum(1, keepdim=True) / d - hat * ((dn * hat).sum(1, keepdim=True) / d))
    out = dict(y=y, dscale=(dy * hat).sum(0), dbias=dy.sum(0))
    if s["dres"] is not None:  # the residual stream's gradient, and its column sums below the norm
        dx = dx + s["dres"].float()
        out["dcolumns"] = s["alpha"] * dx.sum(0)
    out["dx"] = dx.to(dt)
    return out


def _plain_adam(s):
    a, c, n = ADAM, s["case"], s["n"]
    s["step"] += 1
    t = s["step"].float()
    warm = torch.clamp(t / a["warmup_steps"], max=1.0)
    at = torch.clamp((t - a["warmup_steps"]) / (a["total_steps"] - a["warmup_steps"]), 0.0, 1.0)
    low = a["min_lr_ratio"]
    lr = a["learning_rate"] * warm * (low + (1 - low) * (0.5 * (1 + torch.cos(math.pi * at))))
    norm = torch.sqrt((s["grads"] * s["grads"]).sum()) * a["grad_scale"]
    gscale = torch.full_like(norm, a["grad_scale"])
    if c["clip"]:
        gscale = gscale * torch.clamp(c["clip"] / (norm + 1e-6), max=1.0)
    row = torch.stack([s["loss"][0], lr[0], norm]).view(1, 3)
    s["history"].index_copy_(0, (s["step"].long() - 1).clamp(max=HISTORY - 1), row)
    each = torch.repeat_interleave(s["mult"], s["sizes"], 0, output_size=n)
    decays = torch.repeat_interleave(s["decays"], s["sizes"], 0, output_size=n)
    g = s["grads"] * gscale
    b1, b2 = np.float32(a["beta1"]), np.float32(a["beta2"])
    m = float(b1) * _decode_m(s) + float(np.float32(1) - b1) * g
    r = _decode_r(s)
    r = torch.sqrt(float(b2) * (r * r) + float(np.float32(1) - b2) * (g * g))
    inv1 = 1 / (1 - torch.pow(float(b1), t))
    inv2 = 1 / torch.sqrt(1 - torch.pow(float(b2), t))
    p = s["params"]
    update = (m * inv1) / (r * inv2 + a["eps"] * each[:, 1])
    p = p - (lr * each[:, 0]) * (update + (decays * a["weight_decay"] * each[:, 2]) * p)
    bits = _dither(n, s["seed"], s["step"].long())
    code, exponent = _encode(m, ((bits >> 16) << 4).to(I32), 3, True)
    s["m"].copy_(code + 128 * ((m < 0) & (code > 0)))
    s["m_exp"].copy_(exponent)
    code, exponent = _encode(r, ((bits & 0xFFFF) << 3).to(I32), 4, False)
    s["v"].copy_(code)
    s["v_exp"].copy_(exponent)
    s["params"].copy_(p)
    s["mirror"].copy_(p)
    return dict(params=s["params"], mirror=s["mirror"], m=_decode_m(s).to(BF16),
                v_root=_decode_r(s).to(BF16), step=s["step"], history=s["history"])


def _ops():
    package = os.path.abspath("gpt-speedrun-tpu_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    from rig_b200 import ops

    return ops


def _own_attention(s):
    ops, c = _ops(), s["case"]
    q, k, v = s["q"], s["k"], s["v"]
    b, t, h, _ = q.shape
    how = dict(scale=s["scale"], layout="bthd", softcap=c["softcap"], slopes=s["slopes"],
               segment_ids=s["segments"], prefix_lens=s["prefix"])
    o = torch.empty(b, t, h, HEAD_DIM, device=q.device, dtype=BF16)
    lse = torch.empty(b, h, t, device=q.device)
    ops.score_attention_fwd(q, k, v, o, lse, **how)
    if not c["train"]:
        return dict(o=o)
    grads = torch.empty(b, t, h + 2 * k.shape[2], HEAD_DIM, device=q.device, dtype=BF16)
    dq, dk, dv = grads.split([h, k.shape[2], k.shape[2]], 2)
    ops.score_attention_bwd(q, k, v, o, s["do"], lse, dq, dk, dv, **how)
    return dict(o=o, dq=dq, dk=dk, dv=dv)


def _own_norm(s):
    ops, c, x = _ops(), s["case"], s["x"]
    n, d = x.shape
    y = torch.empty_like(x)
    mean, rstd = torch.empty(2, n, device=x.device).unbind()
    ops.layer_norm_fwd(x, s["scale"], s["bias"], y, mean, rstd, eps=LN_EPS)
    if not c["train"]:
        return dict(y=y)
    dscale, dbias, dcolumns = torch.zeros(3, d, device=x.device).unbind()
    dx = torch.empty_like(x)
    below = {} if s["dres"] is None else dict(dx_colsum=dcolumns, colsum_alpha=s["alpha"])
    ops.layer_norm_bwd(x, s["scale"], mean, rstd, s["dy"], s["dres"], dx, dscale, dbias, **below)
    out = dict(y=y, dx=dx, dscale=dscale, dbias=dbias)
    if s["dres"] is not None:
        out["dcolumns"] = dcolumns
    return out


def _own_adam(s):
    ops = _ops()
    if "plan" not in s:  # what a trainer makes once
        from rig_b200 import _lib

        cfg = _lib.AdamWConfig(horizon_lr_scale=1.0, eps_horizon_scale=1.0, wd_horizon_scale=1.0,
                               grad_clip=s["case"]["clip"], **ADAM)
        s["plan"] = (cfg, ops.adamw_workspace(s["n"], s["params"].device))
    cfg, workspace = s["plan"]
    state = (s["m"], s["m_exp"], s["v"], s["v_exp"])
    ops.adamw8_step(s["params"], state, s["grads"], s["groups"], s["n_groups"], cfg, s["step"],
                    s["loss"], s["history"], s["mirror"], s["seed"], workspace)
    m, v_root = ops.adamw8_values(state)
    return dict(params=s["params"], mirror=s["mirror"], m=m, v_root=v_root, step=s["step"],
                history=s["history"])


# ------------------------------------------------------------------ the least work
def _pairs(case):
    """Expected visible (query, key) pairs of one batch row and head."""
    t = case["seq"]
    if case["mask"] == "documents":
        stay = 1 - 1 / _mean_document(case)
        return sum((1 - stay ** (i + 1)) / (1 - stay) for i in range(t))
    if case["mask"] == "padded":
        return 7 / 24 * t * t + 0.375 * t
    return t * (t + 1) / 2 + (t * t / 24 if case["mask"] == "prefix" else 0)


def work(case):
    if case["op"] == "attention":
        b, h, kv, t = case["batch"], case["heads"], case["kv_heads"], case["seq"]
        rows = b * t * HEAD_DIM * 2  # bytes of one head's rows
        pairs = b * h * _pairs(case)
        if case["train"]:  # q, k, v, do in; o, dq, dk, dv out; 2 + 5 products
            return {"bytes": rows * (4 * h + 4 * kv), "flops": pairs * 7 * 2 * HEAD_DIM}
        return {"bytes": rows * (2 * h + 2 * kv), "flops": pairs * 2 * 2 * HEAD_DIM}
    if case["op"] == "layer_norm":
        size = case["rows"] * case["width"] * (2 if case["dtype"] == "bfloat16" else 4)
        # y; with training dy in and dx out, and the residual stream's gradient in
        moves = 2 + (2 + case["residual"] if case["train"] else 0)
        return {"bytes": size * moves, "flops": 8.0 * case["rows"] * case["width"] * (3 if case["train"] else 1)}
    n = sum(_padded(t[0]) for t in _adam_tensors(case))
    # parameters, both codes and exponents in and out, gradients in, the bf16 copy and the
    # states' values out
    return {"bytes": n * (8 + 4 + 4 + 4 / BLOCK + 2 + 4), "flops": 30.0 * n}


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"attention": _exact_attention, "layer_norm": _exact_norm, "adamw8": _exact_adam}[case["op"]](s)


def _exact_attention(s):
    """Softmax attention of one (batch, head) after the other, gradients by autograd."""
    c = s["case"]
    b, t, h, _ = s["q"].shape
    group = h // c["kv_heads"]
    q, k, v = (s[n].double() for n in "qkv")
    o = torch.zeros(b, t, h, HEAD_DIM, device=q.device, dtype=torch.float64)
    dq, dk, dv = (torch.zeros_like(x) for x in (q, k, v))
    at = torch.arange(t, device=q.device, dtype=torch.float64)
    for i in range(b):
        hidden = at[None, :] > at[:, None]
        if s["prefix"] is not None:
            hidden = hidden & (at[None, :] >= s["prefix"][i])
        if s["segments"] is not None:
            g = s["segments"][i]
            hidden = hidden | (g[:, None] != g[None, :]) | (g < 0)[:, None]
        empty = hidden.all(1, keepdim=True)
        for j in range(h):
            one = [x.clone().requires_grad_(True) for x in (q[i, :, j], k[i, :, j // group], v[i, :, j // group])]
            x = s["scale"] * one[0] @ one[1].T
            if c["softcap"]:
                x = c["softcap"] * torch.tanh(x / c["softcap"])
            if s["slopes"] is not None:
                x = x - s["slopes"][j].double() * (at[:, None] - at[None, :]).abs()
            p = torch.softmax(x.masked_fill(hidden & ~empty, -math.inf), 1).masked_fill(empty, 0.0)
            y = p @ one[2]
            o[i, :, j] = y.detach()
            if c["train"]:
                grads = torch.autograd.grad(y, one, s["do"][i, :, j].double())
                dq[i, :, j] = grads[0]
                dk[i, :, j // group] += grads[1]
                dv[i, :, j // group] += grads[2]
    return dict(o=o, dq=dq, dk=dk, dv=dv) if c["train"] else dict(o=o)


def _exact_norm(s):
    x, w, bias, dy = (s[n].double() for n in ("x", "scale", "bias", "dy"))
    var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
    hat = (x - mean) * torch.rsqrt(var + LN_EPS)
    out = dict(y=torch.addcmul(bias, hat, w))
    if s["case"]["train"]:
        dn = dy * w
        dx = (dn - dn.mean(1, keepdim=True) - hat * (dn * hat).mean(1, keepdim=True)) * torch.rsqrt(var + LN_EPS)
        if s["dres"] is not None:
            dx = dx + s["dres"].double()
            out["dcolumns"] = s["alpha"] * dx.sum(0)
        out.update(dx=dx, dscale=torch.einsum("nd,nd->d", dy, hat), dbias=dy.sum(0))
    return out


def _exact_round(x, u, mantissa, flush):
    """x to `mantissa` bits below its leading one by floor(x / unit + u), within 16 powers of
    two of its block's largest."""
    x = x.view(-1, BLOCK)
    sign, x = torch.sign(x), x.abs()
    _, e = torch.frexp(x)
    part, top = torch.frexp(x.amax(1, keepdim=True))
    top = top + (2 * part > 2 - 2.0 ** -mantissa).to(top.dtype)
    unit = torch.ldexp(torch.ones_like(x), e - 1 - mantissa)
    y = torch.floor(x / unit + u.view(-1, BLOCK)) * unit
    least = torch.ldexp(torch.full_like(x, 1 + 2.0 ** -mantissa), top - 16)
    y = torch.where(y < least, 0.0 if flush else least, y)
    return (sign * torch.where(x == 0, 0.0, y)).view(-1)


def _exact_adam(s):
    a, c, n = ADAM, s["case"], s["n"]
    step = int(s["step"]) + 1
    low = a["min_lr_ratio"]
    along = min(max((step - a["warmup_steps"]) / (a["total_steps"] - a["warmup_steps"]), 0.0), 1.0)
    lr = a["learning_rate"] * min(1.0, step / a["warmup_steps"])
    lr *= low + (1 - low) * 0.5 * (1 + math.cos(math.pi * along))
    g = s["grads"].double()
    norm = float(torch.linalg.vector_norm(g))
    if c["clip"]:
        g = g * min(1.0, c["clip"] / (norm + 1e-6))

    def spread(values):
        return values.double().repeat_interleave(s["sizes"])

    b1, b2 = float(np.float32(a["beta1"])), float(np.float32(a["beta2"]))
    m = b1 * _decode_m(s).double() + (1 - b1) * g
    r = torch.sqrt(b2 * _decode_r(s).double() ** 2 + (1 - b2) * g ** 2)
    update = m / (1 - b1 ** step) / (r / math.sqrt(1 - b2 ** step) + a["eps"] * spread(s["mult"][:, 1]))
    p = s["params"].double()
    decay = a["weight_decay"] * spread(s["decays"] * s["mult"][:, 2])
    p = p - lr * spread(s["mult"][:, 0]) * (update + decay * p)
    bits = _dither(n, s["seed"], torch.full((1,), step, device=p.device, dtype=torch.int64))
    history = s["history"].double()
    history[step - 1] = torch.tensor([float(s["loss"]), lr, norm], dtype=torch.float64)
    return dict(params=p, mirror=p, m=_exact_round(m, (bits >> 16).double() / 65536, 3, True),
                v_root=_exact_round(r, (bits & 0xFFFF).double() / 65536, 4, False), step=step,
                history=history)
