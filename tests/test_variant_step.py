"""The training step of the variant configuration (layer norm, capped and
distance-biased attention, 8-bit Adam moments) against a restatement of the model
in 64 bits.

Tolerances: the step keeps activations and gradients in bf16 where the restatement
rounds nothing but the parameters. A bf16 rounding is off by 2^-9 rms or so; about
ten of them a block in either direction, independent, over four blocks and the
head add up to sqrt(2 * 45) * 2^-9 = 1.9% of a gradient: 4% with room for the
small ones. The loss averages 2,048 tokens: 1e-3, as for the plain step.
"""

import dataclasses

import numpy as np
import pytest
import torch

from rig_b200 import kernels, ops, runlog
from rig_b200.config import load_config, resolve_config, tensor_multipliers, tpp_parameters
from rig_b200.model import GPTTrainer, ParamLayout, block_fields, init_params
from rig_b200.tokens import zipf_tokens


def _config(**kw):
    cfg = load_config("variant_125m", tier="smoke_256", context="smoke_256")
    return dataclasses.replace(cfg, **kw)


def _batch(cfg, seed=0):
    b, t = cfg.batch_size, cfg.seq_len
    w = zipf_tokens(b * (t + 1), cfg.vocab_size, seed).astype(np.int32).reshape(b, t + 1)
    return torch.from_numpy(w[:, :-1].copy()), torch.from_numpy(w[:, 1:].copy())


def _norm(x, scale, bias):
    x = x - x.mean(-1, keepdim=True)
    return x * (x.square().mean(-1, keepdim=True) + 1e-5).rsqrt() * scale + bias


def _restatement(cfg, params, x, y, dev):
    """(loss, gradients) in 64 bits, from bf16-rounded parameters."""

    p = {k: torch.from_numpy(v).to(dev).bfloat16().double().requires_grad_(True) for k, v in params.items()}
    b, t, d, h = cfg.batch_size, cfg.seq_len, cfg.d_model, cfg.heads
    cos, sin = (c.double() for c in ops.rope_tables(t, 64, dev))
    at = torch.arange(t, device=dev)
    distance = (at[:, None] - at[None]).abs()
    seg = None
    if cfg.document_masking:
        seg = ops.document_segments(x.to(dev), cfg.document_boundary_token)

    def rope(z):  # [b, h, t, 64], pairs (2i, 2i + 1)
        even, odd = z[..., 0::2], z[..., 1::2]
        return torch.stack((even * cos - odd * sin, even * sin + odd * cos), -1).flatten(-2)

    act = p["token_embedding"][x.to(dev).long()]
    for l in range(cfg.layers):
        w = {k.split("/")[-1]: v for k, v in p.items() if k.startswith(f"blocks/{l}/")}
        n = _norm(act, w["ln1_scale"], w["ln1_bias"])
        qkv = (n @ w["qkv_w"] + w["qkv_b"]).view(b, t, 3, h, 64).permute(2, 0, 3, 1, 4)
        q, k, v = rope(qkv[0]), rope(qkv[1]), qkv[2]
        s = cfg.softmax_scale * q @ k.transpose(-1, -2)
        s = cfg.attention_softcap * torch.tanh(s / cfg.attention_softcap)
        s = s - kernels.distance_slopes(h, dev).double()[:, None, None] * distance
        see = at[None] <= at[:, None]
        if seg is not None:
            see = see & (seg[:, None, :, None] == seg[:, None, None, :])
        a = torch.softmax(s.masked_fill(~see, -torch.inf), -1) @ v
        a = a.transpose(1, 2).reshape(b, t, d)
        act = act + cfg.branch_scale * (a @ w["attn_w"] + w["attn_b"])
        n = _norm(act, w["ln2_scale"], w["ln2_bias"])
        u = torch.nn.functional.gelu(n @ w["mlp_up_w"] + w["mlp_up_b"], approximate="tanh")
        act = act + cfg.branch_scale * (u @ w["mlp_down_w"] + w["mlp_down_b"])
    act = _norm(act, p["final_ln_scale"], p["final_ln_bias"])
    logits = act @ p["token_embedding"].T
    loss = torch.nn.functional.cross_entropy(logits.view(b * t, -1), y.to(dev).long().view(-1))
    loss.backward()
    return loss.item(), {k: v.grad.cpu().numpy() for k, v in p.items()}


@pytest.mark.gpu
@pytest.mark.parametrize("documents", [False, True])
def test_loss_and_gradients(cuda, documents):
    cfg = _config(document_masking=documents, document_boundary_token=3)
    params = init_params(cfg, 0)
    rng = np.random.default_rng(1)
    for k, v in params.items():  # biases and scales away from 0 and 1, scores that meet the cap
        if k.endswith(("_b", "_bias", "_scale")):
            params[k] = v + 0.1 * rng.standard_normal(v.shape).astype(np.float32)
        if k.endswith("qkv_w"):
            params[k] = v * 8
    x, y = _batch(cfg)
    want, grads = _restatement(cfg, params, x, y, cuda)
    tr = GPTTrainer(cfg, cfg.batch_size, cuda)
    tr.load_params(params)
    tr.set_batch(x.to(cuda), y.to(cuda))
    tr.forward()
    tr.backward()
    torch.cuda.synchronize()
    assert ops.device_error() == 0
    assert abs(tr.loss.item() - want) <= 1e-3 * abs(want)
    got = tr.export(tr.grads)
    for k, g in grads.items():
        off = np.linalg.norm(got[k] - g) / np.linalg.norm(g)
        assert off <= 4e-2, (k, off)


@pytest.mark.gpu
def test_training_with_8_bit_moments(cuda):
    """Same data, moments in 32 and in 8 bits: the loss falls alike (a code is within
    2^-4 and the roundings of 11 M parameters are independent and unbiased)."""

    curves = []
    for bits in (32, 8):
        cfg = _config(optimizer_state_bits=bits, steps=30, warmup_steps=3)
        tr = GPTTrainer(cfg, cfg.batch_size, cuda)
        tr.load_params(init_params(cfg, 0))
        for i in range(cfg.steps):
            x, y = _batch(cfg, i % 4)
            tr.train_step(x.to(cuda), y.to(cuda))
        curves.append([tr.checked_metrics(i + 1)["train_loss"] for i in range(cfg.steps)])
    a, b = (np.array(c) for c in curves)
    assert a[0] == b[0] and a[0] - a[-1] > 1.0
    assert np.abs(a - b).max() <= 0.1 * (a[0] - a[-1])


@pytest.mark.gpu
def test_graph_overlap_and_repeat(cuda):
    """A captured step, and the update in buckets on its own stream, follow plain
    eager steps (not bit for bit: dQ's parts add up in any order)."""

    cfg = _config(steps=6, warmup_steps=1)
    finals = []
    for how in ("eager", "overlap", "graph"):
        tr = GPTTrainer(cfg, cfg.batch_size, cuda, overlap_optimizer=how == "overlap")
        tr.load_params(init_params(cfg, 0))
        for i in range(4):
            x, y = _batch(cfg, i)
            tr.train_step(x.to(cuda), y.to(cuda))
            if how == "graph" and i == 0:
                tr.capture()
        torch.cuda.synchronize()
        assert ops.device_error() == 0 and int(tr.step_dev) == 4
        finals.append([tr.history[i].cpu().numpy() for i in range(4)])
    for other in finals[1:]:
        for a, b in zip(finals[0], other):
            np.testing.assert_allclose(a, b, rtol=5e-3)


def test_configuration_and_layout():
    cfg = load_config("variant_125m")
    assert (cfg.normalization, cfg.attention_softcap, cfg.attention_bias, cfg.optimizer_state_bits) == \
        ("layer_norm", 30.0, "distance", 8)
    plain = load_config("baseline_125m")
    assert not plain.score_attention and plain.optimizer_state_bits == 32
    extra = {s.name for s in ParamLayout(cfg).slots} - {s.name for s in ParamLayout(plain).slots}
    assert extra == {f"blocks/{b}/ln{i}_bias" for b in range(12) for i in (1, 2)} | {"final_ln_bias"}
    assert block_fields(cfg)[:3] == ("ln1_scale", "ln1_bias", "qkv_w")
    params = init_params(cfg.replace(layers=1, vocab_size=64, semantic_vocab_size=64), 0)
    assert not params["blocks/0/ln1_bias"].any() and not params["final_ln_bias"].any()
    assert tensor_multipliers("final_ln_bias", False, cfg) == (1.0, 1.0, 1.0)
    model = dict(d_model=8, layers=2, vocab_size=10)
    assert tpp_parameters({**model, "normalization": "layer_norm"}) == tpp_parameters(model) + 5 * 8
    meta = runlog.checkpoint_metadata(cfg, 0)["model"]
    assert meta["normalization"] == "layer_norm" and meta["attention_softcap"] == 30.0
    assert "attention_softcap" not in runlog.checkpoint_metadata(plain, 0)["model"]


@pytest.mark.parametrize("where,key,value", [("model", "normalization", "batch_norm"),
                                             ("model", "attention_softcap", -1.0),
                                             ("model", "attention_bias", "learned"),
                                             ("optimizer", "state_bits", 4)])
def test_configuration_refusals(where, key, value):
    import yaml

    from rig_b200.config import CONFIG_DIR

    doc = yaml.safe_load((CONFIG_DIR / "variant_125m.yaml").read_text())
    target = doc["run"]["optimizer"] if where == "optimizer" else \
        doc["family"]["tiers"]["125m_768_tied"]["model"]
    target[key] = value
    with pytest.raises(ValueError):
        resolve_config(doc)
