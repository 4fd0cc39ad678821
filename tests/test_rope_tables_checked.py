"""RoPE tables are read up to the last position: what does not cover it, or has
another type or layout, is refused before anything runs."""

import pytest
import torch

from rig_b200 import kernels, ops

T = 40


def _bad(dev):
    cos, sin = ops.rope_tables(T, 64, dev)
    return {
        "short cos": (cos[: T - 1], sin),
        "short sin": (cos, sin[:1]),
        "other head dimension": ops.rope_tables(T, 128, dev),
        "fp32": (cos.float(), sin.float()),
        "strided": (cos.t().contiguous().t(), sin),
        "host": (cos.cpu(), sin.cpu()),
        "one row of numbers": (cos[0], sin[0]),
    }


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["short cos", "short sin", "other head dimension", "fp32", "strided",
                                  "host", "one row of numbers"])
def test_refused(cuda, name):
    rope = _bad(cuda)[name]
    q, k, v, o, do, dq, dk, dv = (torch.zeros(1, 2, T, 64, device=cuda, dtype=torch.bfloat16)
                                  for _ in range(8))
    lse = torch.zeros(1, 2, T, device=cuda)
    before = ops.launch_count()
    with pytest.raises(ValueError, match="rope"):
        ops.rope_apply(q.transpose(1, 2), rope)
    for bwd in (ops.score_attention_bwd, ops.attention_bwd):
        with pytest.raises(ValueError, match="rope"):
            bwd(q, k, v, o, do, lse, dq, dk, dv, scale=0.125, rope=rope)
    for make in (kernels.make_score_attention, kernels.make_causal_attention):
        with pytest.raises(ValueError, match="rope"):
            make(rope_tables=rope)(q, k, v)
    assert ops.launch_count() == before


@pytest.mark.gpu
def test_longer_tables_are_taken(cuda):
    q, k, v = (torch.randn(1, 2, T, 64, device=cuda).bfloat16() for _ in range(3))
    want = kernels.make_score_attention(rope_tables=ops.rope_tables(T, 64, cuda))(q, k, v)
    got = kernels.make_score_attention(rope_tables=ops.rope_tables(T + 9, 64, cuda))(q, k, v)
    assert torch.equal(got, want)
