"""Causal attention with capped and biased scores, behind a factory like `make_causal_attention`.

The returned callable is differentiable in q, k and v through the libgptb200
forward/backward kernels:

    s'_ij = softcap * tanh(scale q_i.k_j / softcap) - slopes[h] |i - j|

with optional key/value heads shared by several query heads, segment ids
(negative: padding) and a per-sequence prefix that every query sees. A query
that sees no key gives zeros. What the masks hide must still be finite numbers
(0 * NaN is NaN in the products). The reference has no counterpart.
"""

from __future__ import annotations

import dataclasses
import math
from typing import Callable

import torch

from .. import ops


@dataclasses.dataclass(frozen=True)
class ScoreAttentionConfig:
    softmax_scale: float | None = None  # None: head_dim ** -0.5
    softcap: float = 0.0                # 0: no cap

    def __post_init__(self) -> None:
        if self.softmax_scale is not None and not 0.0 < self.softmax_scale < math.inf:
            raise ValueError("softmax_scale must be positive")
        if not 0.0 <= self.softcap < math.inf:
            raise ValueError("softcap must be zero (no cap) or positive")


def distance_slopes(heads: int, device) -> torch.Tensor:
    """Geometric distance slopes 2^(-8 (h + 1) / heads), fp32 [heads]."""

    h = torch.arange(1, heads + 1, dtype=torch.float32, device=device)
    return torch.pow(2.0, -8.0 * h / heads)


def _validate(q, k, v) -> None:
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError("q, k, and v must use BHSD rank-4 layout; "
                         f"got {tuple(q.shape)}, {tuple(k.shape)}, and {tuple(v.shape)}")
    if k.shape != v.shape or q.shape[0] != k.shape[0] or q.shape[2:] != k.shape[2:]:
        raise ValueError("q, k and v must agree but for the number of heads; "
                         f"got {tuple(q.shape)}, {tuple(k.shape)}, and {tuple(v.shape)}")
    if not all(q.shape) or not all(k.shape):
        raise ValueError(f"q/k/v dimensions must be nonzero, got {tuple(q.shape)}, {tuple(k.shape)}")
    if q.shape[1] % k.shape[1]:
        raise ValueError(f"{q.shape[1]} query heads cannot share {k.shape[1]} key/value heads")
    if q.shape[-1] != 64:
        raise ValueError(f"the B200 kernel requires head_dim 64, got {q.shape[-1]}")
    if any(t.dtype != torch.bfloat16 for t in (q, k, v)):
        raise TypeError(f"q, k, and v must be bfloat16, got {q.dtype}, {k.dtype}, {v.dtype}")


_MASKS = ("slopes", "segment_ids", "prefix_lens")


class _ScoreAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, scale, softcap, rope, *masks):
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
        if rope is not None:  # rotate copies of q and k (BHSD viewed as BTHD)
            q, k = q.clone(), k.clone()
            ops.rope_apply(q.transpose(1, 2), rope)
            ops.rope_apply(k.transpose(1, 2), rope)
        b, h, t, _ = q.shape
        o = torch.empty_like(q)
        lse = torch.empty(b, h, t, dtype=torch.float32, device=q.device)
        how = dict(scale=scale, softcap=softcap)
        ops.score_attention_fwd(q, k, v, o, lse, **how, **dict(zip(_MASKS, masks)))
        # the masks may be the caller's own buffers: autograd notices if they are written to
        # before the backward (tensors of inference mode have no versions, hence copies)
        ctx.save_for_backward(q, k, v, o, lse, *(
            m.clone() if m is not None and m.is_inference() else m for m in masks))
        ctx.how, ctx.rope = how, rope
        return o

    @staticmethod
    def backward(ctx, do):
        q, k, v, o, lse, *masks = ctx.saved_tensors
        do = do.contiguous().to(torch.bfloat16)
        dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
        ops.score_attention_bwd(q, k, v, o, do, lse, dq, dk, dv, rope=ctx.rope, **ctx.how,
                                **dict(zip(_MASKS, masks)))
        return dq, dk, dv, *[None] * (3 + len(masks))


def make_score_attention(config: ScoreAttentionConfig = ScoreAttentionConfig(), *,
                         rope_tables=None) -> Callable:
    """Returns attention(q, k, v, *, slopes, segment_ids, prefix_lens) over BHSD
    bf16 tensors; k and v may have fewer heads than q. Slopes are constants: those
    that require a gradient are refused. With `rope_tables` (from
    `ops.rope_tables`) q and k are rotated first, as in `make_causal_attention`."""

    def attention(q, k, v, *, slopes=None, segment_ids=None, prefix_lens=None):
        _validate(q, k, v)
        scale = config.softmax_scale if config.softmax_scale is not None else q.shape[-1] ** -0.5
        if slopes is not None:
            if slopes.requires_grad and torch.is_grad_enabled():
                raise ValueError("slopes are constants: the attention gives them no gradient "
                                 "(pass slopes.detach())")
            slopes = slopes.detach().to(device=q.device, dtype=torch.float32).contiguous()
        ints = [None if t is None else t.to(device=q.device, dtype=torch.int32).contiguous()
                for t in (segment_ids, prefix_lens)]
        return _ScoreAttention.apply(q, k, v, float(scale), float(config.softcap), rope_tables,
                                     slopes, *ints)

    return attention
