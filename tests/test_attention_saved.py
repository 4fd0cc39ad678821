"""What the attention factories keep of a call for its backward: the caller may reuse
its mask buffers for the next batch, and hears of it where that comes too early."""

import pytest
import torch

from rig_b200 import kernels, ops

B, H, KV, T = 2, 4, 2, 150


def _inputs(dev):
    g = torch.Generator().manual_seed(4)
    q = torch.randn(B, H, T, 64, generator=g).bfloat16().to(dev)
    k, v = (torch.randn(B, KV, T, 64, generator=g).bfloat16().to(dev) for _ in range(2))
    do = torch.randn(B, H, T, 64, generator=g).bfloat16().to(dev)
    masks = dict(slopes=kernels.distance_slopes(H, dev),
                 segment_ids=(torch.arange(T, device=dev) // 40).int().expand(B, T).contiguous(),
                 prefix_lens=torch.tensor([9, 70], dtype=torch.int32, device=dev))
    return [x.requires_grad_(True) for x in (q, k, v)], do, masks


def _reuse(name, t):
    t.copy_(t * 2 if name == "slopes" else t // 2)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["slopes", "segment_ids", "prefix_lens"])
def test_mask_overwritten_before_the_backward(cuda, name):
    qkv, do, masks = _inputs(cuda)
    attention = kernels.make_score_attention(kernels.ScoreAttentionConfig(softcap=30.0))
    y = attention(*qkv, **masks)
    _reuse(name, masks[name])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(do)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["slopes", "segment_ids", "prefix_lens"])
@pytest.mark.parametrize("kind", ["converted", "inference"])
def test_mask_that_was_copied_may_be_overwritten(cuda, name, kind):
    """A mask of another type, which the call converts, and one without versions."""

    qkv, do, masks = _inputs(cuda)
    attention = kernels.make_score_attention(kernels.ScoreAttentionConfig(softcap=30.0))
    y = attention(*qkv, **masks)
    want = torch.autograd.grad(y, qkv, do)
    if kind == "converted":
        masks[name] = masks[name].double() if name == "slopes" else masks[name].long()
    else:
        with torch.inference_mode():
            masks[name] = masks[name].clone()
    y = attention(*qkv, **masks)
    with torch.inference_mode():
        _reuse(name, masks[name])
    got = torch.autograd.grad(y, qkv, do)
    assert torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])
    assert (got[0].float() - want[0].float()).norm() <= 1e-3 * want[0].float().norm()


@pytest.mark.gpu
def test_gradients_twice_and_without_masks(cuda):
    qkv, do, masks = _inputs(cuda)
    for how in (masks, {}):
        attention = kernels.make_score_attention(rope_tables=ops.rope_tables(T, 64, cuda))
        y = attention(*qkv, **how)
        first = torch.autograd.grad(y, qkv, do, retain_graph=True)
        again = torch.autograd.grad(y, qkv, do)
        assert torch.equal(first[1], again[1]) and torch.equal(first[2], again[2])


def test_slopes_have_no_gradient():
    """Learned slopes are refused (before anything runs), not left without a gradient."""

    q, k, v = (torch.randn(1, 2, 8, 64).bfloat16() for _ in range(3))
    attention = kernels.make_score_attention()
    slopes = torch.zeros(2, requires_grad=True)
    with pytest.raises(ValueError, match="gradient"):
        attention(q, k, v, slopes=slopes)
    with pytest.raises(ValueError, match="gradient"):
        attention(q, k, v, slopes=torch.exp(slopes))
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):  # as any CPU tensor
        attention(q, k, v, slopes=slopes)


@pytest.mark.gpu
def test_slopes_that_require_a_gradient_without_one(cuda):
    qkv, _, masks = _inputs(cuda)
    attention = kernels.make_score_attention()
    want = attention(*qkv, **masks)
    learned = masks["slopes"].clone().requires_grad_(True)
    with torch.no_grad():
        got = attention(*qkv, **{**masks, "slopes": learned})
    assert torch.equal(got, want)


@pytest.mark.gpu
def test_plain_attention_ids_overwritten_before_the_backward(cuda):
    qkv, do, masks = _inputs(cuda)
    q, k, v = (x.detach()[:, :KV].contiguous().requires_grad_(True) for x in qkv)
    do, ids = do[:, :KV].contiguous(), masks["segment_ids"]
    attention = kernels.make_causal_attention()
    want = torch.autograd.grad(attention(q, k, v, ids), (q, k, v), do)
    with torch.inference_mode():
        other = ids.clone()
    y = attention(q, k, v, other)
    with torch.inference_mode():
        _reuse("segment_ids", other)
    got = torch.autograd.grad(y, (q, k, v), do)
    assert torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])
    y = attention(q, k, v, ids)
    _reuse("segment_ids", ids)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(do)
