"""Score-modified attention against its formula in 64 bits, forward and gradients.

Tolerances, element by element from the formula's own matrices. H = 2^-8 bounds
the relative rounding to bf16 (8 significant bits). The kernels round P and dS to
bf16 before their products and the results once, and compute p in fp32 with a
relative error E: tanh's 7e-6 times |s'| <= 60, exp2 and fp32 scores of the same
order, so E = 2^-10 is ample. Hence
  o:  (H + E) sum_j p |v| + H |o|
  dv: (H + E) sum_i p |do| + H |dv|
  ds: (H + E) |ds| + p (delta's error, sum_e |do| tol(o)) + E p (|dp| + |delta|) / 8
      (the last for the slope 1 - tanh^2 of saturated scores and fp32 sums)
  dq: scale sum_j tol(ds) |k| + H |dq|, dk: scale sum_i tol(ds) |q| + H |dk|,
and a group's heads add up. A few units of 1e-6 stand for the fp32 sums of zero.
"""

import ctypes
import math

import numpy as np
import pytest
import torch

from rig_b200 import _lib, kernels, ops

H, E = 2.0 ** -8, 2.0 ** -10


def _inputs(b, h, kv, t, seed=0, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    q = (spread * torch.randn(b, h, t, 64, generator=g)).bfloat16()
    k, v = (torch.randn(b, kv, t, 64, generator=g).bfloat16() for _ in range(2))
    do = torch.randn(b, h, t, 64, generator=g).bfloat16()
    return q, k, v, do


def _masks(kind, b, t, seed=0):
    """(segment ids, prefix lengths)."""

    rng = np.random.default_rng(seed)
    seg = prefix = None
    if "docs" in kind:
        seg = np.cumsum(rng.random((b, t)) < min(0.5, 5.0 / t), 1)
    if "random" in kind:  # ids that are not monotone, with holes of padding
        seg = rng.integers(-1, 3, (b, t))
    if "padded" in kind:  # right padding; the first sequence is padding alone when b > 1
        keep = rng.integers(1, t + 1, b)
        keep[0] = 0 if b > 1 else keep[0]
        seg = np.where(np.arange(t) < keep[:, None], 4 if seg is None else seg, -7)
    if "prefix" in kind:
        prefix = rng.integers(0, t + 1, b)
        prefix[-1] = {0: 0, 1: t, 2: t + 9, 3: -3}[seed % 4]
    to = lambda a: None if a is None else torch.from_numpy(np.ascontiguousarray(a.astype(np.int32)))  # noqa: E731
    return to(seg), to(prefix)


def _formula(q, k, v, do, scale, cap, slopes, seg, prefix):
    """Values and tolerances of o, dq, dk, dv (module docstring), and the lse."""

    q, k, v, do = (x.double() for x in (q, k, v, do))
    b, h, t, d = q.shape
    group = h // k.shape[1]
    kx, vx = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    i = torch.arange(t, device=q.device)
    see = (i[None] <= i[:, None])[None]
    if prefix is not None:
        see = see | (i[None, None] < prefix[:, None, None])
    if seg is not None:
        see = see & (seg[:, :, None] == seg[:, None]) & (seg[:, :, None] >= 0)
    see = see[:, None].expand(b, h, t, t)
    s = scale * q @ kx.transpose(-1, -2)
    slope = torch.ones_like(s)
    if cap:
        th = torch.tanh(s / cap)
        s, slope = cap * th, 1 - th * th
    if slopes is not None:
        s = s - slopes.double()[:, None, None] * (i[None] - i[:, None]).abs()
    s = s.masked_fill(~see, -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - torch.where(lse == -math.inf, 0.0, lse)[..., None])
    o = p @ vx
    dp, delta = do @ vx.transpose(-1, -2), (do * o).sum(-1, keepdim=True)
    ds = p * (dp - delta) * slope
    to = (H + E) * p @ vx.abs() + H * o.abs()
    tds = (H + E) * ds.abs() + p * slope * (do.abs() * to).sum(-1, keepdim=True) + \
        E / 8 * p * (dp.abs() + delta.abs())
    back = lambda x: x.view(b, -1, group, t, d).sum(2)  # noqa: E731
    dq = scale * ds @ kx
    dk = back(scale * ds.transpose(-1, -2) @ q)
    dv = back(p.transpose(-1, -2) @ do)
    tol = dict(o=to, dq=scale * tds @ kx.abs() + H * dq.abs(),
               dk=back(scale * tds.transpose(-1, -2) @ q.abs()) + H * dk.abs(),
               dv=back((H + E) * p.transpose(-1, -2) @ do.abs()) + H * dv.abs())
    return dict(o=o, dq=dq, dk=dk, dv=dv), {n: x + 4e-6 for n, x in tol.items()}, lse


def _run(q, k, v, do, **how):
    b, h, t, _ = q.shape
    o, lse = torch.empty_like(q), torch.empty(b, h, t, device=q.device)
    ops.score_attention_fwd(q, k, v, o, lse, **how)
    grads = [torch.full_like(x, 7.0) for x in (q, k, v)]
    ops.score_attention_bwd(q, k, v, o, do, lse, *grads, **how)
    torch.cuda.synchronize()
    assert ops.device_error() == 0
    return dict(zip(("o", "dq", "dk", "dv"), (o, *grads))), lse


def _check(got, lse, want, tol, want_lse):
    for n in want:
        off = (got[n].double() - want[n]).abs()
        assert (off <= tol[n]).all(), (n, off.max().item(), (off / tol[n]).max().item())
    empty = want_lse == -math.inf
    assert torch.equal(lse == -math.inf, empty)
    # fp32 statistics: scores to 7e-6 relative, their sum's logarithm
    near = (lse.double() - want_lse)[~empty].abs() <= 1e-4 + 1e-5 * want_lse[~empty].abs()
    assert near.all()
    assert (got["o"][empty] == 0).all() and (got["dq"][empty] == 0).all()


CASES = [
    # b, h, kv, t, mask, softcap, bias
    (1, 1, 1, 1, "causal", 30.0, True),
    (2, 2, 1, 2, "causal", 0.0, False),
    (2, 2, 2, 7, "padded", 30.0, True),
    (1, 3, 1, 64, "prefix", 0.0, True),
    (2, 4, 2, 127, "docs", 50.0, False),
    (1, 2, 2, 128, "causal", 5.0, False),
    (2, 2, 1, 129, "random", 30.0, True),
    (3, 4, 1, 200, "prefix", 20.0, True),
    (2, 6, 2, 257, "padded", 0.0, False),
    (3, 2, 2, 300, "docs+prefix", 30.0, True),
    (2, 3, 3, 385, "random+prefix", 0.0, True),
    (1, 4, 4, 640, "padded+prefix", 15.0, False),
    (3, 2, 1, 1000, "docs+padded", 30.0, True),
    (1, 2, 2, 1025, "causal", 50.0, True),
    (1, 2, 1, 2049, "docs", 30.0, True),
    (1, 2, 2, 2300, "prefix", 30.0, True),
    (2, 3, 1, 2111, "causal", 0.0, False),
]


@pytest.mark.gpu
@pytest.mark.parametrize("b,h,kv,t,mask,cap,bias", CASES)
def test_formula(cuda, b, h, kv, t, mask, cap, bias):
    for seed in (0, 1) if t < 1000 else (2,):
        q, k, v, do = (x.to(cuda) for x in _inputs(b, h, kv, t, seed))
        seg, prefix = (None if x is None else x.to(cuda) for x in _masks(mask, b, t, seed))
        slopes = kernels.distance_slopes(h, cuda) if bias else None
        want, tol, want_lse = _formula(q, k, v, do, 0.125, cap, slopes, seg, prefix)
        got, lse = _run(q, k, v, do, scale=0.125, softcap=cap, slopes=slopes, segment_ids=seg,
                        prefix_lens=prefix)
        _check(got, lse, want, tol, want_lse)


@pytest.mark.gpu
@pytest.mark.parametrize("edges", [(64,), (192,), (256,), (320,), (64, 128), (128, 192, 320)])
def test_padding_from_chunk_and_tile_boundaries(cuda, edges):
    """Padding that starts or ends where the kernels' 64- and 128-position tiles do,
    with whole tiles of it between tokens of one id; prefixes over both."""

    t = 400
    seg = torch.zeros(2, t, dtype=torch.int32)
    for i in range(t):  # tokens and padding in turn, from edge to edge
        seg[:, i] = 0 if sum(i >= e for e in edges) % 2 == 0 else -1
    seg[1] = torch.where(seg[1] < 0, 2, -1)
    seg = seg.to(cuda)
    for cap, bias, prefix in ((30.0, True, None), (0.0, False, [t, 100])):
        q, k, v, do = (x.to(cuda) for x in _inputs(2, 2, 1, t, 12))
        how = dict(softcap=cap, slopes=kernels.distance_slopes(2, cuda) if bias else None,
                   segment_ids=seg,
                   prefix_lens=None if prefix is None else torch.tensor(prefix, dtype=torch.int32, device=cuda))
        want, tol, want_lse = _formula(q, k, v, do, 0.125, cap, how["slopes"], seg, how["prefix_lens"])
        got, lse = _run(q, k, v, do, scale=0.125, **how)
        _check(got, lse, want, tol, want_lse)


@pytest.mark.gpu
@pytest.mark.parametrize("cap,spread", [(1.5, 12.0), (30.0, 40.0), (4.0, 3.0), (1e4, 3.0)])
def test_cap_from_linear_to_saturated(cuda, cap, spread):
    """Both forms of tanh, and scores around the limit between them."""

    q, k, v, do = (x.to(cuda) for x in _inputs(1, 2, 2, 330, 3, spread))
    want, tol, want_lse = _formula(q, k, v, do, 0.125, cap, None, None, None)
    got, lse = _run(q, k, v, do, scale=0.125, softcap=cap)
    _check(got, lse, want, tol, want_lse)


@pytest.mark.gpu
def test_slopes_of_either_sign_and_zero(cuda):
    """slopes 0, large, and negative (favouring far keys), one per head."""

    q, k, v, do = (x.to(cuda) for x in _inputs(2, 4, 2, 300, 4))
    slopes = torch.tensor([0.0, 3.0, -0.02, 0.5], device=cuda)
    prefix = torch.tensor([40, 290], dtype=torch.int32, device=cuda)
    want, tol, want_lse = _formula(q, k, v, do, 0.125, 0.0, slopes, None, prefix)
    got, lse = _run(q, k, v, do, scale=0.125, slopes=slopes, prefix_lens=prefix)
    _check(got, lse, want, tol, want_lse)


@pytest.mark.gpu
def test_plain_options_agree_with_causal_attention(cuda):
    """Without cap, bias, prefix and padding this is the plain kernels' attention.
    The two round P against different row maxima, so each is within the formula's
    bounds and they are within twice those of each other."""

    for t, ids in ((300, False), (300, True), (2100, False)):
        q, k, v, do = (x.to(cuda) for x in _inputs(2, 2, 2, t, 5))
        seg = _masks("docs", 2, t)[0].to(cuda) if ids else None
        got, lse = _run(q, k, v, do, scale=0.125, segment_ids=seg)
        o, plain = torch.empty_like(q), torch.empty_like(lse)
        ops.attention_fwd(q, k, v, o, plain, scale=0.125, segment_ids=seg)
        grads = [torch.empty_like(x) for x in (q, k, v)]
        ops.attention_bwd(q, k, v, o, do, plain, *grads, scale=0.125, segment_ids=seg)
        assert (lse - plain).abs().max() <= 32 * 2.0 ** -24 * (1 + plain.abs().max())
        _, tol, _ = _formula(q, k, v, do, 0.125, 0.0, None, seg, None)
        for n, want in zip(("o", "dq", "dk", "dv"), (o, *grads)):
            assert ((got[n].double() - want.double()).abs() <= 2 * tol[n]).all(), n


@pytest.mark.gpu
@pytest.mark.parametrize("mask", ["causal", "docs+padded", "prefix"])
def test_layouts_and_strides(cuda, mask):
    """Slices of one packed [B, T, H + 2 KV, 64] projection with gradients into its
    twin, a padded do, against contiguous BHSD tensors; the gaps stay untouched."""

    b, h, kv, t = 2, 4, 2, 333
    q, k, v, do = (x.to(cuda) for x in _inputs(b, h, kv, t, 6))
    seg, prefix = (None if x is None else x.to(cuda) for x in _masks(mask, b, t))
    how = dict(scale=0.125, softcap=30.0, slopes=kernels.distance_slopes(h, cuda), segment_ids=seg,
               prefix_lens=prefix)
    want, lse = _run(q, k, v, do, **how)
    packed = torch.cat([x.transpose(1, 2) for x in (q, k, v)], 2)
    wide = torch.full((b, t, h + 1, 72), float("nan"), device=cuda).bfloat16()
    wide[:, :, :h, :64] = do.transpose(1, 2)
    qp, kp, vp = packed.split([h, kv, kv], 2)
    dop = wide[:, :, :h, :64]
    o = torch.empty(b, t, h, 64, device=cuda, dtype=torch.bfloat16)
    lse2 = torch.empty_like(lse)
    ops.score_attention_fwd(qp, kp, vp, o, lse2, layout="bthd", **how)
    grads = torch.full((b, t, h + 2 * kv + 1, 64), 9.0, device=cuda).bfloat16()
    dq, dk, dv, gap = grads.split([h, kv, kv, 1], 2)
    ops.score_attention_bwd(qp, kp, vp, o, dop, lse2, dq, dk, dv, layout="bthd", **how)
    assert torch.equal(o.transpose(1, 2), want["o"]) and torch.equal(lse2, lse)
    assert torch.equal(dk.transpose(1, 2), want["dk"]) and torch.equal(dv.transpose(1, 2), want["dv"])
    assert (dq.transpose(1, 2).double() - want["dq"].double()).norm() <= 1e-4 * want["dq"].double().norm()
    assert (gap == 9).all()


@pytest.mark.gpu
def test_masked_places_do_not_leak(cuda):
    """Large finite values at hidden keys and padded queries change nothing."""

    b, h, t = 2, 2, 260
    q, k, v, do = (x.to(cuda) for x in _inputs(b, h, h, t, 7))
    seg = torch.zeros(b, t, dtype=torch.int32, device=cuda)
    seg[0, 100:] = -1
    seg[1, 40:200] = -5
    how = dict(scale=0.125, softcap=30.0, segment_ids=seg)
    a, lse_a = _run(q, k, v, do, **how)
    hidden = (seg < 0)[:, None, :, None]
    big = torch.finfo(torch.bfloat16).max
    q2, k2 = (torch.where(hidden, 1e4, x) for x in (q, k))
    v2, do2 = (torch.where(hidden, 1e30, x) for x in (v, do))
    c, lse_c = _run(q2, k2, v2, do2, **how)
    assert big > 1e30 and torch.equal(lse_a, lse_c)
    for n in ("o", "dk", "dv"):
        assert torch.equal(a[n], c[n]), n
    assert (a["dq"].double() - c["dq"].double()).norm() <= 1e-4 * a["dq"].double().norm()
    assert (a["o"][hidden.expand_as(q)] == 0).all() and (a["dv"][hidden.expand_as(q)] == 0).all()


@pytest.mark.gpu
def test_gradients_against_differences(cuda):
    """Directional differences of the kernel's own forward. Inputs and steps are
    multiples of 2^-4, exact in bf16, along the sign of the gradient, where
    L = sum(o * do) changes by 2 h sum |g|. Each o is off by at most 2^-7 sum p |v|
    (P and the result), about 0.01 an element and independent, so L by 0.01 *
    sqrt(2 * 96 * 64) ~ 1 against changes of 30 and more; the curvature along a
    step of 2^-4 is another few percent: 10% in all."""

    t, cap = 96, 8.0
    g = torch.Generator().manual_seed(8)
    q, k, v = ((torch.randint(-24, 25, (1, n, t, 64), generator=g) / 16).bfloat16().to(cuda)
               for n in (2, 1, 1))
    do = torch.randn(1, 2, t, 64, generator=g).bfloat16().to(cuda)
    how = dict(slopes=kernels.distance_slopes(2, cuda),
               segment_ids=_masks("docs", 1, t)[0].to(cuda),
               prefix_lens=torch.tensor([30], dtype=torch.int32, device=cuda))
    attention = kernels.make_score_attention(kernels.ScoreAttentionConfig(softcap=cap))
    args = [x.clone().requires_grad_(True) for x in (q, k, v)]
    attention(*args, **how).backward(do)
    h = 2.0 ** -4
    for i, a in enumerate(args):
        u = torch.sign(a.grad)
        ends = []
        for s in (h, -h):
            moved = [x + (s * u if j == i else 0) for j, x in enumerate((q, k, v))]
            ends.append((attention(*moved, **how).double() * do.double()).sum().item())
        want = 2 * h * a.grad.double().abs().sum().item()
        assert want > 20
        assert abs(ends[0] - ends[1] - want) <= 0.1 * want, (i, ends[0] - ends[1], want)


@pytest.mark.gpu
def test_rope_and_streams(cuda):
    """RoPE's backward inside the kernel (as the plain attention's), on a side stream."""

    t = 200
    q, k, v, do = (x.to(cuda) for x in _inputs(1, 2, 1, t, 9, 1.0))
    rope = ops.rope_tables(t, 64, cuda)
    attention = kernels.make_score_attention(kernels.ScoreAttentionConfig(softcap=30.0), rope_tables=rope)
    args = [x.clone().requires_grad_(True) for x in (q, k, v)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = attention(*args)
        y.backward(do)
    side.synchronize()
    qr, kr = q.clone(), k.clone()
    for x in (qr, kr):
        ops.rope_apply(x.transpose(1, 2), rope)
    got, _ = _run(qr, kr, v, do, scale=0.125, softcap=30.0)
    assert torch.equal(y, got["o"]) and torch.equal(args[2].grad, got["dv"])
    for a, n in ((args[0], "dq"), (args[1], "dk")):
        back = got[n].clone()
        ops.rope_apply(back.transpose(1, 2), rope, inverse=True)
        # the kernel rotates before it rounds, the other way rounds twice
        assert (a.grad.double() - back.double()).norm() <= 2 * H * back.double().norm()


@pytest.mark.gpu
def test_refusals(cuda):
    q, k, v, do = (x.to(cuda) for x in _inputs(1, 4, 2, 16))
    o, lse = torch.empty_like(q), torch.empty(1, 4, 16, device=cuda)
    run = lambda *a, **kw: ops.score_attention_fwd(*a, **{"scale": 0.125, **kw})  # noqa: E731
    with pytest.raises(ValueError):
        run(q[:, :3], k, v, o[:, :3], lse[:, :3].contiguous())  # 3 heads on 2
    with pytest.raises(ValueError):
        run(q, k, v[:, :, :8], o, lse)
    with pytest.raises(ValueError):
        run(q.float(), k, v, o, lse)
    with pytest.raises(ValueError):
        run(q, k, v, o, lse[..., :8])
    with pytest.raises(ValueError):
        run(q, k, v, o, lse, slopes=torch.zeros(2, device=cuda))
    with pytest.raises(ValueError):
        run(q, k, v, o, lse, segment_ids=torch.zeros(1, 16, device=cuda))
    with pytest.raises(ValueError):
        run(q, k, v, o, lse, prefix_lens=torch.zeros(2, dtype=torch.int32, device=cuda))
    with pytest.raises(ValueError):
        run(q, k, v, o, lse, layout="sbhd")
    for bad in (dict(softcap=-1.0), dict(softcap=float("inf")), dict(softcap=float("nan")),
                dict(scale=0.0), dict(scale=float("nan"))):
        with pytest.raises(_lib.GptB200Error):
            run(q, k, v, o, lse, **bad)
    with pytest.raises(_lib.GptB200Error):  # head_dim 32
        run(q[..., :32], k[..., :32], v[..., :32], o[..., :32], lse)
    wide = torch.empty(1, 4, 16, 68, device=cuda, dtype=torch.bfloat16)[..., :64]  # rows off 16 bytes
    with pytest.raises(_lib.GptB200Error):
        run(wide, k, v, o, lse)
    with pytest.raises(ValueError):
        ops.score_attention_bwd(q, k, v, o, do, lse, q, k, v, scale=0.125,
                                workspace=torch.empty(16, dtype=torch.uint8, device=cuda))


def test_arguments_are_checked_without_a_gpu():
    for bad in (dict(softcap=-1.0), dict(softcap=math.inf), dict(softmax_scale=0.0)):
        with pytest.raises(ValueError):
            kernels.ScoreAttentionConfig(**bad)
    attention = kernels.make_score_attention()
    q, k, v, _ = _inputs(1, 4, 2, 8)
    with pytest.raises(ValueError):
        attention(q, k, v)  # CPU tensors
    with pytest.raises(ValueError):
        attention(q[:, :3], k, v)
    with pytest.raises(TypeError):
        attention(q.float(), k.float(), v.float())
    lib = _lib.load()
    assert lib.gptb200_score_attention_fwd(None, None) == 1
    empty = _lib.ScoreAttention()
    assert lib.gptb200_score_attention_fwd(ctypes.byref(empty), None) == 1
    one = _lib.ScoreAttention(16, 16, 16, (64, 64, 64), (64, 64, 64), 16, (64, 64, 64), 16, 1, 3, 2, 8, 64,
                              0.125, 0.0, None, None, None)
    assert lib.gptb200_score_attention_fwd(ctypes.byref(one), None) == 3  # 3 heads on 2
    one.kv_heads, one.q_stride[2] = 3, 60
    assert lib.gptb200_score_attention_fwd(ctypes.byref(one), None) == 2  # rows off 16 bytes
