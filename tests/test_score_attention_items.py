"""Score-modified attention where every block of the persistent kernels takes several
items of unequal length, at both orders of the items; and its errors by norm.

Every head of every sequence is held against the formula in 64 bits and its
elementwise tolerances (test_score_attention). Those add worst cases up, so a
systematic error of a few percent would pass: the errors are held by norm too. A
rounding to bf16 is off by 0.0017 of a tensor (2^-8 / 2 at most, uniform). o and dv
carry two, P's and their own: 0.0024, bound 0.003. dq and dk carry dS's and their own,
and the errors of o in delta, which weigh up to twice as much where one key holds most
of a row: sqrt(2 + 4) roundings, 0.0042, up to 0.0046 where rows see eight keys or
less. Bound 0.006."""

import pytest
import torch

from rig_b200 import kernels
from test_score_attention import _formula, _inputs, _masks, _run

NORM = dict(o=0.003, dv=0.003, dq=0.006, dk=0.006)


def _hold(cuda, b, h, kv, t, seg, prefix, cap, bias, seed):
    q, k, v, do = (x.to(cuda) for x in _inputs(b, h, kv, t, seed))
    slopes = kernels.distance_slopes(h, cuda) if bias else None
    got, lse = _run(q, k, v, do, scale=0.125, softcap=cap, slopes=slopes, segment_ids=seg, prefix_lens=prefix)
    total = {n: [0.0, 0.0] for n in got}
    for i in range(b):
        one = slice(i, i + 1)
        want, tol, want_lse = _formula(q[one], k[one], v[one], do[one], 0.125, cap, slopes,
                                       None if seg is None else seg[one],
                                       None if prefix is None else prefix[one])
        empty = want_lse == -torch.inf
        assert torch.equal(lse[one] == -torch.inf, empty)
        assert ((lse[one].double() - want_lse)[~empty].abs() <= 1e-4 + 1e-5 * want_lse[~empty].abs()).all()
        for n in want:
            off = (got[n][one].double() - want[n]).abs()
            assert (off <= tol[n]).all(), (n, i, (off / tol[n]).max().item())
            total[n][0] += off.square().sum().item()
            total[n][1] += want[n].square().sum().item()
    for n, (off, size) in total.items():
        assert off ** 0.5 <= NORM[n] * size ** 0.5, (n, (off / size) ** 0.5)


SEVERAL = [  # 960 to 3,072 items of a forward, 1,440 to 2,592 of a backward; 148 blocks
    (16, 12, 12, 1025, "causal", 50.0, True),
    (16, 12, 12, 1025, "causal", 0.0, False),
    (40, 12, 6, 700, "docs+padded", 30.0, False),
    (64, 12, 4, 777, "prefix", 0.0, True),
    (48, 8, 4, 1000, "random+prefix", 15.0, True),
    (30, 12, 12, 513, "padded", 20.0, True),
    (24, 6, 6, 2300, "docs+prefix", 30.0, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("b,h,kv,t,mask,cap,bias", SEVERAL)
def test_several_items_a_block(cuda, b, h, kv, t, mask, cap, bias):
    assert -(-t // 256) * b * h >= 6 * 148 and -(-t // 128) * b * kv >= 6 * 148
    seg, prefix = (None if x is None else x.to(cuda) for x in _masks(mask, b, t, 3))
    _hold(cuda, b, h, kv, t, seg, prefix, cap, bias, 31)


HEAD_BY_HEAD = [  # shared tiles past every limit below which items go by weight
    (64, 16, 16, 521, "causal", 0.0, False),
    (64, 16, 16, 521, "docs", 0.0, True),
    (64, 32, 16, 520, "docs+padded", 30.0, True),
    (64, 32, 16, 515, "prefix", 30.0, False),
    (64, 32, 16, 517, "causal", 200.0, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("b,h,kv,t,mask,cap,bias", HEAD_BY_HEAD)
def test_items_head_by_head(cuda, b, h, kv, t, mask, cap, bias):
    assert b * kv * t * 256 > 128 << 20 and b * h * t * 256 > (256 if cap else 64) << 20
    seg, prefix = (None if x is None else x.to(cuda) for x in _masks(mask, b, t, 5))
    _hold(cuda, b, h, kv, t, seg, prefix, cap, bias, 37)


@pytest.mark.gpu
@pytest.mark.parametrize("t,document", [(16, None), (33, None), (128, None), (129, None), (300, None), (1025, None),
                                        (1024, 8), (1024, 16), (1024, 33), (1024, 64), (1000, 300), (160, 54)])
@pytest.mark.parametrize("cap,bias", [(0.0, False), (30.0, True)])
def test_short_rows(cuda, t, document, cap, bias):
    """Few keys to a row, from short sequences or from short documents in long ones."""

    b, h = 4, 4
    seg = None
    if document:
        seg = (torch.arange(t, device=cuda) // document).int().expand(b, t).contiguous()
    _hold(cuda, b, h, 2, t, seg, None, cap, bias, 41)
