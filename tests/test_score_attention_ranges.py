"""Score-modified attention at the ends of its inputs' ranges, against the formula in
64 bits. Formula and elementwise tolerances are those of test_score_attention."""

import pytest
import torch

from rig_b200 import kernels
from test_score_attention import _check, _formula, _inputs, _run


@pytest.mark.gpu
@pytest.mark.parametrize("cap,bias", [(0.0, False), (0.0, True), (50.0, False), (50.0, True)])
@pytest.mark.parametrize("power", [0, 108, -100])
def test_far_keys_above_the_near_ones(cuda, cap, bias, power):
    """Keys of the first tile whose scores lie 0 to 58 bits above those of a row's own
    tile, which no mask reaches: the row's sums start against a reference that they
    outgrow. Values of 2^108 and 2^-100 too, which the results can hold: an output is
    at most max |v| < 2^111, so nothing on the way may reach 2^17 times it. The
    incoming gradient moves against them (do.v has to be finite), and as everything
    is linear in either, the results go back to the formula's by powers of two."""

    t = 520
    q, k, v, do = (x.to(cuda) for x in _inputs(1, 2, 1, t, 21, 1.0))
    lift = torch.tensor([0.0, 1.0, 1.7, 2.6, 3.2, 4.0, 5.0], device=cuda)  # 8 nats each
    row = torch.arange(t, device=cuda) // 32 % 7  # alike within a warp, which decides as one
    q = (q.float() / 4 + lift[row][None, None, :, None]).bfloat16()
    k = k.float() / 4
    k[:, :, :128] += 1.0
    k = k.bfloat16()
    # small slopes: the bias is there, but does not undo the lift
    slopes = torch.tensor([2.0 ** -9, 2.0 ** -7], device=cuda) if bias else None
    want, tol, want_lse = _formula(q, k, v, do, 0.125, cap, slopes, None, None)
    first, own = (torch.logsumexp((0.125 * q.double() @ k.double().transpose(-1, -2))[..., 256:, w], -1)
                  for w in (slice(0, 128), slice(256, 384)))
    assert (first - own).max() > 40 and (first - own).min() < 8  # nats
    size, back = 2.0 ** power, 2.0 ** (-power // 4)
    got, lse = _run(q, k, (v.double() * size).bfloat16(), (do.double() * back).bfloat16(), scale=0.125,
                    softcap=cap, slopes=slopes)
    got = {n: x.double() / (size if n == "o" else back if n == "dv" else size * back)
           for n, x in got.items()}
    assert all(torch.isfinite(x).all() for x in got.values())
    _check(got, lse, want, tol, want_lse)


@pytest.mark.gpu
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("cap,spread", [(200.0, 30.0), (200.0, 100.0), (1000.0, 150.0), (1000.0, 300.0),
                                        (4000.0, 300.0), (65536.0, 300.0)])
def test_large_caps(cuda, cap, spread, bias):
    """Scores of hundreds under a cap of their size: an error of the tanh counts cap times
    over. fp32 scores and tanh are a few roundings, so s' is off by at most 8 units of
    2^-23 of its largest value, and the lse by that and its own roundings, 16 in all.
    That is at most 0.0027 of a probability here. H + E of the formula holds 0.0049, of
    which bf16 takes 0.0039: 1.2 times as much, 0.0059, has room for both."""

    q, k, v, do = (x.to(cuda) for x in _inputs(1, 2, 2, 300, 17, spread))
    slopes = kernels.distance_slopes(2, cuda) if bias else None
    want, tol, want_lse = _formula(q, k, v, do, 0.125, cap, slopes, None, None)
    s = 0.125 * q.double() @ k.double().transpose(-1, -2)
    top = (cap * torch.tanh(s / cap)).abs().max().item()
    assert top > 100
    got, lse = _run(q, k, v, do, scale=0.125, softcap=cap, slopes=slopes)
    assert (lse.double() - want_lse).abs().max() <= 16 * 2.0 ** -23 * top
    for n in want:
        assert ((got[n].double() - want[n]).abs() <= 1.2 * tol[n]).all(), n


@pytest.mark.gpu
@pytest.mark.parametrize("cap", [1e-40, 1e-38, 1e-20, 1e-6])
def test_tiny_caps(cuda, cap):
    """Next to nothing is left of any score, scores of exactly 0 among them: the mean of
    the values. (Without a bias; 1e-40 is a denormal number, scale / cap overflows.)"""

    q, k, v, do = (x.to(cuda) for x in _inputs(1, 2, 1, 300, 23))
    q[:, :, ::5] = 0
    k[:, :, 7::11] = 0
    want, tol, want_lse = _formula(q, k, v, do, 0.125, cap, None, None, None)
    got, lse = _run(q, k, v, do, scale=0.125, softcap=cap)
    _check(got, lse, want, tol, want_lse)
