"""Layer norm of constant rows and of rows far from zero, at widths that are and are
not powers of two, against the formulas in 64 bits.

Tolerances. The mean is an fp32 number, so the rows' distances from it are off by up
to half a unit of its last place, M = 2^-24 max |x| with room for the sums behind it
(which are small: they are taken again over the distances). hat is off by M rstd from
there and by some 2^-20 of itself and of one from its own operations, W. A sum over the
row weighs that with its terms, so dx, whose sums are means, is off by
rstd max |dn| (1 + |hat|) times a few such errors: 4. Column sums add the rows' errors
and chain at most 64 roundings here."""

import pytest
import torch

from rig_b200 import ops

EPS = 1e-5
W = 2.0 ** -20


def _run(dev, x, w, b, dy):
    x, w, b, dy = (t.to(dev) for t in (x, w, b, dy))
    n, d = x.shape
    y, dx = torch.empty_like(x), torch.empty_like(x)
    mean, rstd = torch.empty(2, n, device=dev).unbind()
    ops.layer_norm_fwd(x, w, b, y, mean, rstd, EPS)
    ds, db = torch.zeros(2, d, device=dev).unbind()
    ops.layer_norm_bwd(x, w, mean, rstd, dy, None, dx, ds, db)
    torch.cuda.synchronize()
    return (t.cpu().double() for t in (y, dx, ds, mean, rstd))


WIDTHS = [8, 40, 257, 512, 768, 771, 1000, 1032, 1999, 4096, 4099, 6000, 16384]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", WIDTHS)
def test_constant_rows_give_the_bias(cuda, d, dtype):
    """Every sum of equal numbers that fp32 holds exactly, and some that it does not
    (0.1, pi): the mean is the number, y the bias, and x counts for nothing in dscale."""

    g = torch.Generator().manual_seed(d)
    values = torch.cat([torch.tensor([1.2578125, 0.1, -3.14159274, 1e-3, 1e4, 65280.0, 0.0, -0.7]),
                        torch.randn(24, generator=g)]).to(dtype)
    x = values[:, None].expand(-1, d).contiguous()
    w, b = (torch.randn(d, generator=g).to(dtype) for _ in range(2))
    dy = torch.randn(x.shape, generator=g).to(dtype)
    y, dx, ds, mean, rstd = _run(cuda, x, w, b, dy)
    assert torch.equal(mean, values.double())
    assert torch.equal(y, b.double().expand_as(y))
    assert (ds == 0).all()
    assert ((rstd * EPS ** 0.5 - 1).abs() < 1e-5).all()


@pytest.mark.gpu
@pytest.mark.parametrize("offset", [100.0, 1e4, 1e5])
@pytest.mark.parametrize("d", WIDTHS)
def test_rows_far_from_zero(cuda, d, offset):
    g = torch.Generator().manual_seed(d + 1)
    rows = 50
    x = offset * (1 + torch.rand(rows, 1, generator=g)) + torch.randn(rows, d, generator=g)
    w, b = 1 + 0.2 * torch.randn(d, generator=g), 0.2 * torch.randn(d, generator=g)
    dy = torch.randn(rows, d, generator=g)
    y, dx, ds, mean, rstd = _run(cuda, x, w, b, dy)
    xd, wd, dyd = x.double(), w.double(), dy.double()
    m = xd.mean(1, keepdim=True)
    r = ((xd - m).square().mean(1, keepdim=True) + EPS).rsqrt()
    hat = (xd - m) * r
    err = (2.0 ** -24 * xd.abs().amax(1, keepdim=True) * r + W) * (1 + hat.abs())
    assert ((mean - m[:, 0]).abs() <= 2.0 ** -24 * m[:, 0].abs()).all()
    assert ((rstd / r[:, 0] - 1).abs() <= err.amax(1)).all()
    assert ((y - (hat * wd + b.double())).abs() <= err * wd.abs() + W * b.double().abs()).all()
    dn = dyd * wd
    want = r * (dn - dn.mean(1, keepdim=True) - hat * (dn * hat).mean(1, keepdim=True))
    size = r * dn.abs().amax(1, keepdim=True) * (1 + hat.abs())
    assert ((dx - want).abs() <= 4 * err * size).all()
    off = (dyd.abs() * err).sum(0) + 64 * 2.0 ** -24 * (dyd * hat).abs().sum(0)
    assert ((ds - (dyd * hat).sum(0)).abs() <= off).all()
