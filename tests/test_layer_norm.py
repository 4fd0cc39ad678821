"""Layer norm forward and backward against the formulas in 64 bits.

Tolerances. fp32 sums here chain at most 32 (a lane's columns) + 5 (a warp) + 16
(a row's warps) roundings, so a row sum is off by at most U = 64 * 2^-24 times
the sum of its terms' magnitudes. With X = max |x| and s = rstd this bounds the
mean's error by U X, hence hat's by U (X s) (1 + |hat|) and more terms of that
size; 8 U covers their number. A stored bf16 (8 significant bits) adds half a unit,
at most 2^-8 of the value.
Column sums chain at most rows / warps + 8 + blocks / 16 + 16 < 512 roundings at
the sizes below.
"""

import pytest
import torch

from rig_b200 import _lib, nn, ops

U = 64 * 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
EPS = 1e-5


def _inputs(rows, d, dtype, seed=0, offset=0.5):
    g = torch.Generator().manual_seed(seed)
    x = (1.5 * torch.randn(rows, d, generator=g) + offset * torch.randn(rows, 1, generator=g)).to(dtype)
    w = (1 + 0.2 * torch.randn(d, generator=g)).to(dtype)
    b = (0.2 * torch.randn(d, generator=g)).to(dtype)
    dy = torch.randn(rows, d, generator=g).to(dtype)
    res = torch.randn(rows, d, generator=g).to(dtype)
    return x, w, b, dy, res


def _formula(x, w, b, dy, res, eps=EPS):
    x, w, dy = x.double(), w.double(), dy.double()
    mean = x.mean(1, keepdim=True)
    rstd = ((x - mean).square().mean(1, keepdim=True) + eps).rsqrt()
    hat = (x - mean) * rstd
    y = hat * w + (0 if b is None else b.double())
    dn = dy * w
    dx = rstd * (dn - dn.mean(1, keepdim=True) - hat * (dn * hat).mean(1, keepdim=True))
    if res is not None:
        dx = dx + res.double()
    return dict(y=y, mean=mean[:, 0], rstd=rstd[:, 0], dx=dx, dscale=(dy * hat).sum(0),
                dbias=dy.sum(0), cols=dx.sum(0), hat=hat, dn=dn, xs=x.abs().amax(1, keepdim=True) * rstd)


def _check(got, want, x, w, b, dy, dtype, res):
    """Elementwise bounds of the module's docstring."""

    hat_err = 8 * U * (1 + want["xs"]) * (1 + want["hat"].abs())
    tol_y = hat_err * w.double().abs() + HALF[dtype] * want["y"].abs() + U * (0 if b is None else b.double().abs())
    assert ((got["y"].double() - want["y"]).abs() <= tol_y).all()
    scale = want["rstd"][:, None]
    size = want["dn"].abs().amax(1, keepdim=True) * (1 + want["hat"].abs()).amax(1, keepdim=True)
    dx_err = 8 * U * (1 + want["xs"]) * scale * size * (1 + want["hat"].abs())
    tol_dx = dx_err + HALF[dtype] * want["dx"].abs() + 2 * U * (0 if res is None else res.double().abs())
    assert ((got["dx"].double() - want["dx"]).abs() <= tol_dx).all()
    chain = 512 * 2.0 ** -24
    ds_tol = (chain * (dy.double() * want["hat"]).abs() + dy.double().abs() * hat_err).sum(0)
    assert ((got["dscale"].double() - want["dscale"]).abs() <= ds_tol).all()
    if got["dbias"] is not None:
        assert ((got["dbias"].double() - want["dbias"]).abs() <= chain * dy.double().abs().sum(0)).all()
    if got["cols"] is not None:
        tol = (chain * want["dx"].abs() + dx_err + 2 * U * (0 if res is None else res.double().abs())).sum(0)
        assert ((got["cols"].double() - want["cols"]).abs() <= tol).all()


def _run(dev, x, w, b, dy, res, cols=True, dbias=True):
    x, w, b, dy, res = (None if t is None else t.to(dev) for t in (x, w, b, dy, res))
    n, d = x.shape
    y = torch.empty_like(x)
    mean, rstd = torch.empty(2, n, device=dev).unbind()
    ops.layer_norm_fwd(x, w, b, y, mean, rstd, EPS)
    ds, db, dc = torch.zeros(3, d, device=dev).unbind()
    dx = torch.empty_like(x)
    ops.layer_norm_bwd(x, w, mean, rstd, dy, res, dx, ds, db if dbias else None, dc if cols else None)
    torch.cuda.synchronize()
    out = dict(y=y, dx=dx, dscale=ds, dbias=db if dbias else None, cols=dc if cols else None,
               mean=mean, rstd=rstd)
    return {k: None if t is None else t.cpu() for k, t in out.items()}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,d", [(1, 1), (2, 8), (3, 40), (33, 256), (700, 771), (1000, 768),
                                    (300, 1024), (65, 1032), (64, 2048), (37, 4104), (19, 4097),
                                    (7, 16384), (5, 16383)])
def test_formula(cuda, rows, d, dtype):
    for residual, bias, cols, dbias in [(True, True, True, True), (False, False, False, False),
                                        (True, True, False, True), (False, True, True, True)]:
        x, w, b, dy, res = _inputs(rows, d, dtype)
        b, res = b if bias else None, res if residual else None
        got = _run(cuda, x, w, b, dy, res, cols, dbias)
        _check(got, _formula(x, w, b, dy, res), x, w, b, dy, dtype, res)


@pytest.mark.gpu
def test_many_rows_accumulate(cuda):
    """Every block walks several rows; the sums add to what is there."""

    x, w, b, dy, res = _inputs(20001, 256, torch.bfloat16, seed=3)
    want = _formula(x, w, b, dy, res)
    _check(_run(cuda, x, w, b, dy, res), want, x, w, b, dy, torch.bfloat16, res)
    xd, wd, dyd = x.to(cuda), w.to(cuda), dy.to(cuda)
    mean, rstd = want["mean"].float().to(cuda), want["rstd"].float().to(cuda)
    once, twice = (torch.zeros(3, 256, device=cuda) for _ in range(2))
    dx = torch.empty_like(xd)
    ops.layer_norm_bwd(xd, wd, mean, rstd, dyd, None, dx, *once, colsum_alpha=0.25)
    for _ in range(2):
        ops.layer_norm_bwd(xd, wd, mean, rstd, dyd, None, dx, *twice, colsum_alpha=0.25)
    assert torch.equal(twice, once + once)  # fixed order: the second call adds the same bits


# For every split of a row over lanes and warps, more rows than six turns of a full
# grid take, and a last turn that is not full: rows in flight wrap around.
TURNS = [(14301, 512), (11003, 768), (7201, 1024), (3601, 2048), (1801, 4096), (903, 8192), (701, 8200),
         (14301, 129), (3603, 771), (1803, 1999), (901, 4095), (703, 6001), (451, 8193)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,d", TURNS)
def test_many_turns_at_every_split(cuda, rows, d, dtype):
    x, w, b, dy, res = _inputs(rows, d, dtype, seed=13)
    for residual in (True, False):
        r = res if residual else None
        _check(_run(cuda, x, w, b, dy, r, cols=residual), _formula(x, w, b, dy, r), x, w, b, dy, dtype, r)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_far_from_zero_and_constant_rows(cuda, dtype):
    """A large common offset does not cancel in the variance; a constant row has
    zero variance and gives the bias."""

    x, w, b, dy, res = _inputs(40, 512, dtype, seed=5, offset=100.0)
    x[7] = 3.0
    got, want = _run(cuda, x, w, b, dy, res), _formula(x, w, b, dy, res)
    _check(got, want, x, w, b, dy, dtype, res)
    assert torch.equal(got["y"][7], b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides_and_alignment(cuda, dtype):
    """Column slices of wider buffers (vector and element paths), a residual
    gradient updated in place, equal to contiguous copies."""

    rows, d = 50, 264
    for start in (0, 8, 3):
        wide = [t.to(cuda) for t in _inputs(rows, d + 24, dtype, seed=7)]
        x, dy, res = (wide[i][:, start:start + d] for i in (0, 3, 4))
        w, b = wide[1][:d].contiguous(), wide[2][:d].contiguous()
        a = _run(cuda, x.contiguous(), w, b, dy.contiguous(), res.contiguous())
        y = torch.full((rows, d + 16), 7.0, dtype=dtype, device=cuda)
        mean, rstd = torch.empty(2, rows, device=cuda).unbind()
        ops.layer_norm_fwd(x, w, b, y[:, 8:8 + d], mean, rstd)
        ds, db, dc = torch.zeros(3, d, device=cuda).unbind()
        buf = wide[4].clone()
        inout = buf[:, start:start + d]
        ops.layer_norm_bwd(x, w, mean, rstd, dy, inout, inout, ds, db, dc)
        want = _formula(x.cpu(), w.cpu(), b.cpu(), dy.cpu(), res.cpu())
        got = dict(y=y[:, 8:8 + d].cpu(), dx=inout.cpu(), dscale=ds.cpu(), dbias=db.cpu(), cols=dc.cpu())
        _check(got, want, x.cpu(), w.cpu(), b.cpu(), dy.cpu(), dtype, res.cpu())
        if start != 3:  # the same path: the same bits
            assert torch.equal(got["y"], a["y"]) and torch.equal(got["dx"], a["dx"])
        assert (y[:, :8] == 7).all() and (y[:, 8 + d:] == 7).all()
        assert torch.equal(buf[:, :start], wide[4][:, :start])
        assert torch.equal(buf[:, start + d:], wide[4][:, start + d:])


@pytest.mark.gpu
def test_non_finite_rows_stay_in_their_rows(cuda):
    x, w, b, dy, res = _inputs(20, 256, torch.float32, seed=9)
    clean = _run(cuda, x, w, b, dy, res)
    x[4, 17] = float("inf")
    x[5, 0] = float("nan")
    got = _run(cuda, x, w, b, dy, res)
    keep = [r for r in range(20) if r not in (4, 5)]
    assert torch.equal(got["y"][keep], clean["y"][keep]) and torch.equal(got["dx"][keep], clean["dx"][keep])
    assert got["y"][4].isnan().any() and got["y"][5].isnan().all()


@pytest.mark.gpu
def test_gradients_against_differences(cuda):
    """Central differences of the kernel's own forward in fp32 along random
    directions. L = sum(y * dy) is summed in 64 bits. With a step h = 2^-6 the
    truncation is h^2/6 L''' (|L'''| is at most a few |dL|, as rstd ~ 2/3), under
    1e-3, and the rounding of y, 2^-24 sqrt(n) / h ~ 1e-4, is far below |dL| ~
    sqrt(n)."""

    g = torch.Generator().manual_seed(1)
    x, w, b, dy = (t.to(cuda) for t in _inputs(16, 200, torch.float32, seed=11)[:4])
    args = [t.clone().requires_grad_(True) for t in (x, w, b)]
    nn.layer_norm(*args).backward(dy)
    h = 2.0 ** -6
    for i, a in enumerate(args):
        u = torch.randn(a.shape, generator=g).to(cuda)
        sides = []
        for s in (h, -h):
            moved = [t.detach() + (s * u if j == i else 0) for j, t in enumerate(args)]
            sides.append((nn.layer_norm(*moved).double() * dy.double()).sum().item())
        slope = (sides[0] - sides[1]) / (2 * h)
        want = (a.grad.double() * u.double()).sum().item()
        size = (a.grad.double().norm() * u.double().norm() / a.numel() ** 0.5).item()
        assert abs(slope - want) <= 2e-3 * max(size, abs(want)), (i, slope, want)


@pytest.mark.gpu
def test_autograd_wrapper(cuda):
    """[B, T, d] bf16 input with fp32 parameters, and another stream than the default."""

    x, w, b, dy, _ = _inputs(60, 320, torch.bfloat16, seed=13)
    want = _formula(x, w.float().bfloat16(), b.float().bfloat16(), dy, None)
    xg = x.to(cuda).view(4, 15, 320).requires_grad_(True)
    wg, bg = w.float().to(cuda).requires_grad_(True), b.float().to(cuda).requires_grad_(True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = nn.layer_norm(xg, wg, bg)
        y.backward(dy.to(cuda).view_as(y))
    side.synchronize()
    got = dict(y=y.detach().view(60, 320).cpu(), dx=xg.grad.view(60, 320).cpu(), dscale=wg.grad.cpu(),
               dbias=bg.grad.cpu(), cols=None)
    assert wg.grad.dtype == torch.float32 and y.shape == (4, 15, 320)
    _check(got, want, x, w, b, dy, torch.bfloat16, None)


@pytest.mark.gpu
def test_refusals(cuda):
    x, w, b, dy, res = (t.to(cuda) for t in _inputs(4, 64, torch.bfloat16))
    y, stat = torch.empty_like(x), torch.empty(4, device=cuda)
    with pytest.raises(TypeError):
        ops.layer_norm_fwd(x.half(), w.half(), None, y.half(), stat, stat)
    with pytest.raises(ValueError):
        ops.layer_norm_fwd(x, w.float(), None, y, stat, stat)  # parameters in another dtype
    with pytest.raises(ValueError):
        ops.layer_norm_fwd(x, w[:32], None, y, stat, stat)
    with pytest.raises(ValueError):
        ops.layer_norm_fwd(x, w, None, y.t().contiguous().t(), stat, stat)
    with pytest.raises(ValueError):
        ops.layer_norm_fwd(x, w, None, y, stat.double(), stat)
    with pytest.raises(ValueError):
        ops.layer_norm_bwd(x, w, stat, stat, dy, res, y, stat)  # dscale of the wrong size
    with pytest.raises(ValueError):
        ops.layer_norm_bwd(x, w, stat, stat, dy, res, y, torch.zeros(64, device=cuda),
                           workspace=torch.empty(16, dtype=torch.uint8, device=cuda))
    with pytest.raises(_lib.GptB200Error):
        ops.layer_norm_fwd(x[:0], w, None, y[:0], stat[:0], stat[:0])
    wide = torch.empty(2, 16385, device=cuda)
    with pytest.raises(_lib.GptB200Error):
        ops.layer_norm_fwd(wide, wide[0], None, torch.empty_like(wide), stat[:2], stat[:2])
    with pytest.raises(TypeError):
        nn.layer_norm(x.half(), w)


def test_cpu_tensors_and_bad_arguments_are_refused():
    x, w, b, dy, _ = _inputs(2, 8, torch.float32)
    with pytest.raises(ValueError):
        ops.layer_norm_fwd(x, w, b, torch.empty_like(x), torch.empty(2), torch.empty(2))
    lib = _lib.load()
    one = 16  # a non-null address: every case below is refused before it is used
    assert lib.gptb200_layer_norm_fwd(None, one, None, one, one, one, 1, 8, 8, 8, 1e-5, 0, None) == 1
    assert lib.gptb200_layer_norm_fwd(one, one, None, one, one, one, 0, 8, 8, 8, 1e-5, 0, None) == 1
    assert lib.gptb200_layer_norm_fwd(one, one, None, one, one, one, 1, 8, 8, 8, float("nan"), 0, None) == 1
    assert lib.gptb200_layer_norm_fwd(one, one, None, one, one, one, 1, 8, 7, 8, 1e-5, 0, None) == 2
    assert lib.gptb200_layer_norm_fwd(one, one, None, one, one, one, 1, 8, 8, 8, 1e-5, 5, None) == 3
    assert lib.gptb200_layer_norm_fwd(one, one, None, one, one, one, 1, 1 << 20, 1 << 20, 1 << 20, 1e-5,
                                      0, None) == 2
    assert lib.gptb200_layer_norm_bwd_workspace_size(0, 8) == 0
    assert lib.gptb200_layer_norm_bwd(one, one, one, one, one, None, one, one, None, None, 1.0, 1, 8, 8,
                                      8, 8, 0, None, None) == 1
