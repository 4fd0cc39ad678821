"""AdamW with 8-bit moments against a numpy restatement of its definition.

Up to the codes every operation is rounded to fp32 by itself, so the restatement
(separate numpy float32 operations) has to give the same codes bit for bit. The
parameter update may contract a product and a sum and divide with the device's
correctly rounded division: p' = p - lr (adam + wd p) is off by at most a few
2^-24 of |p| + lr (|adam| + wd |p|).
"""

import ctypes

import numpy as np
import pytest
import torch

from rig_b200 import _lib, ops

f4 = np.float32
BLOCK = 64


def _config(**kw):
    base = dict(learning_rate=1e-2, horizon_lr_scale=1.0, min_lr_ratio=0.1, warmup_steps=0,
                total_steps=1000, beta1=0.9, beta2=0.95, eps=1e-8, eps_horizon_scale=1.0,
                weight_decay=0.1, wd_horizon_scale=1.0, grad_clip=0.0, grad_scale=1.0)
    return _lib.AdamWConfig(**{**base, **kw})


def _mix32(h):
    h = np.asarray(h, np.uint64)
    m = np.uint64(0xFFFFFFFF)
    h = ((h ^ (h >> np.uint64(16))) * np.uint64(0x85EBCA6B)) & m
    h = ((h ^ (h >> np.uint64(13))) * np.uint64(0xC2B2AE35)) & m
    return h ^ (h >> np.uint64(16))


def _dither(n, seed, step):
    key = _mix32(_mix32(step) ^ np.uint64(seed))
    i = np.arange(n, dtype=np.uint64)
    return _mix32((i * np.uint64(0x9E3779B1) + key) & np.uint64(0xFFFFFFFF)).astype(np.int64)


def _decode(code, exp, mant):
    """Value of a code by the format's definition, in 64 bits."""

    code, e = code.astype(np.int64), np.repeat(exp.astype(np.int64), BLOCK)
    v = np.ldexp(1 + (code % (1 << mant)) / (1 << mant), e - 142 + (code >> mant))
    v = np.where(code == 0, 0.0, v)
    return np.where(e == 255, np.nan, v)


def _encode(x, dither, mant, flush):
    """Codes of |x| (float32, whole blocks) by arithmetic on values: the exponent
    window from the block's largest, then floor(x / unit + u)."""

    a = np.abs(x.astype(np.float64)).reshape(-1, BLOCK)
    u = (dither / (1 << (23 - mant))).reshape(-1, BLOCK)
    top = a.max(1, keepdims=True)
    frac, e = np.frexp(top)  # top = frac 2^e, frac in [.5, 1)
    E = e - 1 + 127 + (2 * frac > 2 - 2.0 ** -mant)
    E = np.maximum(np.where(top == 0, 16, E), 16)
    _, e = np.frexp(a)
    e = np.where(a == 0, -1000, e - 1)
    unit = np.ldexp(1.0, e - mant)
    up = np.floor(a / unit + u) * unit  # may reach the next power of two
    frac, e = np.frexp(up)
    code = ((e - 1) - (E - 142)) * (1 << mant) + np.floor((2 * frac - 1) * (1 << mant))
    code = np.where(a == 0, 0, np.maximum(code, 0 if flush else 1)).astype(np.int64)
    return code.reshape(-1), E.reshape(-1).astype(np.int64)


class Restatement:
    """One flat state, float32 operation by operation."""

    def __init__(self, n, tensors):
        self.n, self.pad = n, -n % BLOCK
        nb = (n + self.pad) // BLOCK
        self.m, self.v = np.zeros(n + self.pad, np.int64), np.zeros(n + self.pad, np.int64)
        self.me, self.ve = np.zeros(nb, np.int64), np.zeros(nb, np.int64)
        self.live = np.zeros(n + self.pad, bool)
        self.mult = np.zeros((4, n + self.pad), f4)
        for off, size, *mult in tensors:
            self.live[off:off + size] = True
            self.mult[:, off:off + size] = np.array(mult, f4)[:, None]

    def step(self, p, g, c, t, seed, gscale=f4(1)):
        p, g = (np.pad(a.astype(f4), (0, self.pad)) for a in (p, g))
        g = np.where(self.live, g, f4(0)) * f4(gscale)
        b1, b2 = f4(c.beta1), f4(c.beta2)
        mag = _decode(self.m & 127, self.me, 3).astype(f4)
        r = _decode(self.v, self.ve, 4).astype(f4)
        m = b1 * np.where(self.m & 128, -mag, mag) + (f4(1) - b1) * g
        r = np.sqrt(b2 * (r * r) + (f4(1) - b2) * (g * g))
        m, r = np.where(self.live, m, f4(0)), np.where(self.live, r, f4(0))
        warm = min(1.0, t / c.warmup_steps) if c.warmup_steps else 1.0
        along = min(max((t - c.warmup_steps) / max(1, c.total_steps - c.warmup_steps), 0.0), 1.0)
        lr = c.learning_rate * warm * (c.min_lr_ratio + (1 - c.min_lr_ratio) * .5 * (1 + np.cos(np.pi * along)))
        mult = self.mult.astype(np.float64)
        adam = m / (1 - float(b1) ** t) / (r / np.sqrt(1 - float(b2) ** t) + c.eps * mult[1] + (~self.live))
        wd = c.weight_decay * mult[2] * mult[3]
        new = p - lr * mult[0] * (adam + wd * p)
        tol = 2.0 ** -20 * (np.abs(p) + lr * mult[0] * (np.abs(adam) + wd * np.abs(p)))
        h = _dither(self.n + self.pad, seed, t)
        code, E = _encode(m, (h >> 16) << 4, 3, True)
        code = code + 128 * ((m < 0) & (code > 0))
        code_v, Ev = _encode(r, (h & 0xFFFF) << 3, 4, False)
        seen = self.live.reshape(-1, BLOCK).any(1)  # blocks of padding alone are not touched
        self.m, self.v = np.where(self.live, code, self.m), np.where(self.live, code_v, self.v)
        self.me, self.ve = np.where(seen, E, self.me), np.where(seen, Ev, self.ve)
        keep = slice(0, self.n)
        return np.where(self.live, new, p)[keep], tol[keep]


def _groups(tensors, dev):
    arr = (_lib.TensorGroup * len(tensors))(*(_lib.TensorGroup(*t) for t in tensors))
    return torch.frombuffer(bytearray(bytes(arr)), dtype=torch.uint8).to(dev)


# (offset, size, lr, eps, decay multipliers, decays): sizes that end inside a block, a
# quad and a lane; padding between tensors; offsets that are multiples of 4 only
LAYOUTS = {
    "one_element": [(0, 1, 1.0, 1.0, 1.0, 1)],
    "padded": [(0, 1000, 1.0, 0.5, 2.0, 1), (1024, 64, 2.0, 1.0, 1.0, 0), (1088, 3, 1.0, 1.0, 1.0, 0),
               (1152, 5000, 0.5, 1.0, 1.0, 1)],
    "packed": [(0, 70, 1.0, 1.0, 1.0, 1), (72, 129, 0.5, 2.0, 1.0, 0), (204, 40, 1.0, 1.0, 1.0, 1)],
    "whole_empty_blocks": [(0, 10, 1.0, 1.0, 1.0, 1), (640, 10, 1.0, 1.0, 1.0, 1)],
    "large": [(64 * 5000 * i, 64 * 5000 - 7 * i, 1.0, 1.0, 1.0, i % 2) for i in range(9)],
}


def _run(dev, tensors, n, cfg, grads, p0, seed=5):
    dv = {k: torch.zeros(1, dtype=torch.int32, device=dev) for k in ("step",)}
    p = torch.from_numpy(p0.copy()).to(dev)
    state = ops.adamw8_state(n, dev)
    mirror = torch.full((n,), 9.0, dtype=torch.bfloat16, device=dev)
    loss, history = torch.ones(1, device=dev), torch.zeros(cfg.total_steps, 3, device=dev)
    ws, table = ops.adamw_workspace(n, dev), _groups(tensors, dev)
    for g in grads:
        ops.adamw8_step(p, state, torch.from_numpy(g).to(dev), table, len(tensors), cfg, dv["step"],
                        loss, history, mirror, seed, ws)
        yield p.cpu().numpy(), [t.cpu().numpy() for t in state], mirror.cpu(), history.cpu().numpy(), state


def _draw(n, live, seed, steps):
    rng = np.random.default_rng(seed)
    spread = np.exp(2 * rng.standard_normal(n))  # elements of a block differ by powers of ten
    out = [(rng.standard_normal(n) * spread * 1e-3).astype(f4) for _ in range(steps)]
    return [np.where(live, g, f4(0)) for g in out], np.where(live, rng.standard_normal(n) * .05, 0).astype(f4)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", LAYOUTS)
def test_codes_and_parameters_match_restatement(cuda, layout):
    tensors = LAYOUTS[layout]
    n = tensors[-1][0] + tensors[-1][1]
    ref = Restatement(n, tensors)
    grads, p0 = _draw(n, ref.live[:n], 1, 4)
    cfg = _config(warmup_steps=3)
    p = p0
    for t, got in enumerate(_run(cuda, tensors, n, cfg, grads, p0), 1):
        want, tol = ref.step(p, grads[t - 1], cfg, t, 5)
        p, (m, me, v, ve), mirror, history, state = got
        assert np.array_equal(m, ref.m) and np.array_equal(v, ref.v)
        assert np.array_equal(me, ref.me) and np.array_equal(ve, ref.ve)
        assert (np.abs(p - want) <= tol).all()
        live = ref.live[:n]
        assert torch.equal(mirror[live], torch.from_numpy(p)[live].bfloat16())
        assert (p[~live] == p0[~live]).all() and (mirror[~live] == 9).all()
        norm = np.linalg.norm(grads[t - 1].astype(np.float64))
        np.testing.assert_allclose(history[t - 1, 2], norm, rtol=1e-6)
        mv, rv = ops.adamw8_values(state)
        sign = np.where(m & 128, -1.0, 1.0)
        assert np.array_equal(mv.cpu().double().numpy(), sign * _decode(m & 127, me, 3))
        assert np.array_equal(rv.cpu().double().numpy(), _decode(v, ve, 4))


@pytest.mark.gpu
def test_clipping_and_repeatability(cuda):
    """The clip factor min(1, c / (norm + 1e-6)); the same inputs give the same
    bits; another seed rounds differently but within one unit (2^-3, 2^-4)."""

    tensors, n = LAYOUTS["padded"], 6152
    ref = Restatement(n, tensors)
    grads, p0 = _draw(n, ref.live[:n], 2, 2)
    norm = float(np.linalg.norm(grads[0].astype(np.float64)))
    cfg = _config(grad_clip=norm / 3)
    a, b, c = ([g[:2] + (ops.adamw8_values(g[4])[0].cpu().double(),) for g in
                _run(cuda, tensors, n, cfg, grads, p0, seed)] for seed in (5, 5, 6))
    assert np.array_equal(a[1][0], b[1][0]) and all(np.array_equal(x, y) for x, y in zip(a[1][1], b[1][1]))
    clip = cfg.grad_clip / (norm + 1e-6)
    want, tol = ref.step(p0, grads[0], cfg, 1, 5, clip)
    assert (np.abs(a[0][0] - want) <= tol + 2.0 ** -20 * np.abs(want - p0)).all()
    # fp32 norms may differ in the last bit: the codes then agree but for rare cuts
    assert (a[0][1][0] != ref.m).mean() < 1e-3 and (a[0][1][2] != ref.v).mean() < 1e-3
    diff = (a[0][2] - c[0][2]).abs()
    assert diff.max() > 0
    assert (diff <= torch.maximum(a[0][2].abs(), c[0][2].abs()) / 8 + a[0][2].abs().max() * 2.0 ** -14).all()


@pytest.mark.gpu
def test_rounding_is_unbiased_and_v_can_fall(cuda):
    """64 seeds of one step from zero: the mean code value approaches (1 - beta1) g.
    One rounding takes one of two values a unit of at most 2^-3 |m| apart, so its
    deviation is at most half of that and the mean of 64 has at most 2^-3 / 2 / 8 =
    0.0078 |m|; 5 of those at 4,096 elements. And with no gradient r falls by sqrt(beta2) a step on average:
    over 40 steps v falls by 0.95^40 = 0.128, where rounding to nearest would hold it."""

    n, tensors = 4096, [(0, 4096, 1.0, 1.0, 1.0, 1)]
    rng = np.random.default_rng(3)
    g = np.exp(rng.uniform(np.log(1e-3), np.log(1e-1), n)).astype(f4)
    total = torch.zeros(n, dtype=torch.float64)
    cfg = _config()
    for seed in range(64):
        *_, last = _run(cuda, tensors, n, cfg, [g], np.zeros(n, f4), seed * 7919 + 1)
        total += ops.adamw8_values(last[4])[0].cpu().double()
    m = (f4(1) - f4(0.9)).astype(np.float64) * g
    assert (np.abs(total.numpy() / 64 - m) <= 5 * 0.0078 * m).all()
    zero = np.zeros(n, f4)
    *_, last = _run(cuda, tensors, n, cfg, [g] + [zero] * 40, np.zeros(n, f4))
    v = ops.adamw8_values(last[4])[1].cpu().double().square().numpy()
    # a rounding of r is unbiased with a relative variance of at most 2^-8 / 4 (one of two
    # neighbours a unit of 2^-4 apart), so E[v] grows by at most that factor a step beside
    # the 0.95: 40 steps, at most 1.04; the mean of 4,096 elements strays by 1% or so
    ratio = (v / (float(f4(1) - f4(0.95)) * g.astype(np.float64) ** 2)).mean()
    assert 0.95 ** 40 * 0.9 <= ratio <= 0.95 ** 40 * 1.2


@pytest.mark.gpu
def test_small_elements_of_a_block_stay_bounded(cuda):
    """One huge element per block: the others fall out of the window. Their m is 0
    or right to a unit and their r never below the truth, so no update is larger
    than the exact one by more than the rounding of r (2^-4) and m (2^-3)."""

    n, tensors = 640, [(0, 640, 1.0, 1.0, 1.0, 0)]
    g = np.full(n, 1e-7, f4)
    g[::64] = 1e4
    cfg = _config(weight_decay=0.0)
    p = None
    for got in _run(cuda, tensors, n, cfg, [g] * 6, np.zeros(n, f4)):
        step = got[0] - (0 if p is None else p)
        p = got[0]
        assert np.abs(step).max() <= 1e-2 * (1 + 2.0 ** -3 + 2.0 ** -4) * 1.02
    small = np.ones(n, bool)
    small[::64] = False
    assert ops.adamw8_values(got[4])[1].float().cpu().numpy()[small].min() > 0


@pytest.mark.gpu
def test_non_finite_gradients_are_kept_and_reported(cuda):
    n, tensors = 256, [(0, 256, 1.0, 1.0, 1.0, 1)]
    g = np.full(n, 1e-3, f4)
    g[70], g[140] = np.nan, np.inf
    ops.device_error()
    *_, last = _run(cuda, tensors, n, _config(), [g], np.zeros(n, f4))
    m, r = (t.float().cpu() for t in ops.adamw8_values(last[4]))
    assert m[64:192].isnan().all() and r[64:192].isnan().all()
    assert m[:64].isfinite().all() and m[192:].isfinite().all()
    assert np.isnan(last[0][70]) and np.isfinite(last[0][:64]).all()
    assert _lib.load().gptb200_device_error_flags(1) & _lib.DEVERR_NONFINITE


@pytest.mark.gpu
def test_ranges_equal_one_step(cuda):
    """begin / per-range updates / end give the codes and parameters of one call."""

    tensors = LAYOUTS["large"]
    n = (tensors[-1][0] + tensors[-1][1] + 63) // 64 * 64
    ref = Restatement(n, tensors)
    grads, p0 = _draw(n, ref.live[:n], 4, 1)
    cfg = _config()
    *_, whole = _run(cuda, tensors, n, cfg, grads, p0)
    p, g = torch.from_numpy(p0).to(cuda), torch.from_numpy(grads[0]).to(cuda)
    state, ws, table = ops.adamw8_state(n, cuda), ops.adamw_workspace(n, cuda), _groups(tensors, cuda)
    step = torch.zeros(1, dtype=torch.int32, device=cuda)
    loss, history = torch.ones(1, device=cuda), torch.zeros(10, 3, device=cuda)
    ops.adamw_begin(cfg, step, ws)
    cuts = [0, 64, 64 * 3001, 64 * 20000, n]
    for slot, (a, b) in enumerate(zip(cuts, cuts[1:])):
        ops.adamw8_update_range(p, state, g, a, b, table, len(tensors), cfg, slot, None, 5, ws)
    ops.adamw_end(len(cuts) - 1, cfg, step, loss, history, ws)
    assert np.array_equal(p.cpu().numpy(), whole[0])
    assert all(np.array_equal(t.cpu().numpy(), w) for t, w in zip(state, whole[1]))
    np.testing.assert_allclose(history[0].cpu(), whole[3][0], rtol=1e-6)


@pytest.mark.gpu
def test_refusals(cuda):
    n, cfg = 128, _config()
    p, g = torch.zeros(n, device=cuda), torch.zeros(n, device=cuda)
    state, ws = ops.adamw8_state(n, cuda), ops.adamw_workspace(n, cuda)
    table = _groups([(0, n, 1.0, 1.0, 1.0, 1)], cuda)
    step = torch.zeros(1, dtype=torch.int32, device=cuda)
    with pytest.raises(ValueError):
        ops.adamw8_step(p, ops.adamw8_state(64, cuda), g, table, 1, cfg, step, None, None, None, 0, ws)
    with pytest.raises(ValueError):
        ops.adamw8_step(p, state, g.bfloat16(), table, 1, cfg, step, None, None, None, 0, ws)
    with pytest.raises(ValueError):
        ops.adamw8_step(p, state, g, table, 1, cfg, step, None, None, p, 0, ws)
    with pytest.raises(_lib.GptB200Error):
        ops.adamw8_step(p, state, g, table, 0, cfg, step, None, None, None, 0, ws)
    with pytest.raises(_lib.GptB200Error):  # not whole blocks
        ops.adamw8_update_range(p, state, g, 0, 100, table, 1, cfg, 0, None, 0, ws)
    with pytest.raises(ValueError):
        ops.adamw8_update_range(p, state, g, 0, 192, table, 1, cfg, 0, None, 0, ws)
    with pytest.raises(_lib.GptB200Error):  # clipping needs the norm first
        ops.adamw8_update_range(p, state, g, 0, 128, table, 1, _config(grad_clip=1.0), 0, None, 0, ws)
    assert int(step) == 0


def test_cpu_and_null_arguments_are_refused():
    with pytest.raises(ValueError):
        ops.adamw8_values(ops.adamw8_state(64, "cpu"))
    lib, cfg = _lib.load(), _config()
    none = _lib.AdamW8State()
    assert lib.gptb200_adamw8_step(16, ctypes.byref(none), 16, 64, 16, 1, ctypes.byref(cfg), 16, None,
                                   None, None, 0, 16, None) == 1
    assert lib.gptb200_adamw8_values(ctypes.byref(none), 64, 16, 16, None) == 1
