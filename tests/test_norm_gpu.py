"""The residual update with its norms (moearc_norm_residual) against float64.

Bounds, u = 2^-24: a sum of squares goes over at most 64 terms in one thread and 14 additions across
threads, all positive, so it is within 78 u, its root within 39 u; with the mean, eps, root and
reciprocal 45 u. z takes three more roundings, h two. x's own root sees h's error."""
from __future__ import annotations

import numpy as np
import pytest

import fixtures as fx
from moearc_amd import OUT_F16, OUT_F32, DeviceView

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _np(io):
    return np.float16 if io == OUT_F16 else np.float32


def _reference(h, y, w_post, gate, scale, w_pre, eps):
    """(h, bound of h, x, bound of x before x's own rounding) in float64."""
    h = h.astype(np.float64)
    eh = np.zeros_like(h)
    if y is not None:
        z = y.astype(np.float64)
        if w_post is not None:
            z = z / np.sqrt((z * z).mean(1, keepdims=True) + eps) * w_post
        if gate is not None:
            z = z * gate
        h = h + scale * z
        eh = 50 * U * np.abs(scale * z) + U * np.abs(h)
    ms = (h * h).mean(1, keepdims=True)
    r = 1 / np.sqrt(ms + eps)
    w = 1.0 if w_pre is None else w_pre.astype(np.float64)
    x = h * r * w
    # the root of a mean of squares moves by at most the root mean square of the changes
    moved = np.sqrt((eh * eh).mean(1, keepdims=True)) * r
    return h, eh, x, np.abs(x) * (50 * U + moved) + eh * r * np.abs(w)


def _run(ctx, rows, cols, y_type=OUT_F32, x_type=OUT_F32, post=True, gate="row", pre=True, scale=0.5, eps=1e-5,
         seed=0x2021, shift=0, with_y=True, with_x=True, size=1.0):
    """Buffers start `shift` bytes past an aligned address."""
    def draw(i, *shape):
        return fx.synth.normal(seed + i, int(np.prod(shape))).reshape(shape)
    h = draw(0, rows, cols) * np.float32(size)
    y = draw(1, rows, cols).astype(_np(y_type)) if with_y else None
    wp = 1 + draw(2, cols) * np.float32(0.2) if post and with_y else None
    wq = 1 + draw(3, cols) * np.float32(0.2) if pre and with_x else None
    stride = {"none": 0, "shared": 0, "row": cols + 4 if cols % 4 == 0 else cols + 3}[gate]
    g = None
    if gate != "none" and with_y:
        g = draw(4, rows, stride)[:, :] if stride else draw(4, 1, cols)
    keep = []

    def up(a):
        if a is None:
            return None
        raw = np.concatenate([np.zeros(shift, np.uint8), np.ascontiguousarray(a).view(np.uint8).reshape(-1)])
        keep.append(ctx.upload(raw))
        return DeviceView(keep[-1], shift)
    bh, by, bp, bq, bg = (up(a) for a in (h, y, wp, wq, g))
    bx = up(np.full((rows, cols), -7, _np(x_type))) if with_x else None
    ctx.norm_residual(bx, bh, by, bp, bg, stride, scale, bq, rows, cols, eps, x_type, y_type)
    eh = _reference(h, y, wp, None if g is None else g[:, :cols].astype(np.float64), np.float64(np.float32(scale)), wq, eps)
    got_h = ctx.download(bh, np.float32, (rows, cols))
    if with_y:
        assert bool(np.all(np.abs(got_h - eh[0]) <= eh[1]))
    else:
        assert np.array_equal(got_h, h)
    if with_x:
        got = ctx.download(bx, _np(x_type), (rows, cols)).astype(np.float64)
        # f16: half a step, 2^-11 of the value, or half the smallest subnormal
        tol = eh[3] + (2.0 ** -11 * np.abs(eh[2]) * (1 + 2.0 ** -10) + 2.0 ** -25 if x_type == OUT_F16 else 0)
        assert bool(np.all(np.abs(got - eh[2]) <= tol + 1e-30))
    return got_h


@pytest.mark.parametrize("cols", [1, 3, 16, 64, 100, 128, 255, 256, 257, 1024, 1028, 2880, 4096, 4100, 5001, 16384,
                                  16385, 40000])
def test_each_row_length(ctx, cols):
    for rows in (1, 5, 33):
        _run(ctx, rows, cols)


@pytest.mark.parametrize("cols", [128, 2880, 20000])
@pytest.mark.parametrize("y_type,x_type", [(0, 0), (0, 1), (1, 0), (1, 1)])
@pytest.mark.parametrize("post,gate,pre", [(True, "none", True), (False, "shared", True), (True, "shared", False),
                                           (False, "none", False), (True, "row", True)])
def test_each_part_and_type(ctx, cols, y_type, x_type, post, gate, pre):
    _run(ctx, 7, cols, y_type, x_type, post, gate, pre, scale=-1.25)


@pytest.mark.parametrize("cols", [64, 2880, 4099, 17000])
def test_plain_norm_and_update_alone(ctx, cols):
    _run(ctx, 9, cols, with_y=False)
    _run(ctx, 9, cols, with_y=False, x_type=OUT_F16)
    _run(ctx, 9, cols, with_x=False)


@pytest.mark.parametrize("shift", [4, 8, 12])
def test_unaligned_buffers(ctx, shift):
    _run(ctx, 5, 2880, shift=shift)
    _run(ctx, 5, 2880, shift=shift, x_type=OUT_F16, y_type=OUT_F16)


def test_many_short_rows(ctx):
    _run(ctx, 70001, 64, with_y=False)


def test_large_and_small_values(ctx):
    _run(ctx, 3, 2880, size=1e15)
    _run(ctx, 3, 2880, size=1e-18, scale=0.0)
    h = np.zeros((2, 96), np.float32)
    bh, bx = ctx.upload(h), ctx.upload(h + 1)
    ctx.norm_residual(bx, bh, None, None, None, 0, 1.0, None, 2, 96, 1e-6)
    assert np.array_equal(ctx.download(bx, np.float32, (2, 96)), h)  # a row of zeros stays one


def test_nan_and_inf_stay_in_their_row(ctx):
    for cols in (64, 2880):
        h = fx.synth.normal(5, 4 * cols).reshape(4, cols)
        want = h.copy()
        h[1, 3], h[2, 5] = np.nan, np.inf
        bh, bx = ctx.upload(h), ctx.alloc(h.nbytes)
        ctx.norm_residual(bx, bh, None, None, None, 0, 1.0, None, 4, cols, 1e-6)
        got = ctx.download(bx, np.float32, (4, cols))
        assert np.isnan(got[1]).all() and np.isnan(got[2, 5]) and np.all(got[2][np.arange(cols) != 5] == 0)
        for r in (0, 3):
            x = want[r] / np.sqrt((want[r].astype(np.float64) ** 2).mean() + 1e-6)
            assert np.all(np.abs(got[r] - x) <= 50 * U * np.abs(x))


@pytest.mark.parametrize("cols", [128, 2880, 20000])
def test_x_over_y(ctx, cols):
    for io in (OUT_F32, OUT_F16):
        h, y = fx.synth.normal(8, 6 * cols).reshape(6, cols), fx.synth.normal(9, 6 * cols).reshape(6, cols).astype(_np(io))
        w = 1 + fx.synth.normal(10, cols) * np.float32(0.1)
        bh, bh2, by, bx, bw = ctx.upload(h), ctx.upload(h), ctx.upload(y), ctx.alloc(y.nbytes), ctx.upload(w)
        ctx.norm_residual(bx, bh, by, bw, None, 0, 0.7, bw, 6, cols, 1e-5, io, io)
        ctx.norm_residual(by, bh2, by, bw, None, 0, 0.7, bw, 6, cols, 1e-5, io, io)
        for a, b, t in ((bx, by, _np(io)), (bh, bh2, np.float32)):
            assert np.array_equal(ctx.download(a, t, (6, cols)), ctx.download(b, t, (6, cols)))


def test_nothing_around_the_rows_is_written(ctx):
    for cols in (60, 100, 2880, 4099):
        n, pad = 3 * cols, 64
        raw = np.full(n + 2 * pad, 3.5, np.float32)
        bh, bx = ctx.upload(raw), ctx.upload(raw)
        by = ctx.upload(np.ones(n, np.float32))
        ctx.norm_residual(DeviceView(bx, 4 * pad, 4 * n), DeviceView(bh, 4 * pad, 4 * n), by, None, None, 0, 1.0, None, 3, cols, 1e-5)
        for b in (bh, bx):
            got = ctx.download(b, np.float32, (n + 2 * pad,))
            assert np.all(got[:pad] == 3.5) and np.all(got[-pad:] == 3.5) and not np.any(got[pad:-pad] == 3.5)
