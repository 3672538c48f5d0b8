"""The router (moearc_moe_route): ids exactly, weights against float64.

Bound of a weight, u = 2^-24: v - m rounds once (u |v - m| in the exponent), expf is within 2 ulp (4 u), the sums
take at most 64 + 4 terms of one sign, the quotient, the scale and the product 3 more."""
from __future__ import annotations

import numpy as np
import pytest

import fixtures as fx
from moearc_amd import RouteMode

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _route(ctx, logits, k, mode, scale=1.0):
    t, e = logits.shape
    bi, bw, bl = ctx.upload(np.full(t * k + 8, 77, np.uint32)), ctx.upload(np.full(t * k + 8, -7, np.float32)), ctx.upload(logits)
    ctx.moe_route(bi, bw, bl, t, e, k, mode, scale)
    ids, w = ctx.download(bi, np.uint32, (t * k + 8,)), ctx.download(bw, np.float32, (t * k + 8,))
    assert np.all(ids[-8:] == 77) and np.all(w[-8:] == -7)
    return ids[:-8].reshape(t, k), w[:-8].reshape(t, k)


def _check(ctx, logits, k, mode, scale=1.0):
    ids, w = _route(ctx, logits, k, mode, scale)
    v = np.where(np.isnan(logits), -np.inf, logits).astype(np.float64) + 0.0
    # NaN after every -inf, ties by index
    order = np.lexsort((np.broadcast_to(np.arange(v.shape[1]), v.shape), np.isnan(logits), -v), axis=-1)[:, :k]
    assert np.array_equal(ids, order)
    m = v.max(1, keepdims=True)
    with np.errstate(invalid="ignore"):
        e = np.where(v == m, 1.0, np.exp(v - m))
        d = np.where(np.isfinite(v - m), np.abs(v - m), 0.0)
    e = np.where(m == -np.inf, 0.0, e)
    chosen, dc = np.take_along_axis(e, order, 1), np.take_along_axis(d, order, 1)
    base, db = (e, d) if mode == RouteMode.SOFTMAX_ALL else (chosen, dc)
    total = base.sum(1, keepdims=True)
    rel_total = (base * (db + 4)).sum(1, keepdims=True) / np.where(total > 0, total, 1) + 70
    want = np.where(total > 0, np.float64(np.float32(scale)) * chosen / np.where(total > 0, total, 1), 0.0)
    # an exponential below the normal range is off by 2^-149 at most, or lost
    assert np.all(np.abs(w - want) <= np.abs(want) * (dc + 8 + rel_total) * U + abs(scale) * 2.0 ** -126)


@pytest.mark.parametrize("experts", [1, 2, 8, 15, 16, 17, 32, 60, 64, 128, 129, 256, 500, 512, 1000, 1024])
@pytest.mark.parametrize("mode", list(RouteMode), ids=lambda m: m.name)
def test_each_size(ctx, experts, mode):
    for tokens in (1, 3, 70):
        logits = fx.synth.normal(experts + tokens, tokens * experts).reshape(tokens, experts) * np.float32(3)
        for k in sorted({1, min(2, experts), min(8, experts), min(16, experts), min(17, experts), min(40, experts), experts}):
            _check(ctx, logits, k, mode, 1.0 if k != 2 else 2.5)


def test_many_tokens(ctx):
    logits = fx.synth.normal(3, 9001 * 128).reshape(9001, 128)
    for mode in RouteMode:
        _check(ctx, logits, 8, mode)


@pytest.mark.parametrize("mode", list(RouteMode), ids=lambda m: m.name)
def test_ties_masks_and_not_a_number(ctx, mode):
    rng = np.random.default_rng(4)
    logits = rng.integers(-2, 3, (64, 40)).astype(np.float32)  # ties everywhere
    logits[0] = 1.0
    logits[1] = -np.inf
    logits[2] = np.nan
    logits[3, 5:] = -np.inf
    logits[4, ::2] = np.nan
    logits[5, 1:] = np.nan
    logits[6, 7] = np.inf
    logits[7, 7] = logits[7, 9] = np.inf
    logits[8] = np.where(np.arange(40) % 2, 0.0, -0.0)
    logits[9] = -np.float32(3.4e38)
    logits[10, 3] = 3.4e38
    logits[11, 4:] = np.where(np.arange(36) % 2, np.nan, -np.inf)
    logits[12] = np.float32(1e-41) * np.arange(40)[::-1]  # subnormals in order
    logits.view(np.uint32)[13, 6] = 0xFFC00001  # a negative NaN
    for k in (1, 4, 8, 20, 40):
        _check(ctx, logits, k, mode)


def test_repeats_bit_for_bit(ctx):
    logits = fx.synth.normal(11, 300 * 128).reshape(300, 128)
    a, b = _route(ctx, logits, 8, RouteMode.SOFTMAX_ALL), _route(ctx, logits, 8, RouteMode.SOFTMAX_ALL)
    assert all(np.array_equal(x.view(np.uint32), y.view(np.uint32)) for x, y in zip(a, b))
