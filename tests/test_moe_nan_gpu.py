"""Values of an expert's gate, up or input that are not finite reach the output, through both activations and on every form
(one token, up to 64 slots, light tiles, tiles)."""
from __future__ import annotations

import numpy as np
import pytest

from moearc_amd import OUT_F16, OUT_F32, MoeAct, MoeDesc, QuantType
from test_moe_gpu import ALPHA, LIMIT, TYPES, U, activation, ids_of, product, weights

pytestmark = pytest.mark.gpu
E, K, EMBD, FF = 3, 2, 256, 256
TOKENS = [1, 7, 40, 150]


def _layer(ty):
    return [weights(ty, E, r, c, 50 + i) for i, (r, c) in enumerate([(FF, EMBD), (FF, EMBD), (EMBD, FF)])]


def _run(ctx, ty, made, bias, act, x, ids, io, limit=LIMIT):
    desc = MoeDesc.make([ty] * 3, made, bias, E, EMBD, FF, act, ALPHA, limit)
    t = len(x)
    by, bt = ctx.alloc(x.nbytes), ctx.upload(np.full((t, K), 0.5, np.float32))
    ctx.moe_ffn(desc, by, ctx.upload(x), ctx.upload(ids), bt, t, K, io_type=io)
    return ctx.download(by, x.dtype, x.shape)


def _draw(t, io):
    rng = np.random.default_rng(t)
    x = rng.standard_normal((t, EMBD)).astype(np.float16 if io == OUT_F16 else np.float32)
    return x, ids_of(rng, t, K, E)


@pytest.mark.parametrize("ty", TYPES, ids=lambda t: t.name)
@pytest.mark.parametrize("io", [OUT_F32, OUT_F16], ids=["f32", "f16"])
@pytest.mark.parametrize("act", list(MoeAct), ids=lambda a: a.name)
@pytest.mark.parametrize("spoilt", [0, 1], ids=["gate", "up"])
def test_a_channel_that_is_not_a_number(ctx, ty, io, act, spoilt):
    """One channel of one expert's gate (up) is NaN: so are all results of the tokens that ask for it, and no others."""
    made = [ctx.upload(m[0]) for m in _layer(ty)]
    for t in TOKENS:
        x, ids = _draw(t, io)
        ids[:2] = [[1, 0], [2, 0]][:t]
        bad = np.zeros((E, FF), np.float32)
        good = _run(ctx, ty, made, [ctx.upload(bad), ctx.upload(bad), None], act, x, ids, io)
        for bits in (0x7FC00000, 0xFFC12345):
            bad.view(np.uint32)[1, 5] = bits
            bias = [ctx.upload(bad if i == spoilt else np.zeros_like(bad)) for i in (0, 1)] + [None]
            got = _run(ctx, ty, made, bias, act, x, ids, io)
            hit = (ids == 1).any(1)
            assert hit[0] and (t == 1 or not hit.all())
            assert np.isnan(got[hit]).all() and np.array_equal(got[~hit], good[~hit]) and np.isfinite(good).all()


@pytest.mark.parametrize("ty", TYPES, ids=lambda t: t.name)
@pytest.mark.parametrize("io", [OUT_F32, OUT_F16], ids=["f32", "f16"])
@pytest.mark.parametrize("act", list(MoeAct), ids=lambda a: a.name)
def test_inputs_that_are_not_a_number_or_too_large(ctx, ty, io, act):
    """NaN on every form, and f32 values that f16 does not hold where they enter as halves: the token's results are NaN."""
    made = [ctx.upload(m[0]) for m in _layer(ty)]
    for t in TOKENS:
        x, ids = _draw(t, io)
        good = _run(ctx, ty, made, [None] * 3, act, x, ids, io)
        x[0, 100] = np.nan
        bad = [0]
        if t > 1 and io == OUT_F32:
            x[3, 7], x[5, 255] = 7e4, -3e38
            bad = [0, 3, 5]
        got = _run(ctx, ty, made, [None] * 3, act, x, ids, io)
        rest = [i for i in range(t) if i not in bad]
        assert np.isnan(got[bad]).all() and np.array_equal(got[rest], good[rest]) and np.isfinite(good).all()


@pytest.mark.parametrize("t", TOKENS)
def test_infinite_gates_and_ups_are_clamped(ctx, t):
    """+inf clamps to the limit and -inf of an up to its negative, as min and max have it; -inf of a gate is no number."""
    layer = _layer(QuantType.Q8_0)
    made = [ctx.upload(m[0]) for m in layer]
    x, ids = _draw(t, OUT_F32)
    bias = [np.zeros((E, FF), np.float32) for _ in range(2)]
    bias[0][:, 3] = np.inf
    bias[1][:, 9], bias[1][:, 11] = np.inf, -np.inf
    got = _run(ctx, QuantType.Q8_0, made, [ctx.upload(b) for b in bias] + [None], MoeAct.SWIGLU_CLAMPED, x, ids, OUT_F32)
    (g, dg), (u, du) = (product(layer[i][1], None, x[:, None], ids, False) for i in (0, 1))
    g, u = (v + bias[i][ids] for i, v in ((0, g), (1, u)))
    a, da = activation(MoeAct.SWIGLU_CLAMPED, g, u, dg, du)
    o, do = product(layer[2][1], None, a, ids, True)
    want, tol = 0.5 * o.sum(1), np.zeros((t, EMBD))
    for j in range(K):
        tol += 0.5 * (do[:, j] + 1.01 * np.einsum("tio,to->ti", np.abs(layer[2][1])[ids[:, j]], da[:, j]) + (K + 2) * U * np.abs(o[:, j]))
    assert np.all(np.abs(got - want) <= tol)
    bias[0][:, 3] = -np.inf
    got = _run(ctx, QuantType.Q8_0, made, [ctx.upload(b) for b in bias] + [None], MoeAct.SWIGLU_CLAMPED, x, ids, OUT_F32)
    assert np.isnan(got).all()
