"""The experts' products (moearc_matmul_experts, moearc_moe_ffn) against float64 over the formats' exact values.

Bounds, u = 2^-24: a product is within 2 (32 + cols / 32 + 5) u sum|w x| (moearc_matmul_q's); through the activation
an error of g moves the result by at most 1.1 |u| (the largest slope of g sigmoid(g)), one of u by |g sigmoid(g)|, and it
rounds 8 times itself; the second product adds its own and sum|w| times the first's; the sum over a token's experts
one rounding each. f16 activations add half a step of f16, 2^-11, where values are rounded to it: between the
products, and at the end. Below the f16 range the steps are 2^-24."""
from __future__ import annotations

import numpy as np
import pytest

import fixtures as fx
from moearc_amd import (NO_EXPERT, OUT_F16, OUT_F32, Context, DeviceView, MoeAct, MoeDesc, QuantType, RouteMode)
from moearc_amd.context import Failed
from oracle import oracle

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = [QuantType.F16, QuantType.Q8_0, QuantType.Q4_K, QuantType.Q5_K, QuantType.Q6_K, QuantType.MXFP4]
ALPHA, LIMIT = 1.702, 7.0


def weights(ty, experts, rows, cols, seed):
    """(bytes, float64 [experts, rows, cols]): random payloads, blocks scaled to about 1 / sqrt(cols)."""
    ty = QuantType(ty)
    n = experts * rows * cols // ty.block_elems
    rng = np.random.default_rng(seed)
    b = rng.integers(0, 256, (n, ty.block_bytes), dtype=np.uint8)
    size = 1 / np.sqrt(cols)

    def half(at, v):
        b[:, at:at + 2] = (v * rng.uniform(0.5, 1.5, n)).astype(np.float16).view(np.uint8).reshape(n, 2)
    if ty == QuantType.F16:
        b[:] = (rng.standard_normal(n) * size).astype(np.float16).view(np.uint8).reshape(n, 2)
    elif ty == QuantType.Q8_0:
        half(0, size / 74)
    elif ty == QuantType.MXFP4:
        b[:, 0] = rng.integers(120, 124, n)
    elif ty == QuantType.Q6_K:
        half(208, size / 1300)
    else:
        half(0, size / (320 if ty == QuantType.Q4_K else 640))
        half(2, size / 40)
    w = oracle.dequant(int(ty), b.reshape(-1), n).astype(np.float64).reshape(experts, rows, cols)
    return b.reshape(-1), w


def round_io(v, io):
    return v.astype(np.float16 if io == OUT_F16 else np.float32)


def product(w, bias, x, ids, per_slot):
    """(y, bound) [tokens, used, rows] in float64."""
    t, k = ids.shape
    rows, cols = w.shape[1:]
    y, tol = np.zeros((t, k, rows)), np.zeros((t, k, rows))
    for i in range(t):
        for j in range(k):
            e = ids[i, j]
            if e < len(w):
                v = x[i, j if per_slot else 0].astype(np.float64)
                y[i, j] = w[e] @ v + (0 if bias is None else bias[e])
                tol[i, j] = (2 * (32 + cols / 32 + 5) * U * (np.abs(w[e]) @ np.abs(v)) + U * np.abs(y[i, j]) +
                             2.0 ** -24 * np.abs(w[e]).sum(1))
    return y, tol


def activation(act, g, u, dg, du):
    """(a, bound)."""
    if act == MoeAct.SWIGLU_CLAMPED:
        g, u = np.minimum(g, LIMIT), np.clip(u, -LIMIT, LIMIT) + 1
        s = g / (1 + np.exp(-ALPHA * g))
    else:
        s = g / (1 + np.exp(-g))
    a = s * u
    return a, 1.1 * np.abs(u) * dg + np.abs(s) * du + 1.1 * dg * du + 8 * U * (1 + np.abs(g)) * np.abs(a)


def step16(v, io):
    return 2.0 ** -11 * np.abs(v) * (1 + 2.0 ** -10) + 2.0 ** -25 if io == OUT_F16 else 0.0


def ids_of(rng, t, k, e, skip=0.0):
    ids = np.stack([rng.permutation(max(e, k))[:k] % e for _ in range(t)]).astype(np.uint32)
    if skip:
        ids[rng.random(ids.shape) < skip] = NO_EXPERT
    return ids


def run_linear(ctx, ty, t, k, e, rows, cols, io=OUT_F32, bias=True, per_slot=False, ids=None, skip=0.0, seed=1, shift=0,
               ws=None, made=None):
    rng = np.random.default_rng(seed)
    raw, w = made or weights(ty, e, rows, cols, seed)
    b = rng.standard_normal((e, rows)).astype(np.float32) if bias else None
    x = round_io(rng.standard_normal((t, k if per_slot else 1, cols)), io)
    ids = ids_of(rng, t, k, e, skip) if ids is None else ids
    bw = DeviceView(ctx.upload(np.concatenate([np.zeros(shift, np.uint8), raw])), shift)
    bx, bi = ctx.upload(x), ctx.upload(ids)
    bb = ctx.upload(b) if bias else None
    pad = 64
    by = ctx.upload(np.full(t * k * rows + pad, 9, x.dtype))
    ctx.matmul_experts(ty, by, bw, bx, bb, bi, t, k, e, rows, cols, io, per_slot, ws)
    got = ctx.download(by, x.dtype, (t * k * rows + pad,))
    assert np.all(got[t * k * rows:] == 9)
    got = got[:t * k * rows].reshape(t, k, rows)
    want, tol = product(w, b, x, ids, per_slot)
    tol = tol + step16(want, io)
    worst = np.max(np.abs(got - want) / np.where(tol > 0, tol, 1))
    assert np.all(np.abs(got - want) <= tol), worst
    return got


def run_ffn(ctx, types, t, k, e, embd, ff, io=OUT_F32, act=MoeAct.SWIGLU, bias=True, add=False, ids=None, skip=0.0,
            seed=1, ws=None):
    rng = np.random.default_rng(seed)
    shapes = [(ff, embd), (ff, embd), (embd, ff)]
    made = [weights(types[i > 1], e, r, c, seed + i) for i, (r, c) in enumerate(shapes)]
    bs = [rng.standard_normal((e, r)).astype(np.float32) * np.float32(0.2) if bias else None for r, _ in shapes]
    x = round_io(rng.standard_normal((t, embd)), io)
    ids = ids_of(rng, t, k, e, skip) if ids is None else ids
    wt = rng.random((t, k)).astype(np.float32)
    wt[ids >= e] = np.nan  # not read
    y0 = rng.standard_normal((t, embd)).astype(x.dtype)
    bufs = [ctx.upload(m[0]) for m in made]
    bb = [ctx.upload(b) if bias else None for b in bs]
    desc = MoeDesc.make([types[0], types[0], types[1]], bufs, bb, e, embd, ff, act, ALPHA, LIMIT)
    by, bx, bi, bt = ctx.upload(y0), ctx.upload(x), ctx.upload(ids), ctx.upload(wt)
    ctx.moe_ffn(desc, by, bx, bi, bt, t, k, io, add, ws)
    got = ctx.download(by, x.dtype, (t, embd))
    (g, dg), (u, du) = (product(made[i][1], bs[i], x[:, None], ids, False) for i in (0, 1))
    a, da = activation(act, g, u, dg, du)
    da = da + step16(a, io)
    o, do = product(made[2][1], bs[2], a, ids, True)
    want, tol = np.zeros((t, embd)), np.zeros((t, embd))
    for i in range(t):
        for j in range(k):
            if ids[i, j] < e:
                moved = np.abs(made[2][1][ids[i, j]]) @ da[i, j]
                want[i] += wt[i, j] * o[i, j]
                tol[i] += wt[i, j] * (do[i, j] + 1.01 * moved + (k + 2) * U * np.abs(o[i, j]))
    if add:
        want = want + y0
        tol += U * np.abs(want)
    tol = tol + step16(want, io)
    assert np.all(np.abs(got - want) <= tol), np.max(np.abs(got - want) / np.where(tol > 0, tol, 1))
    return got


@pytest.mark.parametrize("ty", TYPES, ids=lambda t: t.name)
@pytest.mark.parametrize("io", [OUT_F32, OUT_F16], ids=["f32", "f16"])
@pytest.mark.parametrize("t,k,e,rows,cols", [
    (1, 1, 1, 1, 256), (1, 2, 4, 31, 256), (3, 2, 5, 33, 512), (16, 4, 8, 48, 256), (17, 1, 2, 64, 768), (64, 1, 1, 40, 256),
    (33, 2, 3, 40, 256), (100, 2, 3, 70, 512), (70, 8, 40, 24, 256), (300, 1, 2, 129, 256), (65, 4, 4, 257, 512)])
def test_each_format(ctx, ty, io, t, k, e, rows, cols):
    run_linear(ctx, ty, t, k, e, rows, cols, io, seed=t + rows)
    run_linear(ctx, ty, t, k, e, rows, cols, io, bias=False, per_slot=True, seed=t + rows + 1)


@pytest.mark.parametrize("ty,cols", [(QuantType.F16, c) for c in (288, 320, 1000 - 1000 % 32)] +
                         [(t, c) for t in (QuantType.Q8_0, QuantType.MXFP4) for c in (288, 320, 352, 992)] +
                         [(t, c) for t in (QuantType.Q4_K, QuantType.Q5_K, QuantType.Q6_K) for c in (1280, 2304)], ids=str)
def test_odd_row_lengths(ctx, ty, cols):
    for t in (2, 40, 90):
        run_linear(ctx, ty, t, 3, 7, 50, cols, seed=cols)
        run_linear(ctx, ty, t, 3, 7, 50, cols, OUT_F16, seed=cols)


@pytest.mark.parametrize("ty", TYPES, ids=lambda t: t.name)
def test_scales_of_every_size(ctx, ty):
    """Blocks whose scales are zero, negative, or orders of magnitude from their neighbours'."""
    e, rows, cols = 3, 70, 1024
    raw, _ = weights(ty, e, rows, cols, 5)
    b = raw.reshape(-1, ty.block_bytes).copy()
    rng = np.random.default_rng(6)
    pick = rng.integers(0, 4, len(b))
    at = {QuantType.Q6_K: [208], QuantType.Q8_0: [0], QuantType.Q4_K: [0, 2], QuantType.Q5_K: [0, 2]}.get(ty, [])
    for i in at:
        d = b[:, i:i + 2].copy().view(np.float16)[:, 0]
        d = np.where(pick == 0, 0, np.where(pick == 1, -d, np.where(pick == 2, d * np.float16(100), d))).astype(np.float16)
        b[:, i:i + 2] = d.view(np.uint8).reshape(-1, 2)
    if ty == QuantType.MXFP4:  # some windows within f16's normal range, most not; the smallest exponents too
        b[:, 0] = np.where(np.arange(len(b)) % 32 < 8, rng.integers(114, 140, len(b)), rng.integers(90, 150, len(b)))
        b[rng.integers(0, len(b), 40), 0] = 0
        b[:32 * rows // 2, 0] = rng.integers(114, 140, 32 * rows // 2)  # half an expert all within it
    raw = b.reshape(-1)
    w = oracle.dequant(int(ty), raw, len(b)).astype(np.float64).reshape(e, rows, cols)
    for t in (4, 100):
        for io in (OUT_F32, OUT_F16) if ty != QuantType.MXFP4 else (OUT_F32,):  # f16 could not hold the sums
            run_linear(ctx, ty, t, 2, e, rows, cols, io, bias=False, made=(raw, w))


@pytest.mark.parametrize("ty", TYPES, ids=lambda t: t.name)
def test_weights_at_any_even_address(ctx, ty):
    for shift in (2, 6, 14):
        run_linear(ctx, ty, 4, 2, 4, 33, 512, shift=shift)
        run_linear(ctx, ty, 80, 2, 4, 33, 512, shift=shift)


@pytest.mark.parametrize("t", [5, 90])
@pytest.mark.parametrize("io", [OUT_F32, OUT_F16], ids=["f32", "f16"])
def test_skipped_slots(ctx, t, io):
    for ty in (QuantType.MXFP4, QuantType.Q4_K):
        got = run_linear(ctx, ty, t, 4, 6, 40, 256, io, skip=0.4, seed=t)
        assert np.any(got == 0)
        run_linear(ctx, ty, t, 4, 6, 40, 256, io, ids=np.full((t, 4), NO_EXPERT, np.uint32))
        run_ffn(ctx, (ty, ty), t, 4, 6, 256, 256, io, skip=0.4, seed=t)
        run_ffn(ctx, (ty, ty), t, 4, 6, 256, 256, io, ids=np.full((t, 4), NO_EXPERT, np.uint32))


@pytest.mark.parametrize("t", [1, 7, 64, 150])
def test_one_expert_for_all_and_repeats(ctx, t):
    ty = QuantType.Q8_0
    run_linear(ctx, ty, t, 1, 9, 40, 256, ids=np.full((t, 1), 5, np.uint32))
    run_linear(ctx, ty, t, 3, 9, 40, 256, ids=np.full((t, 3), 8, np.uint32), per_slot=True)
    run_ffn(ctx, (ty, ty), t, 3, 9, 256, 256, ids=np.full((t, 3), 0, np.uint32))


@pytest.mark.parametrize("types", [(t, t) for t in TYPES] + [(QuantType.Q4_K, QuantType.Q6_K), (QuantType.MXFP4, QuantType.F16)],
                         ids=lambda p: p[0].name + "_" + p[1].name)
@pytest.mark.parametrize("io", [OUT_F32, OUT_F16], ids=["f32", "f16"])
@pytest.mark.parametrize("t,k,e,embd,ff", [(1, 4, 16, 256, 512), (6, 2, 4, 512, 256), (130, 4, 8, 256, 256)])
def test_ffn(ctx, types, io, t, k, e, embd, ff):
    for act in MoeAct:
        run_ffn(ctx, types, t, k, e, embd, ff, io, act, seed=t)
    run_ffn(ctx, types, t, k, e, embd, ff, io, bias=False, add=io == OUT_F32, seed=t + 5)


@pytest.mark.parametrize("ty", TYPES, ids=lambda t: t.name)
@pytest.mark.parametrize("io", [OUT_F32, OUT_F16], ids=["f32", "f16"])
def test_ffn_of_a_single_token(ctx, ty, io):
    wide = 2304 if ty in (QuantType.Q4_K, QuantType.Q5_K, QuantType.Q6_K) else 2080
    for k, e, embd, ff in ((1, 3, 256, 512), (4, 9, 768, 256), (8, 8, 512, 768), (13, 20, 256, 256), (2, 3, wide, 256), (2, 3, 256, wide),
                           (64, 5, 256, 256), (65, 70, 256, 256), (1, 2, 5120, 256), (8, 9, 256, 5120)):
        run_ffn(ctx, (ty, ty), 1, k, e, embd, ff, io, MoeAct(k % 2), bias=k != 4, add=io == OUT_F32 and k % 2 == 0, seed=k)
    for k, ids in ((4, [NO_EXPERT, 2, NO_EXPERT, 1]), (4, [NO_EXPERT] * 4), (3, [5, 5, 5]), (8, [NO_EXPERT] * 7 + [3])):
        for add in (False, True) if io == OUT_F32 else (False,):
            run_ffn(ctx, (ty, ty), 1, k, 6, 256, 512, io, add=add, ids=np.array([ids], np.uint32))


def test_ffn_odd_widths(ctx):
    run_ffn(ctx, (QuantType.MXFP4, QuantType.Q8_0), 3, 2, 5, 288, 352, add=True)
    run_ffn(ctx, (QuantType.Q8_0, QuantType.MXFP4), 77, 2, 5, 352, 288, act=MoeAct.SWIGLU_CLAMPED)
    run_ffn(ctx, (QuantType.F16, QuantType.F16), 77, 3, 5, 288, 288, OUT_F16)


def test_chunked_calls_equal_their_parts(ctx):
    # 33,000 slots run as two chunks; each token's result is what its own chunk gives
    t, k, e, rows, cols = 8250, 4, 16, 32, 256
    made = weights(QuantType.Q8_0, e, rows, cols, 3)
    rng = np.random.default_rng(3)
    x, ids = rng.standard_normal((t, cols)).astype(np.float32), ids_of(rng, t, k, e)
    bw, bx, bi = ctx.upload(made[0]), ctx.upload(x), ctx.upload(ids)
    by, bz = ctx.alloc(t * k * rows * 4), ctx.alloc(t * k * rows * 4)
    ctx.matmul_experts(QuantType.Q8_0, by, bw, bx, None, bi, t, k, e, rows, cols)
    cut = 8192
    for a, n in ((0, cut), (cut, t - cut)):
        ctx.matmul_experts(QuantType.Q8_0, DeviceView(bz, a * k * rows * 4), bw, DeviceView(bx, a * cols * 4), None,
                           DeviceView(bi, a * k * 4), n, k, e, rows, cols)
    y = ctx.download(by, np.float32, (t, k, rows))
    assert np.array_equal(y, ctx.download(bz, np.float32, (t, k, rows)))
    at = rng.integers(0, t, 50)
    want, tol = product(made[1], None, x[at][:, None], ids[at], False)
    assert np.all(np.abs(y[at] - want) <= tol)


@pytest.mark.parametrize("t", [4, 100])
def test_results_repeat_bit_for_bit(ctx, t):
    a, b = (run_ffn(ctx, (QuantType.MXFP4, QuantType.MXFP4), t, 4, 8, 512, 512, seed=2) for _ in range(2))
    assert np.array_equal(a, b)


@pytest.mark.parametrize("t", [3, 100])
def test_ids_out_of_range_are_reported_and_skipped(t):
    with Context() as cx:
        raw, w = weights(QuantType.Q8_0, 4, 40, 256, 1)
        ids = ids_of(np.random.default_rng(1), t, 2, 4)
        ids[1, 1], ids[2, 0] = 4, 0x80000001
        x = np.random.default_rng(2).standard_normal((t, 1, 256)).astype(np.float32)
        by, bw, bx, bi = cx.alloc(t * 2 * 40 * 4), cx.upload(raw), cx.upload(x), cx.upload(ids)
        cx.matmul_experts(QuantType.Q8_0, by, bw, bx, None, bi, t, 2, 4, 40, 256)
        with pytest.raises(Failed):
            cx.sync()
        cx.sync()
        got = cx.download(by, np.float32, (t, 2, 40))
        want, tol = product(w, None, x, ids, False)
        assert np.all(np.abs(got - want) <= tol) and not got[1, 1].any() and not got[2, 0].any()


def test_the_callers_workspace(ctx):
    for t in (3, 100):
        n = ctx.moe_workspace(t, 4, 8, 256, 512)
        raw = np.full(n + 256, 0xA5, np.uint8)  # what is in it does not matter, and nothing behind it is written
        ws = ctx.upload(raw)
        a = run_ffn(ctx, (QuantType.Q4_K, QuantType.Q6_K), t, 4, 8, 256, 512, ws=DeviceView(ws, 0, n))
        b = run_ffn(ctx, (QuantType.Q4_K, QuantType.Q6_K), t, 4, 8, 256, 512)
        assert np.array_equal(a, b)
        assert np.all(ctx.download(ws, np.uint8, (n + 256,))[n:] == 0xA5)
        n = ctx.moe_workspace(t, 4, 8, 256)
        ws = ctx.upload(np.full(n + 256, 0xA5, np.uint8))
        run_linear(ctx, QuantType.MXFP4, t, 4, 8, 70, 256, per_slot=True, ws=DeviceView(ws, 0, n))
        assert np.all(ctx.download(ws, np.uint8, (n + 256,))[n:] == 0xA5)


@pytest.mark.parametrize("t", [1, 20, 200])
def test_router_to_residual(ctx, t):
    """The expert half of a block as it is used: norm, router logits, choice, experts into the residual."""
    embd, ff, e, k = 512, 256, 16, 4
    rng = np.random.default_rng(t)
    h = rng.standard_normal((t, embd)).astype(np.float32)
    w_norm = 1 + 0.1 * rng.standard_normal(embd).astype(np.float32)
    raw_r, w_r = weights(QuantType.F16, 1, e, embd, 9)
    made = [weights(QuantType.MXFP4, e, r, c, 20 + i) for i, (r, c) in enumerate([(ff, embd), (ff, embd), (embd, ff)])]
    bh, bx, bn = ctx.upload(h), ctx.alloc(h.nbytes), ctx.upload(w_norm)
    bl, bi, bt = ctx.alloc(t * e * 4), ctx.alloc(t * k * 4), ctx.alloc(t * k * 4)
    br, bufs = ctx.upload(raw_r), [ctx.upload(m[0]) for m in made]
    desc = MoeDesc.make([QuantType.MXFP4] * 3, bufs, [None] * 3, e, embd, ff, MoeAct.SWIGLU_CLAMPED, ALPHA, LIMIT)
    ctx.norm_residual(bx, bh, None, None, None, 0, 1.0, bn, t, embd, 1e-5)
    ctx.matmul_q(QuantType.F16, bl, br, bx, None, t, e, embd)
    ctx.moe_route(bi, bt, bl, t, e, k, RouteMode.SOFTMAX_SELECTED)
    ctx.moe_ffn(desc, bh, bx, bi, bt, t, k, accumulate=True)
    ids, wt = ctx.download(bi, np.uint32, (t, k)), ctx.download(bt, np.float32, (t, k))
    hd = h.astype(np.float64)
    x = hd / np.sqrt((hd * hd).mean(1, keepdims=True) + 1e-5) * w_norm
    logits = x @ w_r[0].T
    # the choice is right to the logits' error: each chosen logit is at least what the k-th largest is, less 1e-4
    kth = -np.sort(-logits, 1)[:, k - 1:k]
    assert np.all(np.take_along_axis(logits, ids.astype(np.int64), 1) >= kth - 1e-4)
    v = np.take_along_axis(logits, ids.astype(np.int64), 1)
    p = np.exp(v - v.max(1, keepdims=True))
    assert np.allclose(wt, p / p.sum(1, keepdims=True), rtol=2e-4, atol=0)
    (g, dg), (u, du) = (product(made[i][1], None, x[:, None], ids, False) for i in (0, 1))
    slope = 60 * U  # x's own error, relative
    dg, du = ((d + slope * np.abs(m[1][ids]).sum(-1) * np.abs(x).max(1)[:, None, None]) for d, m in ((dg, made[0]), (du, made[1])))
    a, da = activation(MoeAct.SWIGLU_CLAMPED, g, u, dg, du)
    o, do = product(made[2][1], None, a, ids, True)
    want, tol = hd.copy(), U * np.abs(hd) * 4
    for j in range(k):
        want += wt[:, j:j + 1] * o[:, j]
        tol += wt[:, j:j + 1] * (do[:, j] + 1.01 * np.einsum("tio,to->ti", np.abs(made[2][1])[ids[:, j]], da[:, j]) +
                                 (k + 4) * U * np.abs(o[:, j]))
    assert np.all(np.abs(ctx.download(bh, np.float32, (t, embd)) - want) <= tol)
