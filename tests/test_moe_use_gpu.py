"""The expert half of a block as programs use it: captured and replayed, two contexts at once, after the attention half,
and at sizes whose offsets pass 32 bits."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from moearc_amd import (NO_EXPERT, OUT_F16, OUT_F32, Context, DeviceView, MoeAct, MoeDesc, QuantType, RouteMode)
from moearc_amd.context import Failed
from test_moe_gpu import TYPES, U, activation, ids_of, product, run_ffn, run_linear, step16, weights

pytestmark = pytest.mark.gpu


class Half:
    """Norm, router logits, choice and experts of t tokens on one context, with a workspace of its own."""

    def __init__(self, cx, t, seed, types=(QuantType.MXFP4, QuantType.Q4_K), e=16, k=4, embd=512, ff=256):
        rng = np.random.default_rng(seed)
        self.cx, self.t, self.e, self.k, self.embd = cx, t, e, k, embd
        self.h = rng.standard_normal((t, embd)).astype(np.float32)
        made = [weights(types[i > 1], e, r, c, seed + i)[0] for i, (r, c) in enumerate([(ff, embd), (ff, embd), (embd, ff)])]
        up = cx.upload
        self.bh, self.bx, self.bn = up(self.h), cx.alloc(self.h.nbytes), up(1 + 0.1 * rng.standard_normal(embd).astype(np.float32))
        self.bl, self.bi, self.bt = (cx.alloc(t * n * 4) for n in (e, k, k))
        self.router = up(weights(QuantType.F16, 1, e, embd, 9)[0])
        self.desc = MoeDesc.make([types[0], types[0], types[1]], [up(m) for m in made], [None] * 3, e, embd, ff,
                                 MoeAct.SWIGLU_CLAMPED)
        self.ws = cx.alloc(cx.moe_workspace(t, k, e, embd, ff))

    def run(self, ws=True):
        c = self.cx
        c.norm_residual(self.bx, self.bh, None, None, None, 0, 1.0, self.bn, self.t, self.embd, 1e-5)
        c.matmul_q(QuantType.F16, self.bl, self.router, self.bx, None, self.t, self.e, self.embd)
        c.moe_route(self.bi, self.bt, self.bl, self.t, self.e, self.k, RouteMode.SOFTMAX_SELECTED)
        c.moe_ffn(self.desc, self.bh, self.bx, self.bi, self.bt, self.t, self.k, accumulate=True, workspace=self.ws if ws else None)

    def reset(self):
        self.cx.upload_slice(self.bh, self.h)

    def out(self):
        return self.cx.download(self.bh, np.float32, self.h.shape)


class Graph:
    def __init__(self, cx, fn):
        self.hip, self.stream = ctypes.CDLL("libamdhip64.so"), ctypes.c_void_p(cx.stream)
        graph, self.exe = ctypes.c_void_p(), ctypes.c_void_p()
        assert self.hip.hipStreamBeginCapture(self.stream, 1) == 0
        fn()
        assert self.hip.hipStreamEndCapture(self.stream, ctypes.byref(graph)) == 0
        assert self.hip.hipGraphInstantiate(ctypes.byref(self.exe), graph, None, None, ctypes.c_size_t(0)) == 0
        self.hip.hipGraphDestroy(graph)

    def launch(self):
        assert self.hip.hipGraphLaunch(self.exe, self.stream) == 0

    def close(self):
        self.hip.hipGraphExecDestroy(self.exe)


@pytest.mark.parametrize("t", [1, 9, 150])
def test_replays_equal_eager_calls(t):
    """The half block captured, replayed between eager calls of other sizes that grow the context's own workspace."""
    with Context() as cx:
        a, other = Half(cx, t, 3), Half(cx, 400, 4)
        a.run()
        want = a.out()
        assert not np.array_equal(want, a.h)
        other.run(False)
        want_other = other.out()
        g = Graph(cx, a.run)
        for _ in range(4):
            a.reset()
            g.launch()
            assert np.array_equal(a.out(), want)
            other.reset()
            other.run(False)
            assert np.array_equal(other.out(), want_other)
        # replays see the data of their time: another residual, same buffers
        h = a.h
        a.h = np.roll(h, 1, axis=1)
        a.reset()
        a.run()
        want = a.out()
        a.reset()
        g.launch()
        assert np.array_equal(a.out(), want)
        g.close()


@pytest.mark.parametrize("t", [1, 20, 100])
def test_a_replay_reports_ids_out_of_range(t):
    with Context() as cx:
        a = Half(cx, t, 5)
        a.run()
        good = cx.download(a.bi, np.uint32, (t, a.k))
        g = Graph(cx, lambda: cx.moe_ffn(a.desc, a.bh, a.bx, a.bi, a.bt, t, a.k, workspace=a.ws))
        bad = good.copy()
        bad[0, 1] = a.e
        for ids, fails in ((good, False), (bad, True), (good, False), (bad, True)):
            cx.upload_slice(a.bi, ids)
            g.launch()
            if fails:
                with pytest.raises(Failed):
                    cx.sync()
            cx.sync()
        g.close()


def test_two_contexts_at_once():
    with Context() as c1, Context() as c2:
        halves = [Half(c1, 150, 6), Half(c2, 150, 7), Half(c1, 1, 8), Half(c2, 5, 9)]
        want = []
        for x in halves:
            x.run(False)
            want.append(x.out())
            x.reset()
        for x in halves:
            x.run(False)
        for x, w in zip(halves, want):
            assert np.array_equal(x.out(), w)


@pytest.mark.parametrize("ty", [QuantType.Q8_0, QuantType.MXFP4], ids=lambda t: t.name)
def test_experts_beyond_four_gib(ty):
    """1024 experts of which the last ones, more than 2^32 bytes into the tensor, are used."""
    rows, cols, used = 8192, 1024, [1023, 1020]
    size = rows * ty.row_bytes(cols)
    with Context() as cx:
        bw = cx.alloc(1024 * size)
        raw, w = weights(ty, 2, rows, cols, 4)
        for i, e in enumerate(used):
            view = DeviceView(bw, e * size, size)
            part = np.ascontiguousarray(raw.reshape(2, size)[i])
            cx.upload_slice(view, part)
        assert used[1] * size > 1 << 32
        rng = np.random.default_rng(1)
        for t in (1, 3, 70):
            x = rng.standard_normal((t, 1, cols)).astype(np.float32)
            pick = np.stack([rng.permutation(2) for _ in range(t)])
            bx, bi, by = cx.upload(x), cx.upload(np.array(used, np.uint32)[pick]), cx.alloc(t * 2 * rows * 4)
            cx.matmul_experts(ty, by, bw, bx, None, bi, t, 2, 1024, rows, cols)
            at = rng.integers(0, t, 3)
            want, tol = product(w, None, x[at], pick[at], False)
            assert np.all(np.abs(cx.download(by, np.float32, (t, 2, rows))[at] - want) <= tol)
        # one token through gate, up and down: down [cols][rows] has the same bytes, read with longer rows
        wd, ids = w.reshape(2, cols, rows), np.array([[0, 1]])
        x = rng.standard_normal((1, 1, cols)).astype(np.float32)
        wt = np.array([[0.75, 0.5]], np.float32)
        desc = MoeDesc.make([ty] * 3, [bw] * 3, [None] * 3, 1024, cols, rows)
        for t in (1, 40):
            bx, bi, bt = cx.upload(np.repeat(x[0], t, 0)), cx.upload(np.array(used * t, np.uint32)), cx.upload(np.repeat(wt, t, 0))
            by = cx.alloc(t * cols * 4)
            cx.moe_ffn(desc, by, bx, bi, bt, t, 2)
            g, dg = product(w, None, x, ids, False)
            a, da = activation(MoeAct.SWIGLU, g, g, dg, dg)
            o, do = product(wd, None, a, ids, True)
            want = (wt[0] @ o[0])
            tol = sum(wt[0, j] * (do[0, j] + 1.01 * np.abs(wd[j]) @ da[0, j] + 4 * U * np.abs(o[0, j])) for j in range(2))
            got = cx.download(by, np.float32, (t, cols))
            assert np.all(np.abs(got[[0, t - 1]] - want) <= tol)


def test_outputs_beyond_2_32_elements():
    t, rows, cols = 33000, 131072 + 32, 256
    raw, w = weights(QuantType.Q8_0, 1, rows, cols, 2)
    rng = np.random.default_rng(2)
    x = rng.standard_normal((t, 1, cols)).astype(np.float16)
    with Context() as cx:
        by, ids = cx.alloc(t * rows * 2), np.zeros((t, 1), np.uint32)
        ids[7::1000] = NO_EXPERT
        cx.matmul_experts(QuantType.Q8_0, by, cx.upload(raw), cx.upload(x), None, cx.upload(ids), t, 1, 1, rows, cols, OUT_F16)
        for i in (0, 7, 8191, 8192, 32767, t - 1):
            want, tol = product(w, None, x[i:i + 1], ids[i:i + 1], False)
            got = cx.download(DeviceView(by, i * rows * 2, rows * 2), np.float16, (1, 1, rows)).astype(np.float64)
            assert np.all(np.abs(got - want) <= tol + step16(want, OUT_F16))


def test_norms_beyond_2_32_elements():
    n, cols = (1 << 21) + 3, 2048
    rng = np.random.default_rng(3)
    tail = rng.standard_normal((2, cols)).astype(np.float32)
    with Context() as cx:
        bh, bx = cx.alloc(n * cols * 4), cx.alloc(n * cols * 2)
        for view in (DeviceView(bh, 0, tail.nbytes), DeviceView(bh, (n - 2) * cols * 4, tail.nbytes)):
            cx.upload_slice(view, tail)
        cx.norm_residual(bx, bh, None, None, None, 0, 1.0, None, n, cols, 1e-5, x_type=OUT_F16)
        want = tail / np.sqrt((tail.astype(np.float64) ** 2).mean(1, keepdims=True) + 1e-5)
        tol = 2.0 ** -11 * np.abs(want) * (1 + 2.0 ** -10) + 2.0 ** -25 + 60 * U * np.abs(want)
        for r in (0, n - 2):
            got = cx.download(DeviceView(bx, r * cols * 2, 2 * cols * 2), np.float16, (2, cols)).astype(np.float64)
            assert np.all(np.abs(got - want) <= tol)


def test_more_rows_than_a_launch_has_threads_for():
    n = (1 << 27) + 5
    rng = np.random.default_rng(4)
    v = (rng.standard_normal(n).astype(np.float32))
    v[v == 0] = 1
    with Context() as cx:
        b, bx = cx.upload(v), cx.alloc(n * 4)
        cx.norm_residual(bx, b, None, None, None, 0, 1.0, None, n, 1, 0.0)
        got = cx.download(bx, np.float32, (n,))
        assert np.all(np.abs(got - np.sign(v)) <= 6 * U)
        ids, w = cx.upload(np.full(n, 9, np.uint32)), bx
        cx.moe_route(ids, w, b, n, 1, 1, RouteMode.SOFTMAX_ALL, 2.5)
        assert not cx.download(ids, np.uint32, (n,)).any() and np.all(cx.download(w, np.float32, (n,)) == 2.5)


@pytest.mark.parametrize("ty", TYPES, ids=lambda t: t.name)
@pytest.mark.parametrize("io", [OUT_F32, OUT_F16], ids=["f32", "f16"])
def test_both_sides_of_each_form(ctx, ty, io):
    """64 and 65 slots, 24 and 25 over many experts (without and with a plan), and the slots per expert at which tiles
    grow."""
    for t in (24, 25):
        run_linear(ctx, ty, t, 1, 40, 65, 512, io, seed=t)
        run_ffn(ctx, (ty, ty), t, 1, 32, 256, 256, io, seed=t)
    for t in (64, 65):
        run_linear(ctx, ty, t, 1, 3, 65, 512, io, seed=t)
    for each in (39, 40, 55, 56):
        run_linear(ctx, ty, each, 2, 2, 129, 256, io, seed=each)
        run_linear(ctx, ty, each * 3, 1, 3, 40, 256, io, seed=each, ids=np.full((each * 3, 1), 1, np.uint32))
    run_ffn(ctx, (ty, ty), 56, 2, 2, 256, 288 if ty.block_elems < 256 else 512, io, seed=6)


def test_padded_tokens_leave_the_others_alone(ctx):
    """Rows of a padded batch hold infinities and NaN; their slots choose no expert."""
    ty, e, k, rows, cols = QuantType.MXFP4, 6, 2, 70, 256
    raw, w = weights(ty, e, rows, cols, 8)
    bw = ctx.upload(raw)
    for t in (6, 90):
        rng = np.random.default_rng(t)
        x, ids = rng.standard_normal((t, 1, cols)).astype(np.float32), ids_of(rng, t, k, e)
        x[t // 2:] = np.inf
        x[t - 1] = np.nan
        ids[t // 2:] = NO_EXPERT
        by = ctx.upload(np.full((t, k, rows), 7, np.float32))
        ctx.matmul_experts(ty, by, bw, ctx.upload(x), None, ctx.upload(ids), t, k, e, rows, cols)
        got = ctx.download(by, np.float32, (t, k, rows))
        want, tol = product(w, None, x[:t // 2], ids[:t // 2], False)
        assert np.all(np.abs(got[:t // 2] - want) <= tol) and not got[t // 2:].any()


@pytest.mark.parametrize("ty", TYPES, ids=lambda t: t.name)
@pytest.mark.parametrize("io", [OUT_F32, OUT_F16], ids=["f32", "f16"])
def test_infinities_stay_in_their_token(ctx, ty, io):
    """A live token of infinities and NaN changes no other token's result, not by a bit."""
    e, k, embd, ff = 3, 2, 256, 256
    made = [ctx.upload(weights(ty, e, r, c, 30 + i)[0]) for i, (r, c) in enumerate([(ff, embd), (ff, embd), (embd, ff)])]
    desc = MoeDesc.make([ty] * 3, made, [None] * 3, e, embd, ff)
    for t in (7, 40, 150):
        rng = np.random.default_rng(t)
        dtype = np.float16 if io == OUT_F16 else np.float32
        x, ids = rng.standard_normal((t, embd)).astype(dtype), ids_of(rng, t, k, e)
        bi, bt = ctx.upload(ids), ctx.upload(np.full((t, k), 0.5, np.float32))
        out = []
        for spoilt in (False, True):
            if spoilt:
                x[3], x[5, ::3] = np.inf, np.nan
            by = ctx.alloc(t * embd * 4)
            ctx.moe_ffn(desc, by, ctx.upload(x), bi, bt, t, k, io_type=io)
            out.append(ctx.download(by, dtype, (t, embd)))
        rest = [i for i in range(t) if i not in (3, 5)]
        assert np.array_equal(out[0][rest], out[1][rest]) and np.isfinite(out[0]).all()
        assert not np.isfinite(out[1][[3, 5]]).any()


@pytest.mark.parametrize("io", [OUT_F32, OUT_F16], ids=["f32", "f16"])
@pytest.mark.parametrize("t", [1, 9, 100])
def test_tensors_at_any_element(ctx, io, t):
    """Inputs, outputs, biases, ids and weights one element off the allocation's alignment: the same bits."""
    e, k, embd, ff = 5, 3, 512, 256
    elem = 2 if io == OUT_F16 else 4
    dtype = np.float16 if io == OUT_F16 else np.float32
    for types in ((QuantType.MXFP4, QuantType.Q8_0), (QuantType.F16, QuantType.Q6_K), (QuantType.Q5_K, QuantType.Q4_K)):
        rng = np.random.default_rng(t)
        made = [ctx.upload(weights(types[i > 1], e, r, c, 40 + i)[0]) for i, (r, c) in enumerate([(ff, embd), (ff, embd), (embd, ff)])]
        data = [rng.standard_normal((t, embd)).astype(dtype), ids_of(rng, t, k, e), rng.random((t, k)).astype(np.float32),
                *(rng.standard_normal((e, n)).astype(np.float32) for n in (ff, ff, embd))]
        out = []
        for off in (0, 1):
            def place(a):
                step = off * a.dtype.itemsize
                return DeviceView(ctx.upload(np.concatenate([np.zeros(step, np.uint8), np.ascontiguousarray(a).view(np.uint8).reshape(-1)])), step)
            bx, bi, bt, *bs = (place(a) for a in data)
            desc = MoeDesc.make([types[0], types[0], types[1]], made, bs, e, embd, ff, MoeAct.SWIGLU_CLAMPED)
            by = ctx.upload(np.full((t * embd + 2) * elem, 0x5A, np.uint8))
            ctx.moe_ffn(desc, DeviceView(by, off * elem), bx, bi, bt, t, k, io_type=io)
            raw = ctx.download(by, np.uint8, ((t * embd + 2) * elem,))
            assert np.all(raw[:off * elem] == 0x5A) and np.all(raw[(t * embd + off) * elem:] == 0x5A)
            out.append(raw[off * elem:(t * embd + off) * elem].copy().view(dtype))
        assert np.array_equal(*out)


def test_every_expert_of_1024(ctx):
    for t, per_slot in ((1, False), (2, True)):
        run_linear(ctx, QuantType.Q8_0, t, 1024, 1024, 33, 256, OUT_F16, per_slot=per_slot, seed=t)
    run_ffn(ctx, (QuantType.MXFP4, QuantType.MXFP4), 2, 512, 512, 256, 256, add=True, seed=3)
