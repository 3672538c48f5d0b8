"""The ragged batches' calls as programs use them: one after the other, beside the single-sequence calls, captured and
replayed, on two contexts at once, over rings, and in pools whose offsets pass 32 bits."""
from __future__ import annotations

import numpy as np
import pytest

from moearc_amd import OUT_F16, OUT_F32, Context, DeviceView, KvType, QkvAppendDesc, RopeScaling
from moearc_amd.context import Failed
from test_attn_batch_gpu import Batch, run
from test_moe_use_gpu import Graph

pytestmark = pytest.mark.gpu
YARN = RopeScaling.yarn(64, 4096, 150000.0, 32.0)


class Layer:
    """Append and attention of one layer's ragged batch, with a cache of earlier tokens and a workspace of its own."""

    def __init__(self, cx, new, cached, seed, heads=16, kv_heads=2, dim=64, page=16, out_type=OUT_F16, window=0):
        rng = np.random.default_rng(seed)
        self.cx, self.heads, self.kv_heads, self.dim, self.page, self.out_type, self.window = cx, heads, kv_heads, dim, page, out_type, window
        self.new, self.n_kv = list(new), np.add(new, cached).tolist()
        self.rows = np.concatenate([[0], np.cumsum(new)]).astype(np.uint32)
        n = int(self.rows[-1])
        counts = [-(-k // page) for k in self.n_kv]
        self.n_pages, self.stride = sum(counts), max(counts)
        ids, at = rng.permutation(self.n_pages), 0
        self.tables = np.zeros((len(new), self.stride), np.uint32)
        for b, c in enumerate(counts):
            self.tables[b, :c] = ids[at:at + c]
            at += c
        self.pools = [rng.standard_normal((self.n_pages, page, kv_heads, dim)).astype(np.float16) for _ in range(2)]
        self.qkv = rng.standard_normal((n, (heads + 2 * kv_heads) * dim)).astype(np.float32)
        self.bk, self.bv = (cx.upload(p) for p in self.pools)
        self.bx, self.bt, self.bs = cx.upload(self.qkv), cx.upload(self.tables), cx.upload(rng.standard_normal(heads).astype(np.float32))
        self.bq, self.bo = cx.alloc(n * heads * dim * 2), cx.alloc(n * heads * dim * 4)
        width, k_at, v_at = self.qkv.shape[1], heads * dim * 4, (heads + kv_heads) * dim * 4
        self.desc = QkvAppendDesc.make(self.bx, DeviceView(self.bx, k_at), DeviceView(self.bx, v_at), self.bq, self.bk, self.bv, self.n_pages,
                                       heads, kv_heads, dim, page, dim, 150000.0, YARN, q_stride=width, k_stride=width, v_stride=width)
        self.ws = cx.alloc(max(16, cx.attn_prefill_batched_workspace(self.rows, self.n_kv, window, heads, kv_heads, dim)))

    def append(self):
        self.cx.rope_qkv_append_batched(self.desc, self.bt, self.stride, self.rows, self.n_kv)

    def attend(self, ws=True):
        self.cx.attn_prefill_batched(self.bo, self.bq, self.bk, self.bv, self.n_pages, self.bt, self.stride, self.rows, self.n_kv, self.bs,
                                     self.window, self.heads, self.kv_heads, self.dim, self.page, self.dim ** -0.5, out_type=self.out_type,
                                     workspace=self.ws if ws else None)

    def run(self, ws=True):
        self.append()
        self.attend(ws)

    def reset(self):
        self.cx.upload_slice(self.bk, self.pools[0])
        self.cx.upload_slice(self.bv, self.pools[1])
        self.cx.zero(self.bo, self.bo.len // 4)

    def out(self):
        kind = np.float16 if self.out_type == OUT_F16 else np.float32
        return self.cx.download(self.bo, kind, (int(self.rows[-1]), self.heads, self.dim))


def test_decode_rows_are_decode_calls():
    # new tokens of one: append and attention against moearc_rope_kv_append's places and moearc_attn_decode over the same cache
    with Context() as cx:
        s = Layer(cx, [1, 1, 1], [700, 0, 33], 1, out_type=OUT_F32)
        s.run()
        got = s.out()
        q = cx.download(s.bq, np.float16, got.shape).astype(np.float32)
        out, bq = cx.alloc(got[0].nbytes), cx.alloc(got[0].nbytes)
        for b, n in enumerate(s.n_kv):
            cx.upload_slice(bq, q[b])
            cx.attn_decode_ext(out, bq, s.bk, s.bv, cx.upload(s.tables[b]), s.bs, s.heads, s.kv_heads, s.dim, 0, n, s.page, s.dim ** -0.5, KvType.F16)
            want = cx.download(out, np.float32, got[0].shape)
            # both within 2^-20 of values up to 4: weights to 2^-22 of them, sums of up to 701 terms in f32
            assert np.abs(got[b] - want).max() <= 2 * 4 * 2.0 ** -18


@pytest.mark.parametrize("window", [0, 50])
def test_one_chunk_is_the_prefill_call(window):
    with Context() as cx:
        s = Layer(cx, [200], [300], 2, window=window)
        s.run()
        got = s.out().astype(np.float64)
        out = cx.alloc(s.bo.len)
        cx.attn_prefill(out, s.bq, s.bk, s.bv, s.bt, s.bs, 200, 300, window, s.heads, s.kv_heads, s.dim, s.page, s.dim ** -0.5, out_type=OUT_F16)
        want = cx.download(out, np.float16, got.shape).astype(np.float64)
        # both round weights to f16 (2^-11 of sum w|v - out| <= 4 each) and the output (2^-11 of at most 4)
        assert np.abs(got - want).max() <= 4 * 4 * 2.0 ** -11


@pytest.mark.parametrize("new,cached,dim,out_type", [
    ([1, 1, 1], [3000, 10, 500], 64, OUT_F16), ([3, 7, 0, 90], [2000, 100, 50, 600], 128, OUT_F32), ([130, 1], [0, 4000], 96, OUT_F16)], ids=str)
def test_replays_equal_eager_calls(new, cached, dim, out_type):
    """Captured and replayed between eager calls of other sizes that grow the context's own workspace."""
    with Context() as cx:
        a, other = Layer(cx, new, cached, 3, dim=dim, out_type=out_type), Layer(cx, [1, 300], [9000, 1000], 4, dim=dim)
        a.run()
        want, cache = a.out(), cx.download(a.bk, np.float16, a.pools[0].shape)
        other.run(False)
        want_other = other.out()
        g = Graph(cx, a.run)
        for _ in range(4):
            a.reset()
            g.launch()
            assert np.array_equal(a.out(), want) and np.array_equal(cx.download(a.bk, np.float16, cache.shape), cache)
            other.reset()
            other.run(False)
            assert np.array_equal(other.out(), want_other)
        # replays see the data of their time: other rows, same buffers
        cx.upload_slice(a.bx, np.roll(a.qkv, 1, axis=1))
        a.reset()
        a.run()
        want = a.out()
        a.reset()
        g.launch()
        assert np.array_equal(a.out(), want)
        g.close()


def test_a_captured_call_that_is_cut_needs_a_workspace():
    with Context() as cx:
        s = Layer(cx, [1], [5000], 5)
        s.run()
        want, n_kv = s.out(), np.array(s.n_kv, np.uint32)

        def go():
            # (not through the wrapper, which waits for the stream before it reports an error)
            assert cx._lib.moearc_attn_prefill_batched(
                cx.raw, s.bo.ptr, s.out_type, s.bq.ptr, s.bk.ptr, s.bv.ptr, s.n_pages, s.bt.ptr, s.stride, s.rows.ctypes.data,
                n_kv.ctypes.data, s.bs.ptr, 1, 0, s.heads, s.kv_heads, s.dim, s.page, s.dim ** -0.5, 1, None, 0) == -1
            s.attend()
        g = Graph(cx, go)
        s.cx.zero(s.bo, s.bo.len // 4)
        g.launch()
        assert np.array_equal(s.out(), want)
        g.close()


def test_a_replay_reports_a_page_outside_the_pool():
    with Context() as cx:
        s = Layer(cx, [3, 20], [100, 50], 6)
        s.run()
        g = Graph(cx, s.run)
        bad = s.tables.copy()
        bad[1, 4] = s.n_pages
        for tables, fails in ((s.tables, False), (bad, True), (s.tables, False), (bad, True)):
            cx.upload_slice(s.bt, tables)
            g.launch()
            if fails:
                with pytest.raises(Failed):
                    cx.sync()
            cx.sync()
        g.close()


def test_two_contexts_at_once():
    with Context() as c1, Context() as c2:
        layers = [Layer(c1, [1, 60], [3000, 10], 7, dim=128), Layer(c2, [1, 60], [3000, 10], 8, dim=128), Layer(c1, [5], [2000], 9),
                  Layer(c2, [2, 2, 2], [800, 90, 1], 10)]
        want = []
        for x in layers:
            x.run(False)
            want.append(x.out())
            x.reset()
        c1.sync()
        c2.sync()
        for x in layers:
            x.run(False)
        for x, w in zip(layers, want):
            assert np.array_equal(x.out(), w)


def test_a_window_over_a_ring():
    """Chunks of two sequences through rings of four pages: the same rows as over caches that keep every token."""
    window, page, ring, heads, kv_heads, dim = 20, 8, 4, 4, 2, 64
    rng = np.random.default_rng(11)
    with Context() as cx:
        pages = 16
        shape = (2 * pages, page, kv_heads, dim)
        full = np.arange(2 * pages, dtype=np.uint32).reshape(2, pages)
        rings = np.stack([np.arange(pages) % ring, ring + np.arange(pages) % ring]).astype(np.uint32)
        pools = [[cx.upload(np.zeros(shape, np.float16)) for _ in range(2)] for _ in range(2)]
        at = [0, 0]
        for step in range(9):
            new = [int(rng.integers(0, ring * page - window + 2)) for _ in range(2)]
            if step == 4:
                new = [1, ring * page - window + 1]
            new = [min(n, pages * page - a) for n, a in zip(new, at)]
            at = [a + n for a, n in zip(at, new)]
            rows, n = np.concatenate([[0], np.cumsum(new)]), sum(new)
            if n == 0:
                continue
            x = [cx.upload(rng.standard_normal((n, h, dim)).astype(np.float32)) for h in (heads, kv_heads, kv_heads)]
            outs = []
            for tables, (k, v) in ((full, pools[0]), (rings, pools[1])):
                q, out, bt = cx.alloc(n * heads * dim * 2), cx.alloc(n * heads * dim * 4), cx.upload(tables)
                d = QkvAppendDesc.make(*x, q, k, v, 2 * pages, heads, kv_heads, dim, page, dim, 1e4)
                cx.rope_qkv_append_batched(d, bt, pages, rows, at)
                cx.attn_prefill_batched(out, q, k, v, 2 * pages, bt, pages, rows, at, None, window, heads, kv_heads, dim, page, 0.125)
                outs.append(cx.download(out, np.float32, (n, heads, dim)))
            assert np.array_equal(outs[0], outs[1]), step


@pytest.mark.parametrize("dim,out_type", [(64, OUT_F16), (128, OUT_F32)])
def test_offsets_beyond_32_bits(dim, out_type):
    """Pools of more than 2^32 bytes whose last pages hold everything."""
    with Context() as cx:
        page, kv_heads, heads = 256, 8, 16
        row = kv_heads * dim * 2
        n_pages = (1 << 32) // (page * row) + 40
        s = Batch([40, 1], [500, 900], heads, kv_heads, dim, page, 12)
        want = run(cx, s, out_type=out_type)
        pools = [cx.alloc(n_pages * page * row) for _ in range(2)]
        first = n_pages - s.n_pages
        for pool, x in zip(pools, (s.k, s.v)):
            cx.upload_slice(DeviceView(pool, first * page * row), x)
        tables = np.where(s.tables == 0xFFFFFFFF, s.tables, s.tables + np.uint32(first))
        out, bt = cx.alloc(want.nbytes), cx.upload(tables)
        q = cx.upload(s.q)
        cx.attn_prefill_batched(out, q, *pools, n_pages, bt, s.stride, s.rows, s.n_kv, cx.upload(s.sinks), 0, heads, kv_heads, dim, page,
                                dim ** -0.5, out_type=out_type)
        cx.sync()
        assert np.array_equal(cx.download(out, want.dtype, want.shape), want)
        # the same places take new tokens: f16 rows, unrotated in their last half, so V and that half of K come back as they are
        n = s.n_rows
        x = [np.random.default_rng(13 + i).standard_normal((n, h, dim)).astype(np.float16) for i, h in enumerate((heads, kv_heads, kv_heads))]
        d = QkvAppendDesc.make(*(cx.upload(a) for a in x), cx.alloc(n * heads * dim * 2), *pools, n_pages, heads, kv_heads, dim, page, dim // 2, 1e4,
                               in_type=OUT_F16)
        cx.rope_qkv_append_batched(d, bt, s.stride, s.rows, s.n_kv)
        cx.sync()
        got = [cx.download(DeviceView(p, first * page * row), np.float16, s.k.shape) for p in pools]
        for b, (m, kv) in enumerate(zip(s.new, s.n_kv)):
            for i in range(m):
                p, r = kv - m + i, int(s.rows[b]) + i
                to = s.tables[b, p // page], p % page
                assert np.array_equal(got[1][to], x[2][r]) and np.array_equal(got[0][to][:, dim // 2:], x[1][r][:, dim // 2:])
