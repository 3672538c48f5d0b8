"""Attention of a ragged batch (moearc_attn_prefill_batched) against float64.

Bounds, u = 2^-24, per row of n visible keys: a score is a sum of D exact products in f32, off by at most D u sum|q k|
times the scale, its exponent's argument rounds four times, and the weight is off by r of itself (2^-11 rounded to
f16, 2^-22 as hi + lo) and by 2^-32 of the row's largest. The sums of weights and of weighted values see the same weights, so
an error e of the weights moves the result by at most e sum w|v - out| (the sink counts as a value of zero); the f32
sums add (n + 8) u sum w|v|, the output half a step of its type."""
from __future__ import annotations

import numpy as np
import pytest

from moearc_amd import OUT_F16, OUT_F32, BadArgument, Context
from moearc_amd.context import Failed

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture(scope="module")
def cx():
    with Context() as c:
        yield c


class Batch:
    """new[b] tokens behind the others of n_kv[b] keys, in pages scattered over a pool with one page to spare."""

    def __init__(self, new, n_kv, heads, kv_heads, dim, page, seed, sinks=True, spare_rows=0):
        rng = np.random.default_rng(seed)
        self.new, self.n_kv, self.heads, self.kv_heads, self.dim, self.page = list(new), list(n_kv), heads, kv_heads, dim, page
        self.rows = np.concatenate([[0], np.cumsum(new)]).astype(np.uint32) + np.uint32(spare_rows)
        self.n_rows = int(self.rows[-1])
        counts = [-(-n // page) for n in n_kv]
        self.n_pages, self.stride = sum(counts) + 1, max(counts + [1])
        ids = rng.permutation(self.n_pages)[:sum(counts)]
        self.tables = np.full((len(new), self.stride), 0xFFFFFFFF, np.uint32)  # entries that nobody may look at
        at = 0
        for b, c in enumerate(counts):
            self.tables[b, :c] = ids[at:at + c]
            at += c
        shape = (self.n_pages, page, kv_heads, dim)
        self.k, self.v = (rng.standard_normal(shape).astype(np.float16) for _ in range(2))
        self.q = rng.standard_normal((self.n_rows, heads, dim)).astype(np.float16)
        self.sinks = rng.standard_normal(heads).astype(np.float32) if sinks else None
        for b, n in enumerate(n_kv):  # what lies behind a sequence's last key must not be read
            if counts[b] and n % page:
                self.k[self.tables[b, counts[b] - 1], n % page:] = np.nan
                self.v[self.tables[b, counts[b] - 1], n % page:] = np.nan
        spare = [i for i in range(self.n_pages) if i not in set(ids.tolist())]
        self.k[spare], self.v[spare] = np.nan, np.nan

    def keys(self, b, h, lo, hi):
        j = np.arange(lo, hi)
        at = self.tables[b, j // self.page].astype(np.int64), j % self.page
        return self.k[at][:, h].astype(np.float64), self.v[at][:, h].astype(np.float64)

    def expected(self, window, scale, out_type):
        """(out, bound) of the rows, float64; rows before the first sequence are NaN."""
        out, tol = (np.full((self.n_rows, self.heads, self.dim), np.nan) for _ in range(2))
        r = 2.0 ** -11 if out_type == OUT_F16 else 2.0 ** -22
        for b, (m, n) in enumerate(zip(self.new, self.n_kv)):
            if m == 0:
                continue
            p = np.arange(n - m, n)[:, None]
            first = max(0, n - m + 1 - window) if window else 0
            j = np.arange(first, n)
            sees = (j <= p) & ((p - j < window) if window else True) & (p >= 0)
            count = sees.sum(1)[:, None]
            at = slice(int(self.rows[b]), int(self.rows[b]) + m)
            for h in range(self.heads):
                k, v = self.keys(b, h * self.kv_heads // self.heads, first, n)
                q = self.q[at, h].astype(np.float64)
                s = np.where(sees, scale * (q @ k.T), -np.inf)
                size = np.where(sees, abs(scale) * (np.abs(q) @ np.abs(k).T), 0).max(1, initial=0)[:, None]
                sink = self.sinks[h] if self.sinks is not None else -np.inf
                top = np.maximum(s.max(1, initial=-np.inf), sink)[:, None]
                top = np.where(np.isfinite(top), top, 0)
                w = np.exp(s - top)
                total = w.sum(1, keepdims=True) + np.exp(sink - top)
                w = w / np.where(total == 0, 1, total)
                o, mass = w @ v, w.sum(1, keepdims=True)
                e = (self.dim + 8) * U * size + 8 * U * (np.abs(np.where(sees, s, 0)).max(1, initial=0)[:, None] + np.abs(top) + 16) + r
                # sum w|v - out| <= sqrt(sum w sum w (v - out)^2)
                spread = np.sqrt(mass * np.maximum(0, w @ (v * v) - 2 * o * o + o * o * mass)) + (1 - mass) * np.abs(o)
                bound = 1.01 * e * spread + (count + 8) * U * (w @ np.abs(v)) + count * 2.0 ** -31 * np.abs(v).max(initial=0)
                step = 2.0 ** -11 * np.abs(o) + 2.0 ** -25 if out_type == OUT_F16 else U * np.abs(o)
                out[at, h], tol[at, h] = o, np.where(count > 0, bound + 1.01 * step, 0)
        return out, tol


def run(cx, s, window=0, scale=None, out_type=OUT_F16, q=None, workspace=None, extra=3):
    """The outputs; rows of no sequence (before the first, `extra` behind the last) have to stay as they were."""
    scale = s.dim ** -0.5 if scale is None else scale
    kind = np.float16 if out_type == OUT_F16 else np.float32
    before = np.full((s.n_rows + extra, s.heads, s.dim), 77.0, kind)
    out = cx.upload(before)
    up = cx.upload
    bufs = [up(s.q if q is None else q), up(s.k), up(s.v), up(s.tables), up(s.sinks) if s.sinks is not None else None]
    cx.attn_prefill_batched(out, bufs[0], bufs[1], bufs[2], s.n_pages, bufs[3], s.stride, s.rows, s.n_kv, bufs[4], window,
                            s.heads, s.kv_heads, s.dim, s.page, scale, out_type=out_type, workspace=workspace)
    cx.sync()
    got = cx.download(out, kind, before.shape)
    first = int(s.rows[0])
    assert (got[:first] == 77).all() and (got[s.n_rows:] == 77).all()
    return got[:s.n_rows]


def check(cx, s, window=0, scale=None, out_type=OUT_F16):
    got = run(cx, s, window, scale, out_type)
    want, tol = s.expected(window, s.dim ** -0.5 if scale is None else scale, out_type)
    first = int(s.rows[0])
    err = np.abs(got[first:].astype(np.float64) - want[first:])
    assert np.isfinite(got[first:]).all() and (err <= tol[first:]).all(), (err - tol[first:]).max()


@pytest.mark.parametrize("out_type", [OUT_F16, OUT_F32], ids=["f16", "f32"])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [
    (8, 1, 64, 16), (4, 4, 64, 48), (16, 2, 128, 32), (5, 1, 80, 7), (6, 2, 96, 1), (14, 2, 8, 64), (2, 1, 136, 16),
    (4, 2, 256, 33), (3, 3, 24, 300)], ids=str)
def test_shapes(cx, heads, kv_heads, dim, page, out_type):
    new, cached = [1, 0, 5, 33, 2, 70], [0, 9, 31, 1, 260, 64]
    check(cx, Batch(new, np.add(new, cached), heads, kv_heads, dim, page, dim + page), out_type=out_type)


@pytest.mark.parametrize("n_kv", [32, 64, 96, 128, 160, 192, 224, 256, 288, 320, 321, 351])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_spans_of_whole_tiles(cx, dim, n_kv):
    # what is copied ahead ends where the keys do
    check(cx, Batch([20, 1], [n_kv, n_kv], 8, 1, dim, 32, n_kv), out_type=OUT_F32)


@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 100, 1000])
@pytest.mark.parametrize("dim", [64, 128])
def test_windows(cx, window, dim):
    new, cached = [1, 40, 3, 150], [300, 0, 64, 70]
    check(cx, Batch(new, np.add(new, cached), 8, 2, dim, 16, window), window, out_type=OUT_F32)


@pytest.mark.parametrize("scale", [0.0, 1e-30, -0.2, 1.0, 3.0])
def test_scales(cx, scale):
    new, cached = [3, 17], [40, 5]
    check(cx, Batch(new, np.add(new, cached), 4, 2, 64, 16, 3), scale=scale, out_type=OUT_F32)


@pytest.mark.parametrize("sinks", [False, True])
def test_rows_that_see_nothing(cx, sinks):
    # fewer keys than new tokens: the first rows sit at negative positions
    check(cx, Batch([5, 3, 40], [2, 0, 7], 8, 2, 64, 16, 5, sinks), out_type=OUT_F32)
    check(cx, Batch([5, 3, 40], [2, 0, 7], 8, 2, 128, 16, 5, sinks), 3)


def test_many_sequences_and_rows_of_none(cx):
    # more than a launch carries, every third without new tokens; rows before the first sequence
    rng = np.random.default_rng(8)
    new = [0 if b % 3 == 2 else int(rng.integers(1, 4)) for b in range(150)]
    check(cx, Batch(new, np.add(new, rng.integers(0, 50, 150)), 4, 1, 64, 16, 9, spare_rows=4))


def test_one_token_behind_many(cx):
    # cut into pieces and merged
    new, cached = [1, 2, 1], [5000, 1, 700]
    for dim, out_type in ((64, OUT_F32), (128, OUT_F16), (256, OUT_F32)):
        check(cx, Batch(new, np.add(new, cached), 4, 1, dim, 16, dim), out_type=out_type)


def test_pages_of_one_token_beyond_a_table_segment(cx):
    check(cx, Batch([2], [2600], 2, 1, 64, 1, 4), out_type=OUT_F32)


@pytest.mark.parametrize("dim", [64, 128])
def test_scores_that_grow(cx, dim):
    # each key outweighs the ones before it, and then falls off: the running reference moves again and again
    s = Batch([70], [300], 4, 1, dim, 16, 6)
    size = np.concatenate([np.linspace(0, 8, 200), np.linspace(8, 0, 100)])
    for j in range(300):
        s.k[s.tables[0, j // 16], j % 16] = (np.sign(s.q[60, 0]) * size[j] * 0.25).astype(np.float16)
    check(cx, s, out_type=OUT_F32)


@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("dim,window", [(64, 0), (128, 0), (128, 20)])
def test_values_of_unseen_keys(cx, bad, dim, window):
    # a key with such a value, and one such key: rows that do not see them are as without them
    s = Batch([50, 30], [60, 90], 4, 2, dim, 16, 7, sinks=False)
    clean = run(cx, s, window)
    for b, j in ((0, 40), (1, 75)):
        s.v[s.tables[b, j // 16], j % 16, :, 3] = bad
        s.k[s.tables[b, (j + 9) // 16], (j + 9) % 16, :, 1] = bad
    got = run(cx, s, window)
    for b, j in ((0, 40), (1, 75)):
        for i in range(s.new[b]):
            p, row = s.n_kv[b] - s.new[b] + i, int(s.rows[b]) + i
            unseen = [p < x or (window and p - x >= window) for x in (j, j + 9)]
            if all(unseen):
                err = np.abs(got[row].astype(np.float64) - clean[row])
                assert (err <= 2.0 ** -9 * np.abs(clean[row]) + 2.0 ** -14).all(), (b, i)
            elif not unseen[0] and unseen[1]:  # the one value is lost, the others stand
                assert not np.isfinite(got[row, :, 3]).any()
                assert np.isfinite(np.delete(got[row], 3, -1)).all()


def test_results_repeat(cx):
    new, cached = [1, 200, 7], [3000, 100, 0]
    s = Batch(new, np.add(new, cached), 8, 2, 128, 16, 11)
    first = run(cx, s)
    for _ in range(3):
        assert (run(cx, s) == first).all()


def test_a_page_outside_the_pool(cx):
    s = Batch([2, 3], [40, 50], 4, 2, 64, 16, 12)
    s.tables[1, 1] = s.n_pages
    with pytest.raises(Failed):
        run(cx, s)
    s.tables[1, 1] = 0
    run(cx, s)  # reported once


def test_workspace_of_the_caller(cx):
    new, cached = [1, 4], [4000, 2000]
    s = Batch(new, np.add(new, cached), 8, 1, 128, 16, 13)
    n = cx.attn_prefill_batched_workspace(s.rows, s.n_kv, 0, 8, 1, 128)
    assert n > 0
    ws = cx.alloc(n)
    assert (run(cx, s, workspace=ws) == run(cx, s)).all()
    with pytest.raises(BadArgument):
        run(cx, s, workspace=cx.alloc(n - 16))
