"""Attention of a ragged batch (moearc_attn_prefill_batched) where one work-group's keys have more places than its table
holds at a time, so that it goes over them in segments. The sequences of a batch share their pages, and there are enough of
them that no tile is cut into pieces, which the workspace of 0 bytes shows. Bounds as in test_attn_batch_gpu.py."""
from __future__ import annotations

import copy

import numpy as np
import pytest

from moearc_amd import OUT_F16, OUT_F32, Context
from test_attn_batch_gpu import Batch, run

pytestmark = pytest.mark.gpu
KV_HEADS = {64: 12, 128: 8, 256: 4}  # of 64 sequences: a work-group for each place of 256 CUs, in tiles of either kind
ODD = 2016, 2044, 2045, 2076, 4100   # keys of pages of no multiple of eight tokens
EIGHTS = 16129, 16400, 33000


@pytest.fixture(scope="module")
def cx():
    with Context() as c:
        yield c


class Shared(Batch):
    """64 sequences with `new` tokens each, the last of the same n_kv keys."""

    def __init__(self, new, n_kv, group, dim, page, seed):
        rng = np.random.default_rng(seed)
        self.new, self.n_kv, self.kv_heads, self.dim, self.page = [new] * 64, [n_kv] * 64, KV_HEADS[dim], dim, page
        self.heads = group * self.kv_heads
        self.rows = (new * np.arange(65)).astype(np.uint32)
        self.n_rows = 64 * new
        count = -(-n_kv // page)
        self.n_pages, self.stride = count + 1, count
        ids = rng.permutation(self.n_pages)
        self.tables = np.tile(ids[:count].astype(np.uint32), (64, 1))
        shape = (self.n_pages, page, self.kv_heads, dim)
        self.k, self.v = (rng.standard_normal(shape, np.float32).astype(np.float16) for _ in range(2))
        # heavier keys where segments may end, so that one that enters twice or not at all moves the rows far
        for j in range(n_kv):
            if (j + 8) % 2016 < 16 or (j + 8) % 2044 < 16 or (j + 8) % 2048 < 16:
                self.k[ids[j // page], j % page] *= np.float16(2)
        self.k[ids[count]], self.v[ids[count]] = np.nan, np.nan
        if n_kv % page:  # what lies behind the last key must not be read
            self.k[ids[count - 1], n_kv % page:] = np.nan
            self.v[ids[count - 1], n_kv % page:] = np.nan
        self.q = rng.standard_normal((self.n_rows, self.heads, dim), np.float32).astype(np.float16)
        self.sinks = rng.standard_normal(self.heads).astype(np.float32)

    def part(self, b, h):
        """Sequence b and KV head h alone."""
        p, g = copy.copy(self), self.heads // self.kv_heads
        rows = slice(int(self.rows[b]), int(self.rows[b + 1]))
        p.new, p.n_kv, p.heads, p.kv_heads, p.tables = self.new[b:b + 1], self.n_kv[b:b + 1], g, 1, self.tables[b:b + 1]
        p.rows, p.n_rows = np.array([0, self.new[b]], np.uint32), self.new[b]
        p.k, p.v, p.q, p.sinks = self.k[:, :, h:h + 1], self.v[:, :, h:h + 1], self.q[rows, h * g:(h + 1) * g], self.sinks[h * g:(h + 1) * g]
        return p, rows, slice(h * g, (h + 1) * g)


def check(cx, s, window=0, out_type=OUT_F32):
    assert cx.attn_prefill_batched_workspace(s.rows, s.n_kv, window, s.heads, s.kv_heads, s.dim) == 0
    got = run(cx, s, window, out_type=out_type)
    assert np.isfinite(got).all()
    for b, h in ((0, 0), (63, s.kv_heads - 1)):
        p, rows, heads = s.part(b, h)
        want, tol = p.expected(window, s.dim ** -0.5, out_type)
        err = np.abs(got[rows, heads].astype(np.float64) - want)
        assert (err <= tol).all(), (b, h, (err - tol).max())
    return got


@pytest.mark.parametrize("new,group", [(64, 2), (1, 8)], ids=["full", "small"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page", [1, 7, 20, 100])
def test_odd_pages(cx, page, dim, new, group):
    for n_kv in ODD:
        check(cx, Shared(new, n_kv, group, dim, page, n_kv + page))


@pytest.mark.parametrize("new,group", [(64, 2), (1, 8)], ids=["full", "small"])
@pytest.mark.parametrize("n_kv", EIGHTS)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_pages_of_eights(cx, dim, n_kv, new, group):
    check(cx, Shared(new, n_kv, group, dim, 48, n_kv))


@pytest.mark.parametrize("new,group", [(64, 2), (5, 8)], ids=["full", "small"])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_f16_outputs_and_windows(cx, dim, new, group):
    check(cx, Shared(new, 4100, group, dim, 7, 1), out_type=OUT_F16)
    check(cx, Shared(new, 5000, group, dim, 7, 2), 3001, out_type=OUT_F16)
    check(cx, Shared(new, 5000, group, dim, 9, 3), 2045)


@pytest.mark.parametrize("new,group", [(64, 2), (5, 8)], ids=["full", "small"])
@pytest.mark.parametrize("dim,page,n_kv", [(64, 7, 4500), (128, 20, 4500), (256, 1, 2100), (128, 48, 16500)], ids=str)
def test_values_of_unseen_keys(cx, dim, page, n_kv, new, group):
    # an infinity that only the last two rows of a sequence see: the work-group goes over all segments twice
    s = Shared(new, n_kv, group, dim, page, 5)
    parts = [(s.part(b, h), (b, h)) for b, h in ((0, 0), (63, s.kv_heads - 1))]
    wants = [p.expected(0, dim ** -0.5, OUT_F32) for (p, _, _), _ in parts]
    j = n_kv - 2
    s.v[s.tables[0, j // page], j % page, :, 3] = np.inf
    assert cx.attn_prefill_batched_workspace(s.rows, s.n_kv, 0, s.heads, s.kv_heads, s.dim) == 0
    got = run(cx, s, out_type=OUT_F32)
    ends = got.reshape(64, new, s.heads, dim)
    assert not np.isfinite(ends[:, -2:, :, 3]).any()
    assert np.isfinite(np.delete(ends, 3, -1)).all() and np.isfinite(ends[:, :-2]).all()
    for ((_, rows, heads), at), (want, tol) in zip(parts, wants):  # the other rows, and the other channels of the two
        err = np.abs(got[rows, heads].astype(np.float64) - want)
        assert (err <= tol)[:-2].all() and (np.delete(err, 3, -1) <= np.delete(tol, 3, -1)).all(), at
