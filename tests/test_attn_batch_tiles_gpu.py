"""Attention of a ragged batch on full tiles (moearc_attn_prefill_batched): batches whose tiles of 128 rows give most CUs work,
or rows and keys past what small tiles take. Bounds as in test_attn_batch_gpu.py."""
from __future__ import annotations

import numpy as np
import pytest

from moearc_amd import OUT_F16, OUT_F32, Context
from test_attn_batch_gpu import Batch, check, run

pytestmark = pytest.mark.gpu
ALONE = [70, 0, 130, 65]  # tokens of 64 KV heads with a query head each: tiles 1 + 2 + 1
GROUPS = [30, 1, 50]      # of 44 KV heads with three each: 90, 3 and 150 rows, tiles 1 + 2


@pytest.fixture(scope="module")
def cx():
    with Context() as c:
        yield c


@pytest.mark.parametrize("out_type", [OUT_F16, OUT_F32], ids=["f16", "f32"])
@pytest.mark.parametrize("dim,page", [(64, 16), (64, 7), (128, 48), (128, 1), (80, 32), (256, 24), (200, 9), (8, 64)], ids=str)
def test_shapes(cx, dim, page, out_type):
    check(cx, Batch(ALONE, np.add(ALONE, [0, 9, 31, 260]), 64, 64, dim, page, dim + page), out_type=out_type)
    check(cx, Batch(GROUPS, np.add(GROUPS, [64, 300, 5]), 132, 44, dim, page, dim + page + 1), out_type=out_type)


@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 100, 1000])
@pytest.mark.parametrize("dim", [64, 128])
def test_windows(cx, window, dim):
    check(cx, Batch(ALONE, np.add(ALONE, [300, 0, 64, 70]), 64, 64, dim, 16, window), window, out_type=OUT_F32)


@pytest.mark.parametrize("n_kv", [128, 160, 192, 224, 256, 288, 320, 321, 351])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_spans_of_whole_tiles(cx, dim, n_kv):
    # what is copied ahead ends where the keys do
    check(cx, Batch([66, 128], [n_kv, n_kv], 64, 64, dim, 32, n_kv), out_type=OUT_F32)


@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0])
def test_scales(cx, scale):
    check(cx, Batch(GROUPS, np.add(GROUPS, [40, 5, 9]), 132, 44, 64, 16, 3), scale=scale, out_type=OUT_F32)


def test_rows_that_see_nothing(cx):
    for sinks in (False, True):
        check(cx, Batch([70, 66, 130], [2, 0, 77], 64, 64, 128, 16, 5, sinks))
    check(cx, Batch([70, 66, 130], [2, 0, 77], 64, 64, 64, 16, 5, False), 3, out_type=OUT_F32)


@pytest.mark.parametrize("dim,out_type", [(64, OUT_F32), (128, OUT_F16), (256, OUT_F32), (96, OUT_F32)])
def test_cut_tiles(cx, dim, out_type):
    # more than 256 rows and 2560 keys, few work-groups: cut and merged; a window's last rows and the first's are not
    check(cx, Batch([40, 3], [3001, 50], 8, 1, dim, 16, dim), out_type=out_type)
    check(cx, Batch([300], [2900], 2, 1, dim, 24, dim), 2700, out_type=out_type)


@pytest.mark.parametrize("dim", [64, 128])
def test_scores_that_grow(cx, dim):
    # each key outweighs the ones before it, and then falls off: the running reference moves again and again
    s = Batch([70, 70], [300, 300], 64, 64, dim, 16, 6)
    size = np.concatenate([np.linspace(0, 8, 200), np.linspace(8, 0, 100)])
    for j in range(300):
        s.k[s.tables[0, j // 16], j % 16] = (np.sign(s.q[60, 0]) * size[j] * 0.25).astype(np.float16)
    check(cx, s, out_type=OUT_F32)


@pytest.mark.parametrize("bad", [np.inf, np.nan])
@pytest.mark.parametrize("dim,window", [(64, 0), (128, 0), (128, 20)])
def test_values_of_unseen_keys(cx, bad, dim, window):
    s = Batch([150, 80], [160, 190], 44, 44, dim, 16, 7, sinks=False)
    clean = run(cx, s, window)
    marks = (0, 90), (1, 150)
    for b, j in marks:
        s.v[s.tables[b, j // 16], j % 16, :, 3] = bad
    got = run(cx, s, window)
    for b, j in marks:
        for i in range(s.new[b]):
            p, row = s.n_kv[b] - s.new[b] + i, int(s.rows[b]) + i
            if p < j or (window and p - j >= window):
                err = np.abs(got[row].astype(np.float64) - clean[row])
                assert (err <= 2.0 ** -9 * np.abs(clean[row]) + 2.0 ** -14).all(), (b, i)
            else:
                assert not np.isfinite(got[row, :, 3]).any() and np.isfinite(np.delete(got[row], 3, -1)).all()


def test_results_repeat(cx):
    s = Batch([40, 300], [3001, 400], 8, 1, 128, 16, 11)
    first = run(cx, s)
    for _ in range(3):
        assert (run(cx, s) == first).all()
