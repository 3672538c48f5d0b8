"""The ragged batches' calls at the ends of their ranges: launches that share one workspace, as many heads as a call
takes, sinks that are nothing, rows around whole tiles. Bounds as in test_attn_batch_gpu.py."""
from __future__ import annotations

import numpy as np
import pytest

from moearc_amd import OUT_F16, OUT_F32, Context
from test_attn_batch_gpu import Batch, check, run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def cx():
    with Context() as c:
        yield c


def test_launches_that_share_a_workspace(cx):
    # three launches, the first two cut into pieces, whose records lie in the same memory one after the other
    rng = np.random.default_rng(21)
    new, n_kv = [1] * 140, rng.integers(1, 60, 140)
    n_kv[[10, 40, 100]] = 4000, 3100, 2500
    s = Batch(new, n_kv, 4, 1, 64, 16, 21)
    need = cx.attn_prefill_batched_workspace(s.rows, s.n_kv, 0, 4, 1, 64)
    parts = [cx.attn_prefill_batched_workspace(s.rows[a:b + 1], s.n_kv[a:b], 0, 4, 1, 64) for a, b in ((0, 64), (64, 128), (128, 140))]
    assert min(parts[:2]) > 0 == parts[2] and need == max(parts)
    ws = cx.alloc(need + 256)
    cx.upload_slice(ws, np.full(need // 4 + 64, 77.0, np.float32))
    got = run(cx, s, out_type=OUT_F32, workspace=ws)
    assert np.array_equal(got, run(cx, s, out_type=OUT_F32))
    assert (cx.download(ws, np.float32, (need // 4 + 64,))[need // 4:] == 77).all()
    want, tol = s.expected(0, 0.125, OUT_F32)
    assert (np.abs(got - want) <= tol).all()


@pytest.mark.parametrize("heads,kv_heads,dim", [(1024, 1, 8), (1024, 1024, 8), (1024, 512, 16), (1000, 8, 64), (1024, 2, 128)], ids=str)
def test_many_heads(cx, heads, kv_heads, dim):
    check(cx, Batch([2, 1], [40, 9], heads, kv_heads, dim, 16, heads + kv_heads), out_type=OUT_F32)


@pytest.mark.parametrize("n_kv", [[40, 3], [2600, 3]], ids=["whole", "cut"])
def test_sinks_of_minus_infinity(cx, n_kv):
    s = Batch([2, 5], n_kv, 8, 1, 64, 16, 23)  # two rows of the second sequence see nothing
    s.sinks[:5] = -np.inf
    check(cx, s, out_type=OUT_F32)
    s.sinks[:] = -np.inf
    bare = Batch([2, 5], n_kv, 8, 1, 64, 16, 23)
    bare.sinks = None
    assert np.array_equal(run(cx, s), run(cx, bare))


@pytest.mark.parametrize("rows", [32, 33, 64, 65, 128, 129, 256, 257])
def test_rows_around_the_tiles(cx, rows):
    # as many rows as a tile has, and one more; beside a sequence that keeps the device busy, and alone
    check(cx, Batch([rows], [rows + 70], 1, 1, 64, 8, rows), out_type=OUT_F32)
    check(cx, Batch([rows], [rows + 2600], 1, 1, 64, 8, rows + 1), out_type=OUT_F16)
    check(cx, Batch([rows, 700], [rows + 70, 700], 32, 32, 64, 8, rows + 2), out_type=OUT_F16)
