"""Keys with infinities under the attention of a ragged batch (moearc_attn_prefill_batched), at widths that fill the
kernels' channels and widths that do not: a score of minus infinity is a weight of zero, one of plus infinity a row of NaN."""
from __future__ import annotations

import copy

import numpy as np
import pytest

from moearc_amd import OUT_F16, OUT_F32, Context
from test_attn_batch_gpu import Batch, run

pytestmark = pytest.mark.gpu
FORMS = {"small": ([5, 20], [90, 300], 8, 2), "cut": ([2], [2600], 8, 1), "full": ([70, 130], [90, 300], 64, 64),
         "full, cut": ([40], [3001], 8, 1)}


@pytest.fixture(scope="module")
def cx():
    with Context() as c:
        yield c


def batch(form, dim, page, seed):
    """All rows are -2 at the channels whose keys the tests change."""
    s = Batch(*FORMS[form], dim, page, seed)
    s.q[..., :8] = -2
    return s


def at(s, b, j):
    return s.tables[b, j // s.page], j % s.page


@pytest.mark.parametrize("out_type", [OUT_F16, OUT_F32], ids=["f16", "f32"])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dim,page", [(8, 16), (24, 7), (64, 16), (80, 48), (96, 16), (128, 9), (136, 16), (200, 16), (256, 16)], ids=str)
def test_a_score_of_minus_infinity(cx, dim, page, form, out_type):
    s = batch(form, dim, page, dim)
    for b, n in enumerate(s.n_kv):
        for j in (0, 33, n // 2, n - s.new[b] - 1):
            # a score of about -60, whose weight is below 2^-64 of the largest: as good as none
            s.k[at(s, b, j)][:, j % 8] = 30 * np.sqrt(dim)
    want, tol = s.expected(0, dim ** -0.5, out_type)
    for b, n in enumerate(s.n_kv):
        for j in (0, 33, n // 2, n - s.new[b] - 1):
            s.k[at(s, b, j)][:, j % 8] = np.inf
    got = run(cx, s, out_type=out_type).astype(np.float64)
    assert np.isfinite(got).all() and (np.abs(got - want) <= tol).all()


@pytest.mark.parametrize("bad", [-np.inf, np.nan], ids=["inf", "nan"])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dim,page", [(24, 16), (80, 7), (128, 16), (200, 16)], ids=str)
def test_a_score_of_plus_infinity_or_nan(cx, dim, page, form, bad):
    # at the second last key: the last two rows see it, and only they
    s = batch(form, dim, page, dim + 1)
    want, tol = s.expected(0, dim ** -0.5, OUT_F32)
    for b, n in enumerate(s.n_kv):
        s.k[at(s, b, n - 2)][:, 5] = bad
    got = run(cx, s, out_type=OUT_F32).astype(np.float64)
    for b in range(len(s.new)):
        lo, hi = int(s.rows[b]), int(s.rows[b + 1])
        assert np.isnan(got[hi - 2:hi]).all()
        assert (np.abs(got - want) <= tol)[lo:hi - 2].all()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dim", [64, 128])
def test_sinks_at_the_ends_of_f32(cx, dim, form):
    # the lowest ones are none, the highest leave nothing of a row
    s = Batch(*FORMS[form], dim, 16, dim + 2)
    top = float(np.finfo(np.float32).max)
    s.sinks[:7] = top, 2.4e38, 1e38, 1e6, -top, -2.4e38, -1e38
    want, _ = s.expected(0, dim ** -0.5, OUT_F32)
    assert (want[:, :4] == 0).all()
    # (the bound of these heads without a sink: the formula's for an error of the weights has the sink's size in it)
    bare = copy.copy(s)
    bare.sinks = np.where(np.abs(s.sinks) > 1e5, -np.inf, s.sinks)
    _, tol = bare.expected(0, dim ** -0.5, OUT_F32)
    got = run(cx, s, out_type=OUT_F32).astype(np.float64)
    assert np.isfinite(got).all() and (got[:, :4] == 0).all() and (np.abs(got - want) <= tol)[:, 4:].all()
