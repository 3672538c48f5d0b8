"""The experts' products of f32 activations far from 1, against the bound that the header states.

u = 2^-24. An f32 value enters as hi + lo halves: to 2^-22 relative (4 u, inside the 2 (32 + cols / 32 + 5) u of the sums), or
2^-25 where lo is below f16's normal range (half its smallest step). The second adds 2^-25 sum|w| to a product, to the second
of two once more. w counts with both its terms' sizes, d s q and dmin m, where a type has two."""
from __future__ import annotations

import numpy as np
import pytest

from moearc_amd import OUT_F32, MoeAct, MoeDesc, QuantType
from oracle import oracle
from test_moe_gpu import TYPES, U, activation, ids_of, weights

pytestmark = pytest.mark.gpu
HALF_STEP = 2.0 ** -25


def _sizes(ty, raw, w):
    """|w|, of both terms where there are two."""
    if ty not in (QuantType.Q4_K, QuantType.Q5_K):
        return np.abs(w)
    total = np.zeros_like(w)
    for at in (0, 2):
        b = raw.reshape(-1, ty.block_bytes).copy()
        b[:, at:at + 2] = 0
        total += np.abs(oracle.dequant(int(ty), b.reshape(-1), len(b)).astype(np.float64).reshape(w.shape))
    return total


def _product(w, size, x, ids, per_slot, halves=True):
    """(y, bound) [tokens, used, rows] in float64; x [tokens, 1 or used, cols]."""
    cols = w.shape[2]
    v = x.astype(np.float64)
    if not per_slot:
        v = np.repeat(v, ids.shape[1], 1)
    y, tol = (np.zeros(ids.shape + w.shape[1:2]) for _ in range(2))
    for i, j in np.ndindex(ids.shape):
        e = ids[i, j]
        y[i, j] = w[e] @ v[i, j]
        tol[i, j] = 2 * (32 + cols / 32 + 5) * U * (size[e] @ np.abs(v[i, j])) + (HALF_STEP * size[e].sum(1) if halves else 0)
    return y, tol


@pytest.mark.parametrize("ty", TYPES, ids=lambda t: t.name)
@pytest.mark.parametrize("scale", [1e-1, 1e-3, 1e-6, 1e-10, 1e4])
@pytest.mark.parametrize("t", [1, 9, 40, 150])
def test_products_of_activations_of_any_size(ctx, ty, scale, t):
    e, k, rows, cols = 3, 2, 70, 512
    raw, w = weights(ty, e, rows, cols, 60)
    rng = np.random.default_rng(t)
    x, ids = (rng.standard_normal((t, 1, cols)) * scale).astype(np.float32), ids_of(rng, t, k, e)
    by = ctx.alloc(t * k * rows * 4)
    ctx.matmul_experts(ty, by, ctx.upload(raw), ctx.upload(x), None, ctx.upload(ids), t, k, e, rows, cols)
    got = ctx.download(by, np.float32, (t, k, rows))
    want, tol = _product(w, _sizes(ty, raw, w), x, ids, False)
    assert np.all(np.abs(got - want) <= tol), np.max(np.abs(got - want) / tol)


@pytest.mark.parametrize("ty", TYPES, ids=lambda t: t.name)
@pytest.mark.parametrize("scale", [1e-1, 1e-3, 1e-6])
@pytest.mark.parametrize("t", [1, 9, 40, 150])
def test_ffn_of_activations_of_any_size(ctx, ty, scale, t):
    """Gate and up of that size, so activations between the products of its square."""
    e, k, embd, ff = 3, 2, 512, 256
    shapes = [(ff, embd), (ff, embd), (embd, ff)]
    made = [weights(ty, e, r, c, 70 + i) for i, (r, c) in enumerate(shapes)]
    size = [_sizes(ty, *m) for m in made]
    rng = np.random.default_rng(t)
    x, ids = (rng.standard_normal((t, embd)) * scale).astype(np.float32), ids_of(rng, t, k, e)
    wt = rng.random((t, k)).astype(np.float32)
    desc = MoeDesc.make([ty] * 3, [ctx.upload(m[0]) for m in made], [None] * 3, e, embd, ff)
    by = ctx.alloc(x.nbytes)
    ctx.moe_ffn(desc, by, ctx.upload(x), ctx.upload(ids), ctx.upload(wt), t, k, io_type=OUT_F32)
    got = ctx.download(by, np.float32, (t, embd))
    # a single token's values enter as they are; the halves' share is granted to the other forms alone
    (g, dg), (u, du) = (_product(made[i][1], size[i], x[:, None], ids, False, t > 1) for i in (0, 1))
    a, da = activation(MoeAct.SWIGLU, g, u, dg, du)
    o, do = _product(made[2][1], size[2], a, ids, True, t > 1)
    want, tol = np.zeros((t, embd)), np.zeros((t, embd))
    for j in range(k):
        moved = np.einsum("tio,to->ti", size[2][ids[:, j]], da[:, j])
        want += wt[:, j:j + 1] * o[:, j]
        tol += wt[:, j:j + 1] * (do[:, j] + 1.01 * moved + (k + 2) * U * np.abs(o[:, j]))
    assert np.all(np.abs(got - want) <= tol), np.max(np.abs(got - want) / tol)
