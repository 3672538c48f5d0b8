"""moe_ffn in more than one chunk of tokens (32,768 slots each): the same as a call for each chunk, and right in each."""
from __future__ import annotations

import numpy as np
import pytest

from moearc_amd import NO_EXPERT, OUT_F16, OUT_F32, DeviceView, MoeAct, MoeDesc, QuantType
from test_moe_gpu import ALPHA, LIMIT, U, activation, ids_of, product, step16, weights

pytestmark = pytest.mark.gpu
CHUNK, K = 8192, 4  # tokens of a chunk at four experts each


@pytest.mark.parametrize("t", [8193, 8250, 16500])  # a remainder without a plan, of light tiles; three chunks
@pytest.mark.parametrize("io", [OUT_F32, OUT_F16], ids=["f32", "f16"])
@pytest.mark.parametrize("own_ws", [False, True], ids=["context", "caller"])
def test_chunks_equal_their_calls(ctx, t, io, own_ws):
    e, embd, ff, types = 6, 288, 256, (QuantType.MXFP4, QuantType.Q5_K)
    rng = np.random.default_rng(t)
    dtype = np.float16 if io == OUT_F16 else np.float32
    made = [weights(types[i > 1], e, r, c, 80 + i) for i, (r, c) in enumerate([(ff, embd), (ff, embd), (embd, ff)])]
    bs = [rng.standard_normal((e, n)).astype(np.float32) * np.float32(0.2) for n in (ff, ff, embd)]
    x, y0 = (rng.standard_normal((t, embd)).astype(dtype) for _ in range(2))
    ids, wt = ids_of(rng, t, K, e, 0.1), rng.random((t, K)).astype(np.float32)
    wt[ids >= e] = np.nan  # not read
    desc = MoeDesc.make([types[0], types[0], types[1]], [ctx.upload(m[0]) for m in made], [ctx.upload(b) for b in bs], e, embd, ff,
                        MoeAct.SWIGLU_CLAMPED, ALPHA, LIMIT)
    bx, bi, bt, by, bz = (ctx.upload(v) for v in (x, ids, wt, y0, y0))
    add, ws = io == OUT_F32, None
    if own_ws:
        n_ws = ctx.moe_workspace(t, K, e, embd, ff)
        held = ctx.upload(np.full(n_ws + 256, 0xA5, np.uint8))
        ws = DeviceView(held, 0, n_ws)
    ctx.moe_ffn(desc, by, bx, bi, bt, t, K, io, add, ws)
    row = embd * x.itemsize
    for a in range(0, t, CHUNK):
        n = min(CHUNK, t - a)
        ctx.moe_ffn(desc, DeviceView(bz, a * row), DeviceView(bx, a * row), DeviceView(bi, a * K * 4), DeviceView(bt, a * K * 4), n, K, io, add)
    got, parts = (ctx.download(b, dtype, (t, embd)) for b in (by, bz))
    # a remainder of one token runs in two launches when it is a call of its own
    alike = t - 1 if t % CHUNK == 1 else t
    assert np.array_equal(got[:alike], parts[:alike])
    if own_ws:  # nothing behind it is written
        assert np.all(ctx.download(held, np.uint8, (n_ws + 256,))[n_ws:] == 0xA5)
    at = np.unique(np.concatenate([[0, CHUNK - 1, CHUNK, t - 1], rng.integers(0, t, 40)]))
    x, ids, wt, want = x[at], ids[at], wt[at], np.zeros((len(at), embd))
    (g, dg), (u, du) = (product(made[i][1], bs[i], x[:, None], ids, False) for i in (0, 1))
    v, dv = activation(MoeAct.SWIGLU_CLAMPED, g, u, dg, du)
    o, do = product(made[2][1], bs[2], v, ids, True)
    dv, tol = dv + step16(v, io), np.zeros_like(want)
    for i, j in np.ndindex(ids.shape):
        if ids[i, j] < e:
            want[i] += wt[i, j] * o[i, j]
            tol[i] += wt[i, j] * (do[i, j] + 1.01 * np.abs(made[2][1][ids[i, j]]) @ dv[i, j] + (K + 2) * U * np.abs(o[i, j]))
    if add:
        want, tol = want + y0[at], tol + U * np.abs(want + y0[at])
    assert np.any(ids == NO_EXPERT) and np.all(np.abs(got[at] - want) <= tol + step16(want, io))
