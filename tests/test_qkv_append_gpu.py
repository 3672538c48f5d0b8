"""New tokens of a ragged batch into the cache (moearc_rope_qkv_append_batched) against float64.

Bounds, u = 2^-24: an angle is f64, reduced, then rounded once (1.6 u radians); its sine and cosine are within 4 u, their
scale within 4 u of itself, the rotation rounds three times: 16 u (|x0| + |x1|) times the scale. A head's norm is
within (D + 8) u of itself. Then half a step of the output's type. V and channels that are not rotated (nor normed)
are rounded to it and nothing else."""
from __future__ import annotations

import numpy as np
import pytest

from moearc_amd import OUT_F16, OUT_F32, Context, DeviceView, KvType, QkvAppendDesc, RopeKind, RopeScaling
from moearc_amd.context import Failed

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture(scope="module")
def cx():
    with Context() as c:
        yield c


def io(t):
    return np.float16 if t == OUT_F16 else np.float32  # KvType.F16 is 1 too


def turn(pos, n_rot, base, scaling, factors):
    """(cos, sin) * scale [positions, pairs] in float64."""
    j = np.arange(n_rot // 2)
    f = float(np.float32(base)) ** (-2.0 * j / n_rot)
    if factors is not None:
        f = f / factors.astype(np.float64)
    freq_scale, ext, attn, lo, hi = (float(np.float32(x)) for x in scaling.args())
    size = attn
    if ext:
        mix = (1 - np.clip((j - lo) / max(0.001, hi - lo), 0, 1)) * ext
        f = f * (freq_scale * (1 - mix) + mix)
        size *= 1 + 0.1 * np.log(1 / freq_scale)
    else:
        f = f * freq_scale
    a = np.asarray(pos, np.float64)[:, None] * f
    return np.cos(a) * size, np.sin(a) * size, size


def rotated(x, pos, n_rot, base, scaling, kind, w, eps, factors):
    """(rows, bound) for x [rows, heads, dim] float64."""
    tol = np.zeros_like(x)
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + float(np.float32(eps))) * w.astype(np.float64)
        tol = (x.shape[-1] + 8) * U * np.abs(x)
    cos, sin, size = turn(pos, n_rot, base, scaling, factors)
    cos, sin = cos[:, None], sin[:, None]
    i0 = np.arange(n_rot // 2) if kind == RopeKind.NEOX else np.arange(0, n_rot, 2)
    i1 = i0 + n_rot // 2 if kind == RopeKind.NEOX else i0 + 1
    a, b, ta, tb = x[..., i0], x[..., i1], tol[..., i0], tol[..., i1]
    y, t = x.copy(), tol.copy()
    y[..., i0], y[..., i1] = a * cos - b * sin, a * sin + b * cos
    extra = abs(size) * (16 * U * (np.abs(a) + np.abs(b)) + ta + tb)
    t[..., i0], t[..., i1] = extra, extra
    return y, t


def step(y, half):
    return 2.0 ** -11 * np.abs(y) + 2.0 ** -25 if half else U * np.abs(y)


def check(cx, new, n_kv, heads, kv_heads, dim, page, n_rot=None, base=10000.0, scaling=RopeScaling.NONE, kind=RopeKind.NEOX, norm=False,
          factors=False, in_type=OUT_F32, q_type=OUT_F16, kv=KvType.F16, fused=0, offset=0, in_place=False, seed=0, bad=None, eps=1e-6):
    """fused: channels between the rows of one product (0: three tensors); offset: bytes by which every input and the query
    output lie off their allocation; bad: (sequence, page index) of a block-table entry that is out of range."""
    rng = np.random.default_rng(seed)
    n_rot = dim if n_rot is None else n_rot
    rows = np.concatenate([[0], np.cumsum(new)]).astype(np.uint32)
    total, kind_in, kind_q, kind_kv = int(rows[-1]), io(in_type), io(q_type), io(kv)
    gap = fused if fused else 0
    width = (heads + 2 * kv_heads) * dim + gap
    data = rng.standard_normal((total, width)).astype(kind_in)
    parts = [data[:, :heads * dim], data[:, heads * dim:(heads + kv_heads) * dim], data[:, (heads + kv_heads) * dim:width - gap]]

    def up(x):
        raw = np.zeros(offset + x.nbytes, np.uint8)
        raw[offset:] = np.ascontiguousarray(x).view(np.uint8).reshape(-1)
        return DeviceView(cx.upload(raw), offset)

    if fused:
        whole, size = up(data), data.itemsize
        bufs = [whole, DeviceView(whole, heads * dim * size), DeviceView(whole, (heads + kv_heads) * dim * size)]
        strides = [width] * 3
    else:
        bufs, strides = [up(p) for p in parts], [None] * 3
    counts = [-(-n // page) for n in n_kv]
    n_pages, stride = sum(counts) + 1, max(counts + [1])
    ids = rng.permutation(n_pages)[:sum(counts)]
    tables = np.full((len(new), stride), 0xFFFFFFFF, np.uint32)
    at = 0
    for b, c in enumerate(counts):
        tables[b, :c] = ids[at:at + c]
        at += c
    if bad:
        tables[bad] = n_pages
    pools = [rng.standard_normal((n_pages, page, kv_heads, dim)).astype(kind_kv) for _ in range(2)]
    k_pages, v_pages = (cx.upload(p) for p in pools)
    w = [(1 + 0.3 * rng.standard_normal(dim)).astype(np.float32) if norm else None for _ in range(2)]
    ff = rng.uniform(1, 8, n_rot // 2).astype(np.float32) if factors else None
    q_before = np.full((total, heads, dim), 5.0, kind_q)
    q_out = bufs[0] if in_place else up(q_before)
    desc = QkvAppendDesc.make(*bufs, q_out, k_pages, v_pages, n_pages, heads, kv_heads, dim, page, n_rot, base, scaling, kind, in_type,
                              q_type, kv, *strides, cx.upload(w[0]) if norm else None, cx.upload(w[1]) if norm else None, eps,
                              cx.upload(ff) if factors else None)
    cx.rope_qkv_append_batched(desc, cx.upload(tables), stride, rows, n_kv)
    if bad:
        with pytest.raises(Failed):
            cx.sync()
    else:
        cx.sync()
    pos = np.concatenate([np.arange(n - m, n) for m, n in zip(new, n_kv)]) if total else np.zeros(0)
    x = [p.astype(np.float64).reshape(total, -1, dim) for p in parts]
    want_q, tol_q = rotated(x[0], pos, n_rot, base, scaling, kind, w[0], eps, ff)
    want_k, tol_k = rotated(x[1], pos, n_rot, base, scaling, kind, w[1], eps, ff)
    got_q = cx.download(q_out, kind_q, q_before.shape).astype(np.float64)
    live = pos >= 0
    assert (np.abs(got_q - want_q)[live] <= (1.01 * (tol_q + step(want_q, q_type == OUT_F16)))[live]).all()
    if not in_place:
        assert (got_q[~live] == 5.0).all()
    pages = [p.astype(np.float64) for p in pools]
    tol = np.zeros_like(pages[0])
    for b, (m, n) in enumerate(zip(new, n_kv)):
        for i in range(m):
            p, row = n - m + i, int(rows[b]) + i
            if p < 0 or tables[b, p // page] >= n_pages:
                continue
            to = tables[b, p // page], p % page
            pages[0][to], pages[1][to] = want_k[row], x[2][row].astype(kind_kv)
            tol[to] = 1.01 * (tol_k[row] + step(want_k[row], kv == KvType.F16))
    got = [cx.download(p, kind_kv, pools[0].shape).astype(np.float64) for p in (k_pages, v_pages)]
    assert (np.abs(got[0] - pages[0]) <= tol).all()  # the untouched slots exactly
    assert (got[1] == pages[1]).all()


NEW, CACHED = [1, 0, 5, 33, 2], [0, 9, 31, 1, 260]
KV = np.add(NEW, CACHED).tolist()
YARN = RopeScaling.yarn(64, 4096, 150000.0, 32.0)


@pytest.mark.parametrize("kind", list(RopeKind), ids=str)
@pytest.mark.parametrize("heads,kv_heads,dim,n_rot", [(64, 8, 64, 64), (4, 4, 64, 32), (16, 2, 128, 128), (5, 1, 80, 80), (6, 2, 96, 48),
                                                      (3, 1, 256, 256), (2, 2, 256, 64), (7, 1, 8, 8)], ids=str)
def test_shapes(cx, heads, kv_heads, dim, n_rot, kind):
    check(cx, NEW, KV, heads, kv_heads, dim, 16, n_rot, kind=kind)
    check(cx, NEW, KV, heads, kv_heads, dim, 7, n_rot, kind=kind, norm=True, q_type=OUT_F32, kv=KvType.F32, seed=1)


@pytest.mark.parametrize("kind", list(RopeKind), ids=str)
@pytest.mark.parametrize("heads,kv_heads,dim,n_rot", [(4, 2, 64, 36), (3, 1, 77, 10), (2, 1, 255, 254), (1, 1, 2, 2), (2, 1, 1 + 2, 2), (9, 3, 130, 130)],
                         ids=str)
def test_odd_heads(cx, heads, kv_heads, dim, n_rot, kind):
    check(cx, NEW, KV, heads, kv_heads, dim, 16, n_rot, kind=kind, norm=True, q_type=OUT_F32)


@pytest.mark.parametrize("in_type", [OUT_F32, OUT_F16], ids=["f32", "f16"])
@pytest.mark.parametrize("q_type", [OUT_F32, OUT_F16], ids=["f32", "f16"])
@pytest.mark.parametrize("kv", list(KvType), ids=str)
def test_types_and_one_products_rows(cx, in_type, q_type, kv):
    check(cx, NEW, KV, 8, 2, 64, 16, in_type=in_type, q_type=q_type, kv=kv)
    check(cx, NEW, KV, 8, 2, 64, 16, in_type=in_type, q_type=q_type, kv=kv, fused=4, norm=True)
    check(cx, NEW, KV, 8, 2, 64, 16, in_type=in_type, q_type=q_type, kv=kv, fused=3)  # rows off their alignment


@pytest.mark.parametrize("in_type,offset", [(OUT_F32, 4), (OUT_F32, 8), (OUT_F16, 2), (OUT_F16, 8)], ids=str)
def test_addresses_off_their_alignment(cx, in_type, offset):
    check(cx, NEW, KV, 8, 2, 64, 16, in_type=in_type, q_type=in_type, offset=offset)


def test_in_place(cx):
    check(cx, NEW, KV, 8, 2, 128, 16, norm=True, q_type=OUT_F32, in_place=True)


@pytest.mark.parametrize("kind", list(RopeKind), ids=str)
def test_far_positions(cx, kind):
    # one page holds them all: only the angles are far. Linear scaling, YaRN, factors, both
    for scaling in (RopeScaling.NONE, RopeScaling(0.25), YARN, RopeScaling(1 / 32, 0.5, 1.2, 8.0, 18.0)):
        for factors in (False, True):
            check(cx, [3, 2], [65537, 40000], 2, 1, 64, 8192, base=150000.0, scaling=scaling, kind=kind, factors=factors,
                  q_type=OUT_F32, kv=KvType.F32)


def test_positions_before_the_first(cx):
    check(cx, [5, 3, 40], [2, 0, 7], 8, 2, 64, 16)
    check(cx, [5, 3, 40], [2, 0, 7], 3, 1, 30, 16, norm=True)


def test_many_sequences(cx):
    rng = np.random.default_rng(3)
    new = [0 if b % 3 == 2 else int(rng.integers(1, 4)) for b in range(150)]
    check(cx, new, np.add(new, rng.integers(0, 50, 150)).tolist(), 4, 1, 64, 16)


@pytest.mark.parametrize("dim", [64, 66])
def test_a_page_outside_the_pool(cx, dim):
    check(cx, [3, 20], [40, 50], 4, 2, dim, 16, bad=(1, 2))
    check(cx, [3, 20], [40, 50], 4, 2, dim, 16)  # reported once


# ---- long batches: three heads to a thread (more than eight work-groups to each of 256 CUs with one) ------------------
LONG_NEW, LONG_CACHED = [200, 0, 333, 1, 170], [0, 9, 31, 4000, 260]
LONG_KV = np.add(LONG_NEW, LONG_CACHED).tolist()
# 256 / lanes heads to a work-group, times three: one with room to spare, and a second with few; threads whose three heads
# are of q, k and v
LONG_SHAPES = [(64, 8, 64, 64), (100, 9, 64, 32), (30, 33, 40, 40), (32, 4, 128, 128), (50, 7, 96, 48), (47, 1, 80, 80), (16, 2, 256, 256),
               (21, 3, 136, 64), (2, 11, 200, 200)]


def takes_three(heads, kv_heads, dim, rows):
    at_a_time = 32 if dim <= 64 else 16 if dim <= 128 else 8
    return -(-(heads + 2 * kv_heads) // at_a_time) * rows > 8 * 256


@pytest.mark.parametrize("kind", list(RopeKind), ids=str)
@pytest.mark.parametrize("heads,kv_heads,dim,n_rot", LONG_SHAPES, ids=str)
def test_long_batches(cx, heads, kv_heads, dim, n_rot, kind):
    new = np.array(LONG_NEW)
    while not takes_three(heads, kv_heads, dim, new.sum()):
        new = new * 2
    kv = np.add(new, LONG_CACHED).tolist()
    check(cx, new, kv, heads, kv_heads, dim, 16, n_rot, kind=kind, norm=True, q_type=OUT_F32, kv=KvType.F32)
    check(cx, new, kv, heads, kv_heads, dim, 100, n_rot, kind=kind, in_type=OUT_F16, fused=8, seed=1)


@pytest.mark.parametrize("in_type", [OUT_F32, OUT_F16], ids=["f32", "f16"])
@pytest.mark.parametrize("q_type", [OUT_F32, OUT_F16], ids=["f32", "f16"])
@pytest.mark.parametrize("kv", list(KvType), ids=str)
def test_long_batches_types(cx, in_type, q_type, kv):
    assert takes_three(80, 10, 64, sum(LONG_NEW))
    check(cx, LONG_NEW, LONG_KV, 80, 10, 64, 16, in_type=in_type, q_type=q_type, kv=kv, norm=True, factors=True, scaling=YARN)


@pytest.mark.parametrize("heads,kv_heads,dim", [(64, 16, 64), (32, 8, 128), (17, 4, 256)], ids=str)
def test_long_batches_of_few_positions_and_bad_pages(cx, heads, kv_heads, dim):
    assert takes_three(heads, kv_heads, dim, 704)
    check(cx, [300, 404], [0, 150], heads, kv_heads, dim, 16)  # most rows sit before the first position
    check(cx, [300, 404], [400, 404], heads, kv_heads, dim, 16, bad=(1, 2), norm=True)


def test_a_long_batch_in_place(cx):
    check(cx, LONG_NEW, LONG_KV, 32, 8, 128, 16, norm=True, q_type=OUT_F32, in_place=True)


@pytest.mark.parametrize("rows", [40, 704], ids=["one", "three"])
@pytest.mark.parametrize("normed", ["q", "k"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(50, 30, 64), (31, 5, 128), (13, 7, 256)], ids=str)
def test_a_norm_of_one_kind(cx, heads, kv_heads, dim, normed, rows):
    # a wave's heads are of q, k and v, and only one kind's are normed
    rng = np.random.default_rng(17)
    assert takes_three(heads, kv_heads, dim, rows) == (rows == 704)
    x = [rng.standard_normal((rows, n, dim)).astype(np.float32) for n in (heads, kv_heads, kv_heads)]
    w = (1 + 0.3 * rng.standard_normal(dim)).astype(np.float32)
    q_out, pools = cx.alloc(rows * heads * dim * 4), [cx.alloc(rows * kv_heads * dim * 4) for _ in range(2)]
    d = QkvAppendDesc.make(*(cx.upload(a) for a in x), q_out, *pools, 1, heads, kv_heads, dim, rows, dim, 1e4, q_type=OUT_F32, kv=KvType.F32,
                           **{normed + "_norm": cx.upload(w)})
    cx.rope_qkv_append_batched(d, cx.upload(np.zeros(1, np.uint32)), 1, [0, rows], [rows])
    cx.sync()
    for a, kind, buf in ((x[0], "q", q_out), (x[1], "k", pools[0])):
        want, tol = rotated(a.astype(np.float64), np.arange(rows), dim, 1e4, RopeScaling.NONE, RopeKind.NEOX, w if kind == normed else None, 1e-6, None)
        got = cx.download(buf, np.float32, a.shape).astype(np.float64)
        assert (np.abs(got - want) <= 1.01 * (tol + step(want, False))).all()
    assert np.array_equal(cx.download(pools[1], np.float32, x[2].shape), x[2])
