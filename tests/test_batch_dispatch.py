"""What the ragged batches' calls refuse, launch and take memory for, on the host alone (host_hip.py)."""
from __future__ import annotations

import ctypes
import os
import re

import numpy as np
import pytest

import host_hip
from host_hip import at, launches, names
from moearc_amd import (OUT_F16, OUT_F32, BadArgument, BufferTooSmall, Context, KvType, QkvAppendDesc, native)

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BIG = 1 << 44


@pytest.fixture(scope="module")
def built(tmp_path_factory):
    return host_hip.build(tmp_path_factory.mktemp("host"))


@pytest.fixture
def lib(built, monkeypatch):
    monkeypatch.setattr(native, "_lib", built)
    built.host_hip_reset()
    yield built
    built.host_hip_reset()


@pytest.fixture
def cx(lib):
    with Context() as c:
        yield c


def u32(*values):
    return (ctypes.c_uint * len(values))(*values)


def append(cx, rows=(0, 1, 3), n_kv=(5, 9), bt_stride=4, tables=1 << 30, **kw):
    d = dict(q=1 << 33, k=1 << 34, v=1 << 35, in_type=0, q_stride=256, k_stride=128, v_stride=128, q_norm=None, k_norm=None, eps=1e-6,
             q_out=1 << 36, q_type=1, k_pages=1 << 37, v_pages=1 << 38, kv_type=1, n_pages=7, page_tokens=16, n_heads=4, n_kv_heads=2,
             head_dim=64, n_rot=64, neox=1, freq_base=1e4, freq_scale=1.0, ext_factor=0.0, attn_factor=1.0, corr_lo=0.0, corr_hi=0.0,
             freq_factors=None)
    d.update(kw)
    desc = QkvAppendDesc(**d)
    return cx._lib.moearc_rope_qkv_append_batched(cx.raw, ctypes.byref(desc), tables, bt_stride, u32(*rows), u32(*n_kv), len(n_kv))


NAN, INF = float("nan"), float("inf")


@pytest.mark.parametrize("kw,rc", [
    (dict(), 0), (dict(tables=None), -1), (dict(q=None), -1), (dict(k=None), -1), (dict(v=None), -1), (dict(q_out=None), -1),
    (dict(k_pages=None), -1), (dict(v_pages=None), -1), (dict(in_type=2), -2), (dict(q_type=2), -2), (dict(kv_type=2), -2),
    (dict(n_heads=0), -2), (dict(n_heads=1025, q_stride=1 << 20), -2), (dict(n_kv_heads=0), -2), (dict(n_kv_heads=3, k_stride=192, v_stride=192), 0),
    (dict(n_kv_heads=1025, k_stride=1 << 20, v_stride=1 << 20), -2), (dict(head_dim=0), -2), (dict(head_dim=257, q_stride=2000, k_stride=2000, v_stride=2000), -2),
    (dict(n_rot=0), -2), (dict(n_rot=3), -2), (dict(n_rot=66), -2), (dict(n_rot=2), 0), (dict(page_tokens=0), -2),
    (dict(page_tokens=(1 << 30) + 1), -2), (dict(page_tokens=1 << 30), 0), (dict(n_pages=0), -2), (dict(n_pages=1 << 32), -2),
    (dict(q_stride=255), -2), (dict(k_stride=127), -2), (dict(v_stride=127), -2), (dict(q_stride=1 << 40), -2), (dict(freq_base=0.0), -2),
    (dict(freq_base=NAN), -2), (dict(freq_base=INF), -2), (dict(freq_scale=0.0), -2), (dict(freq_scale=NAN), -2), (dict(eps=-1.0), 0),
    (dict(eps=-1.0, q_norm=64), -2), (dict(eps=NAN, k_norm=64), -2), (dict(eps=0.0, k_norm=64), 0), (dict(rows=(0, 3, 1)), -2),
    (dict(n_kv=(1 << 31, 9)), -2), (dict(n_kv=(1 << 30, 9), bt_stride=1 << 30), -2), (dict(n_kv=((1 << 30) - 1, 9), bt_stride=1 << 30), 0),
    (dict(n_kv=(5, 65)), -2), (dict(n_kv=(5, 64)), 0), (dict(rows=(0, 1, 1), n_kv=(5, 65)), 0),
    (dict(rows=(0, 1, (1 << 20) + 1)), -2), (dict(rows=(0, 1, 1 << 20)), 0), (dict(rows=(3, 3, 3)), 0), (dict(rows=(0,), n_kv=()), 0)], ids=str)
def test_append_refusals(cx, lib, kw, rc):
    assert append(cx, **kw) == rc
    rows = kw.get("rows", (0, 1, 3))
    assert bool(names(lib)) == (rc == 0 and rows[-1] != rows[0])


def test_append_null_arguments(cx, lib):
    f, d = cx._lib.moearc_rope_qkv_append_batched, QkvAppendDesc()
    assert f(None, ctypes.byref(d), 1, 1, u32(0), u32(0), 0) == -1
    assert f(cx.raw, None, 1, 1, u32(0), u32(0), 0) == -1
    assert f(cx.raw, ctypes.byref(d), 1, 1, None, u32(0), 0) == -1
    assert f(cx.raw, ctypes.byref(d), 1, 1, u32(0), None, 0) == -1


@pytest.mark.parametrize("kw,want", [
    (dict(), "l8"), (dict(head_dim=32, n_rot=32), "l8"), (dict(head_dim=128, q_stride=512, k_stride=256, v_stride=256), "l16"),
    (dict(head_dim=136, q_stride=544, k_stride=272, v_stride=272), "l32"), (dict(head_dim=60, n_rot=60), "any"), (dict(n_rot=60), "any"),
    (dict(q_stride=258), "any"), (dict(k_stride=129), "any"), (dict(v_stride=131), "any"), (dict(q=(1 << 33) + 8), "any"),
    (dict(q=(1 << 33) + 8, in_type=1), "l8"), (dict(v=(1 << 35) + 4), "any"), (dict(q_out=(1 << 36) + 4), "any"), (dict(k_pages=(1 << 37) + 4), "any"),
    (dict(v_pages=(1 << 38) + 8, kv_type=0), "any"), (dict(q_norm=68), "any"), (dict(k_norm=64), "l8")], ids=str)
def test_append_kernels(cx, lib, kw, want):
    assert append(cx, **kw) == 0
    assert names(lib) == [f"moearc_qkv_append_{want}_k"]


def test_append_grids(cx, lib):
    # rows x groups of heads; 64 sequences a launch, the ones without rows left out; below 2^32 threads each
    assert append(cx, rows=[2 * b for b in range(130)], n_kv=[9] * 129) == 0
    assert [r[1:] for r in launches(lib)] == [(128, 1, 1, 256), (128, 1, 1, 256), (2, 1, 1, 256)]
    lib.host_hip_reset()
    assert append(cx, rows=[0] * 65 + [4], n_kv=[9] * 65) == 0
    assert [r[1:] for r in launches(lib)] == [(4, 1, 1, 256)]
    lib.host_hip_reset()
    assert append(cx, rows=(0, 1 << 20), n_kv=(1 << 20,), bt_stride=1 << 20, n_heads=1024, q_stride=1 << 16) == 0
    rows = launches(lib)  # 1028 heads, 96 to a work-group
    assert sum(r[1] for r in rows) == 1 << 20 and all(r[0] == "moearc_qkv_append_l8x3_k" and r[2] == 11 and r[1] * 11 * 256 <= 1 << 31 for r in rows)
    lib.host_hip_reset()
    assert append(cx, rows=(0, 2049), n_kv=(2049,), bt_stride=1 << 20) == 0 and append(cx, rows=(0, 2048), n_kv=(2049,), bt_stride=1 << 20) == 0
    assert names(lib) == ["moearc_qkv_append_l8x3_k", "moearc_qkv_append_l8_k"]


def attend(cx, rows=(0, 1, 3), n_kv=(5, 9), **kw):
    a = dict(out=1 << 33, out_type=1, q=1 << 34, k_pages=1 << 35, v_pages=1 << 36, n_pages=99, tables=1 << 30, bt_stride=4,
             rows=u32(*rows), n_kv=u32(*n_kv), sinks=None, n_seqs=len(n_kv), n_swa=0, n_heads=4, n_kv_heads=2, head_dim=64,
             page_tokens=16, scale=0.125, kv_type=1, ws=None, ws_bytes=0)
    a.update(kw)
    return cx._lib.moearc_attn_prefill_batched(cx.raw, *a.values())


@pytest.mark.parametrize("kw,rc", [
    (dict(), 0), (dict(out=None), -1), (dict(q=None), -1), (dict(k_pages=None), -1), (dict(v_pages=None), -1), (dict(tables=None), -1),
    (dict(sinks=64), 0), (dict(kv_type=0), -2), (dict(out_type=2), -2), (dict(n_heads=0), -2), (dict(n_heads=5), -2), (dict(n_kv_heads=0), -2),
    (dict(n_heads=1026), -2), (dict(head_dim=0), -2), (dict(head_dim=60), -2), (dict(head_dim=264), -2), (dict(head_dim=8), 0),
    (dict(head_dim=256), 0), (dict(n_swa=1 << 31), -2), (dict(n_swa=(1 << 31) - 1), 0), (dict(page_tokens=0), -2),
    (dict(page_tokens=(1 << 30) + 1), -2), (dict(n_pages=0), -2), (dict(n_pages=1 << 32), -2), (dict(n_pages=1 << 28), -2),
    (dict(n_pages=(1 << 28) - 1), 0), (dict(scale=NAN), -2), (dict(scale=INF), -2),
    (dict(scale=2.9e38), -2), (dict(scale=-1.0), 0), (dict(scale=0.0), 0), (dict(out=(1 << 33) + 8), -2), (dict(q=(1 << 34) + 2), -2),
    (dict(k_pages=(1 << 35) + 4), -2), (dict(v_pages=(1 << 36) + 8), -2), (dict(rows=(0, 3, 1)), -2), (dict(n_kv=(1 << 31, 9)), -2),
    (dict(n_kv=(5, 65)), -2), (dict(n_kv=(5, 64)), 0), (dict(rows=(0, 1, 1), n_kv=(5, 65)), 0), (dict(rows=(0, 1, (1 << 20) + 1)), -2),
    (dict(rows=(2, 2, 2)), 0), (dict(rows=(0,), n_kv=()), 0), (dict(ws=8, ws_bytes=1 << 40), -2)], ids=str)
def test_attention_refusals(cx, lib, kw, rc):
    assert attend(cx, **kw) == rc
    rows = kw.get("rows", (0, 1, 3))
    assert bool(names(lib)) == (rc == 0 and rows[-1] != rows[0])
    assert cx._lib.moearc_attn_prefill_batched(None, 16, 1, 16, 16, 16, 1, 16, 1, u32(0), u32(0), None, 0, 0, 1, 1, 64, 16, 1.0, 1, None, 0) == -1


@pytest.mark.parametrize("dim,kernel", [(8, "d2"), (64, "d2"), (72, "d4"), (128, "d4"), (136, "d8"), (256, "d8")])
@pytest.mark.parametrize("out_type,form", [(OUT_F16, ""), (OUT_F32, "precise_")])
def test_attention_kernels(cx, lib, dim, kernel, out_type, form):
    assert attend(cx, head_dim=dim, out_type=out_type) == 0
    assert names(lib) == [f"moearc_attn_batch_{form}{kernel}_k"]


def workspace(cx, rows, n_kv, n_swa=0, n_heads=8, n_kv_heads=1, head_dim=128):
    n = ctypes.c_ulong()
    rc = cx._lib.moearc_attn_prefill_batched_workspace(cx.raw, u32(*rows), u32(*n_kv), len(n_kv), n_swa, n_heads, n_kv_heads, head_dim, ctypes.byref(n))
    return n.value if rc == 0 else rc


def test_workspace(cx, lib):
    assert workspace(cx, (0, 4), (100,)) == 0 and workspace(cx, (0,), ()) == 0
    need = workspace(cx, (0, 1), (1 << 16,))
    assert need > 0
    assert workspace(cx, (0, 1), (1 << 16,), n_swa=128) == 0  # a window's keys are few
    for bad in (dict(n_heads=0), dict(n_kv_heads=3), dict(head_dim=12), dict(n_swa=1 << 31)):
        assert workspace(cx, (0, 1), (5,), **bad) == -2
    assert workspace(cx, (1, 0), (5,)) == -2 and workspace(cx, (0, 1), (1 << 31,)) == -2
    f = cx._lib.moearc_attn_prefill_batched_workspace
    assert f(cx.raw, u32(0), u32(0), 0, 0, 1, 1, 64, None) == -1 and f(None, u32(0), u32(0), 0, 0, 1, 1, 64, ctypes.byref(ctypes.c_ulong())) == -1
    kw = dict(rows=(0, 1), n_kv=(1 << 16,), bt_stride=1 << 12, n_heads=8, n_kv_heads=1, head_dim=128)
    assert attend(cx, ws=1 << 40, ws_bytes=need - 1, **kw) == -2 and attend(cx, ws=(1 << 40) + 4, ws_bytes=need, **kw) == -2
    before = lib.host_hip_allocations()
    assert attend(cx, ws=1 << 40, ws_bytes=need, **kw) == 0
    assert lib.host_hip_allocations() == before
    assert names(lib)[-1] == "moearc_attn_batch_merge_k"


def test_memory_of_the_context(cx, lib):
    kw = dict(rows=(0, 1), n_kv=(1 << 16,), bt_stride=1 << 12, n_heads=8, n_kv_heads=1, head_dim=128)
    lib.host_hip_capture(1, 0)
    assert attend(cx, **kw) == -1 and names(lib) == []  # a captured call needs the caller's
    assert attend(cx) == 0  # but where it is not cut
    lib.host_hip_capture(0, 0)
    lib.host_hip_reset()
    lib.host_hip_largest(1 << 10)
    assert attend(cx, **kw) == 0  # without memory: one work-group for the tile
    assert [r[1] for r in launches(lib)] == [1] and lib.host_hip_last_error() == 0
    lib.host_hip_reset()
    lib.host_hip_capture(0, 1)  # another stream's capture goes on
    assert attend(cx, **kw) == 0 and lib.host_hip_broken_captures() == 0
    assert len(names(lib)) == 2


def test_attention_grids(cx, lib):
    # tiles of 128 (token, head) rows x KV heads, of 32 for the few rows of a sequence; sequences without new tokens take no
    # place in a launch
    assert attend(cx, rows=(0, 100, 100, 132, 140), n_kv=(100, 50, 40, 9), n_heads=16, n_kv_heads=2, bt_stride=9) == 0
    assert launches(lib) == [("moearc_attn_batch_d2_k", (25 + 8 + 2) * 2, 1, 1, 256)]
    # up to 64 rows are few; while full tiles would be work-groups for at most half of the CUs, up to 256 or of up to 2560 keys
    for tokens, keys, want in ((992, 2561, 62 + 2 + 3), (992, 2560, 248 + 2 + 3), (1008, 2560, 63 + 2 + 1)):
        lib.host_hip_reset()
        assert attend(cx, rows=(0, tokens, tokens + 8, tokens + 17), n_kv=(keys, 8, 2570), n_heads=16, n_kv_heads=2, bt_stride=999, n_swa=16) == 0
        assert launches(lib) == [("moearc_attn_batch_d2_k", want * 2, 1, 1, 256)]
    lib.host_hip_reset()
    rows = np.concatenate([[0], np.cumsum([b % 2 for b in range(200)])]).tolist()
    assert attend(cx, rows=rows, n_kv=[60] * 200) == 0
    assert [r[1] for r in launches(lib)] == [128, 72]


@pytest.mark.parametrize("page", [1, 2, 3, 5, 7, 16, 48, 100, 255, 256, 1000, 65537, (1 << 30) - 1, 1 << 30])
def test_page_of_a_key_by_multiplication(page):
    # the host's factor and shift (runtime_batch.h) against division, where a wrong quotient would show
    s = (page - 1).bit_length()
    magic = ((1 << (31 + s)) + page - 1) // page
    assert magic < 1 << 32
    top = (1 << 31) - 1
    keys = {0, 1, top, top - 1, *(k * page + d for k in (1, 2, 3, top // page, top // page - 1, top // page // 2) for d in (-1, 0, 1))}
    for key in keys:
        if 0 <= key <= top:
            assert key * magic >> (31 + s) == key // page


def test_wrapper_checks(cx, lib):
    b = lambda n: at(cx, 1 << 34, n)
    mk = lambda **kw: QkvAppendDesc.make(**{**dict(q=b(BIG), k=b(BIG), v=b(BIG), q_out=b(BIG), k_pages=b(BIG), v_pages=b(BIG), n_pages=4, n_heads=4,
                                                  n_kv_heads=2, head_dim=64, page_tokens=16, n_rot=64, freq_base=1e4), **kw})
    go = lambda d, rows=(0, 2), kv=(9,), tables=b(16): cx.rope_qkv_append_batched(d, tables, 1, rows, kv)
    go(mk())
    for kw in (dict(q=b(2 * 1024 - 1)), dict(k=b(2 * 512 - 1)), dict(v=b(2 * 512 - 1)), dict(q_out=b(2 * 512 - 1)), dict(q=b(300 * 4 + 1024 - 1), q_stride=300)):
        with pytest.raises(BufferTooSmall):
            go(mk(**kw))
    go(mk(q=b(300 * 4 + 1024), q_stride=300, k=b(1024), v=b(1024), q_out=b(1024)))
    for kw in (dict(k_pages=b(4 * 16 * 256 - 1)), dict(v_pages=b(4 * 16 * 256 - 1)), dict(q_norm=b(255)), dict(k_norm=b(255)), dict(freq_factors=b(127))):
        with pytest.raises(BufferTooSmall):
            mk(**kw)
    with pytest.raises(BufferTooSmall):
        go(mk(), tables=b(3))
    with pytest.raises(BadArgument):
        go(mk(), rows=(0, 1, 2))

    def attn(**kw):
        a = dict(out=b(BIG), q=b(BIG), k_pages=b(BIG), v_pages=b(BIG), n_pages=4, block_tables=b(BIG), bt_stride=1, row_begin=(0, 2), n_kv=(9,),
                 sinks=None, n_swa=0, n_heads=4, n_kv_heads=2, head_dim=64, page_tokens=16, scale=0.125, out_type=OUT_F16)
        cx.attn_prefill_batched(**{**a, **kw})

    attn()
    attn(out=b(1024), q=b(1024), k_pages=b(16384), v_pages=b(16384), block_tables=b(4), sinks=b(16))
    for kw in (dict(out=b(1023)), dict(out=b(2047), out_type=OUT_F32), dict(q=b(1023)), dict(k_pages=b(16383)), dict(v_pages=b(16383)),
               dict(block_tables=b(3)), dict(sinks=b(15))):
        with pytest.raises(BufferTooSmall):
            attn(**kw)
    for kw in (dict(row_begin=(0,)), dict(head_dim=60), dict(kv=KvType.F32)):
        with pytest.raises(BadArgument):
            attn(**kw)
    with pytest.raises(BadArgument):
        cx.attn_prefill_batched_workspace((0, 1, 2), (5,), 0, 4, 2, 64)


def test_wrapper_lengths(cx, lib):
    """What does not fit 32 bits is refused before it wraps into a length that the library would take."""
    b = lambda n: at(cx, 1 << 34, n)
    d = QkvAppendDesc.make(q=b(BIG), k=b(BIG), v=b(BIG), q_out=b(BIG), k_pages=b(BIG), v_pages=b(BIG), n_pages=4, n_heads=4,
                           n_kv_heads=2, head_dim=64, page_tokens=16, n_rot=64, freq_base=1e4)

    def calls(rows, kv, stride=1):
        yield lambda: cx.rope_qkv_append_batched(d, b(BIG), stride, rows, kv)
        yield lambda: cx.attn_prefill_batched(b(BIG), b(BIG), b(BIG), b(BIG), 4, b(BIG), stride, rows, kv, None, 0, 4, 2, 64, 16, 0.125)
        if stride == 1:
            yield lambda: cx.attn_prefill_batched_workspace(rows, kv, 0, 4, 2, 64)

    i64 = lambda *x: np.array(x, np.int64)
    for rows, kv in (((0, 2), (9,)), (i64(0, 2), i64(9)), (np.array([0, 2], np.uint32), [9]), ((0,), ()), (i64(0), i64())):
        for call in calls(rows, kv):
            call()
    assert len(names(lib)) == 6
    for args in ((i64(0, (1 << 32) + 2), i64(9)), (i64(0, 2), i64((1 << 32) + 9)), ((0, 2), (-1,)), (i64(0, 2), i64(-(1 << 32) + 9)), ((0, 2), (9.5,)),
                 (np.array([[0, 2]]), (9,)), ((), ()), ((0, 2), (9,), -1)):
        for call in calls(*args):
            with pytest.raises(BadArgument):
                call()
    assert len(names(lib)) == 6


def test_rust_descriptor_matches_the_header():
    hdr = open(os.path.join(ROOT, "include", "moearc_attn.h")).read()
    body = re.sub(r"/\*.*?\*/", "", hdr[hdr.index("typedef struct moearc_qkv_append {"):hdr.index("} moearc_qkv_append;")], flags=re.S)
    c_fields = [re.sub(r"[\*]", "", n).strip().split()[-1] for decl in body.split("{", 1)[1].split(";") if decl.strip() for n in decl.split(",")]
    rs = open(os.path.join(ROOT, "crates", "moearc-hip", "src", "ffi.rs")).read()
    rs = rs[rs.index("pub struct MoearcQkvAppend {"):]
    assert c_fields == re.findall(r"pub (\w+):", rs[:rs.index("}")]) == [f[0] for f in QkvAppendDesc._fields_]


@pytest.mark.parametrize("eights", [False, True])
def test_a_segments_keys_are_whole_tiles(eights):
    # the key loops (attn_batch.hip) take 32 keys at a time from a segment's start; copies behind its last key are that one again,
    # and only what a row does not see is masked: each key must enter once
    header = open(os.path.join(ROOT, "moearc_amd", "csrc", "launch_args.h")).read()
    places = int(re.search(r"#define MOEARC_AB_PT (\d+)u", header).group(1))
    seg_keys = places * (8 if eights else 1)
    for lo, hi in ((0, 1), (8, 2048), (0, 4100), (16, 33000), (0, seg_keys), (0, seg_keys + 1), (40, 3 * seg_keys + 77)):
        entered = np.zeros(hi, int)
        for seg in range(lo, hi, seg_keys):
            seg_hi = min(hi, seg + seg_keys)
            for j0 in range(seg, seg_hi, 32):
                for j in range(j0, j0 + 32):
                    if j < hi:  # (the last row sees every key below)
                        entered[min(j, seg_hi - 1)] += 1
        assert (entered[lo:] == 1).all()
