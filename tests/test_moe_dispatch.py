"""What the expert half of a block refuses, launches and takes memory for, on the host alone (host_hip.py)."""
from __future__ import annotations

import ctypes
import os
import re

import pytest

import host_hip
from host_hip import at, names
from moearc_amd import (OUT_F16, OUT_F32, BadArgument, BufferTooSmall, Context, MoeAct, MoeDesc, QuantType, RouteMode,
                        native)
from moearc_amd.context import Failed

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BIG = 1 << 40


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


def norm(cx, **kw):
    a = dict(x=1 << 33, x_type=0, h=1 << 34, y=1 << 35, y_type=0, w_post=None, gate=None, gate_stride=0, scale=1.0, w_pre=None,
             n_rows=4, n_cols=64, eps=1e-5)
    a.update(kw)
    return cx._lib.moearc_norm_residual(cx.raw, *a.values())


@pytest.mark.parametrize("kw,rc", [
    (dict(), 0), (dict(h=None), -1), (dict(x=None, y=None), -1), (dict(x=None), 0), (dict(y=None), 0), (dict(n_rows=0), 0),
    (dict(x_type=2), -2), (dict(y_type=2), -2), (dict(y=None, w_post=64), -2), (dict(y=None, gate=64), -2),
    (dict(x=None, w_pre=64), -2), (dict(n_cols=0), -2), (dict(n_cols=1 << 30), -2), (dict(n_rows=1 << 31), -2),
    (dict(gate=64, gate_stride=63), -2), (dict(gate=64, gate_stride=64), 0), (dict(gate=64), 0), (dict(eps=-1e-9), -2),
    (dict(eps=float("nan")), -2), (dict(eps=0.0), 0)], ids=str)
def test_norm_refusals(cx, lib, kw, rc):
    assert norm(cx, **kw) == rc
    assert len(names(lib)) == (1 if rc == 0 and kw.get("n_rows") != 0 else 0)
    assert cx._lib.moearc_norm_residual(None, 1, 0, 1, 1, 0, None, None, 0, 1.0, None, 1, 1, 0.0) == -1


@pytest.mark.parametrize("cols,kw,want", [
    (256, {}, "r16_v4"), (260, {}, "r64_v4"), (257, {}, "r64_v1"), (1024, {}, "r64_v4"), (1025, {}, "r256_v1"), (2880, {}, "r256_v4"),
    (4100, {}, "r1024_v4"), (16384, {}, "r1024_v4"), (16388, {}, "long"), (2880, dict(h=(1 << 34) + 8), "r256_v1"),
    (2880, dict(x=(1 << 33) + 8), "r256_v1"), (2880, dict(x=(1 << 33) + 8, x_type=1), "r256_v4"),
    (2880, dict(gate=1 << 32, gate_stride=2882), "r256_v1"), (2880, dict(y=(1 << 35) + 8, y_type=1), "r256_v4")], ids=str)
def test_norm_forms(cx, lib, cols, kw, want):
    assert norm(cx, n_cols=cols, **kw) == 0
    assert names(lib) == [f"moearc_norm_{want}_k"]


@pytest.mark.parametrize("kw,rc", [
    (dict(), 0), (dict(ids=None), -1), (dict(weights=None), -1), (dict(logits=None), -1), (dict(n_expert=0), -2),
    (dict(n_expert=1025), -2), (dict(n_used=0), -2), (dict(n_used=33), -2), (dict(n_used=32), 0), (dict(mode=2), -2),
    (dict(n_tok=1 << 31), -2), (dict(n_tok=0), 0)], ids=str)
def test_route_refusals(cx, lib, kw, rc):
    a = dict(ids=64, weights=64, logits=64, n_tok=3, n_expert=32, n_used=4, mode=1, scale=1.0)
    a.update(kw)
    assert cx._lib.moearc_moe_route(cx.raw, *a.values()) == rc
    assert len(names(lib)) == (1 if rc == 0 and a["n_tok"] else 0)


def linear(cx, **kw):
    a = dict(ty=8, y=1 << 33, w=1 << 34, x=1 << 35, io=0, bias=None, ids=1 << 36, n_tok=100, n_used=4, n_expert=8, per=0,
             n_rows=64, n_cols=256, ws=None, ws_bytes=0)
    a.update(kw)
    return cx._lib.moearc_matmul_experts(cx.raw, *a.values())


LINEAR = [
    (dict(), 0), (dict(y=None), -1), (dict(w=None), -1), (dict(x=None), -1), (dict(ids=None), -1), (dict(ty=0), -2),
    (dict(ty=2), -2), (dict(io=2), -2), (dict(per=2), -2), (dict(n_expert=0), -2), (dict(n_expert=1025), -2), (dict(n_used=0), -2),
    (dict(n_used=1025), -2), (dict(n_rows=0), -2), (dict(n_rows=(1 << 20) + 1), -2), (dict(n_cols=224), -2), (dict(n_cols=272), -2),
    (dict(n_cols=288), 0), (dict(ty=12, n_cols=288), -2), (dict(n_cols=(1 << 20) + 256), -2), (dict(w=(1 << 34) + 1), -2),
    (dict(n_tok=0), 0), (dict(n_tok=1 << 31), -2), (dict(ws=256, ws_bytes=16), -2), (dict(ws=128, ws_bytes=BIG), -2),
    (dict(ws=256, ws_bytes=BIG), 0)]


@pytest.mark.parametrize("kw,rc", LINEAR, ids=str)
def test_product_refusals(cx, lib, kw, rc):
    assert linear(cx, **kw) == rc
    assert bool(names(lib)) == (rc == 0 and kw.get("n_tok") != 0)


def ffn(cx, desc=None, **kw):
    d = MoeDesc()
    d.w_type[:] = [8, 8, 8]
    d.w[:] = [1 << 34, 1 << 34, 1 << 34]
    d.n_expert, d.n_embd, d.n_ff, d.act, d.alpha, d.limit = 8, 256, 512, 0, 1.702, 7.0
    for k, v in (desc or {}).items():
        if isinstance(v, list):
            getattr(d, k)[:] = v
        else:
            setattr(d, k, v)
    a = dict(y=1 << 33, x=1 << 35, io=0, ids=1 << 36, weights=1 << 36, n_tok=100, n_used=4, add=0, ws=None, ws_bytes=0)
    a.update(kw)
    return cx._lib.moearc_moe_ffn(cx.raw, ctypes.byref(d), *a.values())


@pytest.mark.parametrize("desc,kw,rc", [
    ({}, {}, 0), ({}, dict(y=None), -1), ({}, dict(x=None), -1), ({}, dict(ids=None), -1), ({}, dict(weights=None), -1),
    ({"w": [0, 64, 64]}, {}, -1), ({"w": [64, 64, 0]}, {}, -1), ({"w_type": [8, 39, 8]}, {}, -2), ({"w_type": [8, 8, 14]}, {}, 0),
    ({"w_type": [0, 0, 8]}, {}, -2), ({"act": 2}, {}, -2), ({"act": 1, "limit": -1.0}, {}, -2), ({"act": 1, "limit": float("nan")}, {}, -2),
    ({"limit": -1.0}, {}, 0), ({}, dict(add=2), -2), ({}, dict(add=1), 0), ({}, dict(add=1, io=1), -2), ({}, dict(io=1), 0),
    ({}, dict(io=2), -2), ({"n_ff": 224}, {}, -2), ({"n_embd": 224}, {}, -2), ({"w_type": [8, 8, 12], "n_ff": 288}, {}, -2),
    ({"n_expert": 0}, {}, -2), ({"n_expert": 1025}, {}, -2), ({}, dict(n_used=0), -2), ({}, dict(n_tok=0), 0),
    ({}, dict(ws=256, ws_bytes=1024), -2), ({}, dict(ws=64, ws_bytes=BIG), -2), ({}, dict(ws=256, ws_bytes=BIG), 0)], ids=str)
def test_ffn_refusals(cx, lib, desc, kw, rc):
    assert ffn(cx, desc, **kw) == rc
    assert bool(names(lib)) == (rc == 0 and kw.get("n_tok") != 0)
    assert cx._lib.moearc_moe_ffn(cx.raw, None, 64, 64, 0, 64, 64, 1, 1, 0, None, 0) == -1


def _kernels(lib):
    return [k[len("moearc_moe_"):-len("_k")] for k in names(lib)]


FORMS = [  # slots per expert, type, f16: the product's form
    (2, 8, 0, "light"), (55, 8, 0, "light"), (56, 8, 0, "tile"), (39, 8, 1, "light"), (40, 8, 1, "tile"), (55, 39, 0, "light"),
    (56, 39, 0, "tile"), (56, 14, 0, "tile"), (400, 12, 0, "tile")]


@pytest.mark.parametrize("each,ty,half,form", FORMS, ids=str)
def test_product_forms(cx, lib, each, ty, half, form):
    name = {8: "q8_0", 39: "mxfp4", 14: "q6_k", 12: "q4_k"}[ty]
    io = "f16" if half else "f32"
    assert linear(cx, ty=ty, io=half, n_tok=each * 40, n_used=1, n_expert=40) == 0
    plan = "plan" if half and ty == 8 else f"plan_{io}"  # f16 rows of Q8_0 products are taken as they are
    assert _kernels(lib) == [plan, f"{form}_{name}_p_{io}"]
    lib.host_hip_reset()
    assert ffn(cx, {"w_type": [ty] * 3, "n_expert": 40}, io=half, n_tok=each * 40, n_used=1) == 0
    assert _kernels(lib) == [plan, f"{form}_{name}_gu_{io}", f"{form}_{name}_p_{io}", "combine"]


def test_grids_cover_every_tile(cx, lib):
    # tiles: at most one partly filled for each expert and for the slots without one
    for tok, used, experts, rows in ((17, 4, 128, 2880), (1000, 8, 128, 768), (8192, 4, 32, 2880), (65, 1, 1, 1)):
        for io in (0, 1):
            for ty in (1, 8, 12, 13, 14, 39):
                lib.host_hip_reset()
                assert linear(cx, ty=ty, io=io, n_tok=tok, n_used=used, n_expert=experts, n_rows=rows) == 0
                (name, gx, gy, gz, block) = host_hip.launches(lib)[-1]
                light = "light" in name
                wide = not light and (ty in (12, 13) or (ty == 39 and not io))
                tile, per, slots = 32 if light else 64, 256 if wide else 128, tok * used
                tiles = min(slots, -(-slots // tile) + experts + 1)
                assert (gy, gz, block) == (1, 1, 256) and gx % 8 == 0 and tiles * -(-rows // per) <= gx < tiles * -(-rows // per) + 8


def test_few_slots_and_single_tokens(cx, lib):
    assert linear(cx, n_tok=16, n_used=4, n_rows=70) == 0
    assert host_hip.launches(lib) == [("moearc_moe_small_q8_0_p_f32_k", 3, 64, 1, 512)]
    lib.host_hip_reset()
    assert ffn(cx, n_tok=16, n_used=4) == 0
    assert _kernels(lib) == ["small_q8_0_gu_f32", "small_q8_0_p_f32", "combine"]
    for desc, kw, want in (
            ({}, {}, ["vec_q8_0_gu_p1", "vec_q8_0_down_p1"]),  # 256 and 512 columns: 16 and 32 pieces
            ({"n_ff": 2880, "n_embd": 2880, "w_type": [39, 39, 39]}, {}, ["vec_mxfp4_gu_p2", "vec_mxfp4_down_p2"]),
            ({"n_ff": 4096, "w_type": [8, 8, 12]}, dict(n_used=2), ["vec_q8_0_gu_p1", "vec_q4_k_down_p2"]),
            ({"n_ff": 2048, "n_embd": 2048, "w_type": [14, 14, 14]}, {}, ["vec_q6_k_gu_p2", "vec_q6_k_down_p2"]),
            ({"n_ff": 4128}, {}, ["small_q8_0_gu_f32", "small_q8_0_p_f32", "combine"]),  # 258 pieces
            ({"n_ff": 4096}, dict(n_used=4), ["small_q8_0_gu_f32", "small_q8_0_p_f32", "combine"])):  # inputs past the LDS
        lib.host_hip_reset()
        assert ffn(cx, desc, n_tok=1, **kw) == 0
        assert _kernels(lib) == want, (desc, kw)
    lib.host_hip_reset()
    assert ffn(cx, n_tok=1, n_used=65) == 0  # more than a wave's lanes
    assert _kernels(lib)[0] == "plan_f32"


@pytest.mark.parametrize("tok,used,experts,types,few", [
    (16, 4, 128, (8, 8), True), (16, 4, 31, (39, 39), True), (16, 4, 32, (39, 39), False), (6, 4, 128, (39, 39), True),
    (7, 4, 128, (39, 39), False), (7, 4, 128, (39, 14), True), (17, 4, 8, (39, 39), False)], ids=str)
def test_few_slots_need_no_plan(cx, lib, tok, used, experts, types, few):
    assert ffn(cx, {"w_type": [types[0], types[0], types[1]], "n_expert": experts}, n_tok=tok, n_used=used) == 0
    assert (_kernels(lib)[0] == "small_%s_gu_f32" % {8: "q8_0", 39: "mxfp4"}[types[0]]) == few


def test_long_calls_run_in_chunks(cx, lib):
    assert ffn(cx, n_tok=8192 * 2 + 1, n_used=4) == 0
    per = ["plan_f32", "tile_q8_0_gu_f32", "tile_q8_0_p_f32", "combine"]
    assert _kernels(lib)[:8] == per * 2 and _kernels(lib)[8:] == ["small_q8_0_gu_f32", "small_q8_0_p_f32", "combine"]


def test_workspace_sizes(lib):
    n = ctypes.c_ulong()

    def size(*a):
        assert lib.moearc_moe_workspace(*a, ctypes.byref(n)) == 0
        return n.value
    last = 0
    for t in (0, 1, 3, 16, 17, 64, 65, 1000, 8192, 8193, 10 ** 6):
        for ff in (0, 512):
            assert size(t, 4, 128, 2880, ff) % 256 == 0
        assert size(t, 4, 128, 2880, 2880) >= last
        last = size(t, 4, 128, 2880, 2880)
    assert last < 1 << 30  # longer calls run in chunks
    assert lib.moearc_moe_workspace(1, 1, 1, 256, 256, None) == -1
    for a in ((1, 0, 8, 256, 0), (1, 1, 0, 256, 0), (1, 1, 1025, 256, 0), (1, 1, 8, 0, 0), (1 << 31, 1, 8, 256, 0)):
        assert lib.moearc_moe_workspace(*a, ctypes.byref(n)) == -2


def test_the_wrapper_checks_sizes(cx):
    b = at(cx, 1 << 33, BIG)
    small = at(cx, 1 << 34, 16)
    for bad in range(5):
        bufs = [small if i == bad else b for i in range(5)]
        with pytest.raises(BufferTooSmall):
            cx.matmul_experts(QuantType.Q8_0, bufs[0], bufs[1], bufs[2], bufs[3], bufs[4], 10, 4, 8, 64, 256)
        with pytest.raises(BufferTooSmall):
            cx.norm_residual(bufs[0], bufs[1], bufs[2], bufs[3], bufs[4], 64, 1.0, None, 10, 64, 1e-5)
    with pytest.raises(BadArgument):
        cx.matmul_experts(QuantType.Q4_K, b, b, b, None, b, 10, 4, 8, 64, 288)
    with pytest.raises(BufferTooSmall):
        MoeDesc.make([QuantType.Q8_0] * 3, [b, small, b], [None] * 3, 8, 256, 256)
    desc = MoeDesc.make([QuantType.Q8_0] * 3, [b, b, b], [None, b, None], 8, 256, 256, MoeAct.SWIGLU)
    for bad in range(4):
        bufs = [small if i == bad else b for i in range(4)]
        with pytest.raises(BufferTooSmall):
            cx.moe_ffn(desc, *bufs, 10, 4)
    with pytest.raises(BufferTooSmall):
        cx.moe_route(small, b, b, 10, 8, 4, RouteMode.SOFTMAX_ALL)
    with pytest.raises(BadArgument):
        cx.moe_workspace(10, 0, 8, 256)


def test_captured_calls_take_the_callers_workspace_only(cx, lib):
    for call in (linear, ffn):
        lib.host_hip_reset()
        lib.host_hip_capture(1, 0)
        assert call(cx) == -1 and not names(lib)
        assert call(cx, ws=256, ws_bytes=BIG) == 0 and names(lib)
        assert lib.host_hip_broken_captures() == 0
        lib.host_hip_capture(0, 1)  # another stream's capture: the context's workspace may grow
        assert call(cx) == 0 and lib.host_hip_broken_captures() == 0
        lib.host_hip_capture(0, 0)


def test_a_workspace_that_cannot_grow_is_an_error(cx, lib):
    lib.host_hip_largest(1 << 10)
    assert ffn(cx, n_tok=2000) == -1
    assert not names(lib) and lib.host_hip_last_error() == 0
    with pytest.raises(Failed):
        cx.matmul_experts(QuantType.Q8_0, *[at(cx, 1 << 33, BIG)] * 3, None, at(cx, 1 << 33, BIG), 3000, 4, 8, 64, 256)


def test_descriptor_matches_the_header():
    hdr = open(os.path.join(ROOT, "include", "moearc_attn.h")).read()
    body = hdr[hdr.index("typedef struct moearc_moe {"):hdr.index("} moearc_moe;")]
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    c = []
    for decl in body.split("{", 1)[1].split(";"):
        if decl.strip():
            c += [re.sub(r"[\*\[\]0-9]", "", n).strip().split()[-1] for n in decl.split(",")]
    rs = open(os.path.join(ROOT, "crates", "moearc-hip", "src", "ffi.rs")).read()
    rs = rs[rs.index("pub struct MoearcMoe {"):]
    assert c == re.findall(r"pub (\w+):", rs[:rs.index("}")]) == [f[0] for f in MoeDesc._fields_]


def test_constants_match_the_header():
    hdr = open(os.path.join(ROOT, "include", "moearc_attn.h")).read()

    def value(name):
        return int(re.search(rf"#define {name} (0x[0-9A-Fa-f]+|\d+)u", hdr).group(1), 0)
    from moearc_amd import NO_EXPERT
    assert value("MOEARC_NO_EXPERT") == NO_EXPERT
    assert [value("MOEARC_ROUTE_SOFTMAX_ALL"), value("MOEARC_ROUTE_SOFTMAX_SELECTED")] == [int(m) for m in RouteMode]
    assert [value("MOEARC_ACT_SWIGLU"), value("MOEARC_ACT_SWIGLU_CLAMPED")] == [int(a) for a in MoeAct]
    assert (OUT_F32, OUT_F16) == (value("MOEARC_OUT_F32"), value("MOEARC_OUT_F16"))


def test_launches_stay_below_the_thread_limit(cx, lib):
    """A launch may not have 2^32 threads: longer calls are cut."""
    def threads():
        return [gx * gy * gz * block for _, gx, gy, gz, block in host_hip.launches(lib)]
    for kw, want in ((dict(n_rows=(1 << 31) - 1, n_cols=1), 16), (dict(n_rows=(1 << 31) - 1, n_cols=2880), 256),
                     (dict(n_rows=1 << 24, n_cols=16388), 8), (dict(n_rows=1 << 23, n_cols=2880), 1)):
        lib.host_hip_reset()
        assert norm(cx, **kw) == 0
        assert len(names(lib)) == want and max(threads()) < 1 << 32
    lib.host_hip_reset()
    assert cx._lib.moearc_moe_route(cx.raw, 64, 64, 64, (1 << 31) - 1, 1024, 4, 1, 1.0) == 0
    assert len(names(lib)) == 16 and max(threads()) < 1 << 32
    for rows, cols in ((1 << 20, 256), (256, 1 << 20), (1 << 20, 1 << 20)):
        for ty in (8, 12):
            lib.host_hip_reset()
            assert linear(cx, ty=ty, n_tok=10000, n_used=4, n_expert=1024, n_rows=rows, n_cols=cols, ws=256, ws_bytes=BIG) == 0
            assert max(threads()) < 1 << 32
    lib.host_hip_reset()
    assert ffn(cx, {"n_embd": 1 << 20, "n_ff": 256}, n_tok=2000, ws=256, ws_bytes=BIG) == 0
    assert max(threads()) < 1 << 32 and _kernels(lib).count("combine") == 8  # 1024 slots at a time
