"""The experts' calls at their largest sizes, on the host alone (host_hip.py)."""
from __future__ import annotations

import ctypes

import pytest

import host_hip
from host_hip import names
from test_moe_dispatch import BIG, built, cx, ffn, lib, linear  # noqa: F401


def _threads(lib):
    return [gx * gy * gz * block for _, gx, gy, gz, block in host_hip.launches(lib)]


@pytest.mark.parametrize("io", [0, 1], ids=["f32", "f16"])
@pytest.mark.parametrize("ty", [1, 8, 12, 13, 14, 39])
def test_wide_gate_and_up_stay_below_the_thread_limit(cx, lib, ty, io):  # noqa: F811
    """A tile of gate and up has half as many rows as one of a product alone."""
    for ff in (1 << 20, (1 << 20) - 256, 1 << 19, 1 << 15, (1 << 14) + 256):
        for used, experts in ((1, 1024), (4, 1024), (4, 8), (511, 1024), (513, 1024), (1023, 1024)):
            lib.host_hip_reset()
            d = {"w_type": [ty] * 3, "n_ff": ff, "n_expert": experts}
            assert ffn(cx, d, io=io, n_tok=2100 // used + 1, n_used=used, ws=256, ws_bytes=BIG) == 0
            assert max(_threads(lib)) < 1 << 32 and any("gu" in n for n in names(lib))


def test_a_token_too_wide_for_a_launch_is_refused(cx, lib):  # noqa: F811
    for ff, rc in ((1 << 20, -2), ((1 << 20) - 32, -2), ((1 << 20) - 64, 0)):
        for tok in (0, 1, 3):
            lib.host_hip_reset()
            assert ffn(cx, {"n_ff": ff, "n_expert": 1024}, n_tok=tok, n_used=1024, ws=256, ws_bytes=BIG) == rc
            assert bool(names(lib)) == (rc == 0 and tok > 0)  # refused before anything is enqueued
            n = ctypes.c_ulong()
            assert cx._lib.moearc_moe_workspace(tok, 1024, 1024, 256, ff, ctypes.byref(n)) == rc


@pytest.mark.parametrize("ff", [512, 1 << 14, 1 << 15, 1 << 20])
def test_the_stated_workspace_is_enough(cx, lib, ff):  # noqa: F811
    """A call takes what moearc_moe_workspace says, no more and no less."""
    n = ctypes.c_ulong()
    for tok in (1, 3, 100, 40000):
        assert cx._lib.moearc_moe_workspace(tok, 4, 8, 256, ff, ctypes.byref(n)) == 0
        for less, rc in ((0, 0), (1, -2)):
            assert ffn(cx, {"n_ff": ff}, n_tok=tok, ws=256, ws_bytes=n.value - less) == rc
    assert linear(cx, n_tok=100, ws=256, ws_bytes=BIG) == 0


def test_the_workspace_refuses_what_the_calls_refuse(cx, lib):  # noqa: F811
    n = ctypes.c_ulong()
    for embd, ff in ((224, 512), (256, 224), (256, 32), (272, 512), (256, 272), (100, 0), (255, 0), (1, 1), ((1 << 20) + 32, 256), (256, (1 << 20) + 32)):
        for tok in (0, 5):
            n.value = 7
            assert cx._lib.moearc_moe_workspace(tok, 4, 8, embd, ff, ctypes.byref(n)) == -2 and n.value == 7
            call = ffn(cx, {"n_embd": embd, "n_ff": ff}, n_tok=tok) if ff else linear(cx, n_cols=embd, n_tok=tok)
            assert call == -2
    for embd, ff in ((256, 0), (288, 0), (256, 288), (1 << 20, 256)):
        assert cx._lib.moearc_moe_workspace(5, 4, 8, embd, ff, ctypes.byref(n)) == 0
