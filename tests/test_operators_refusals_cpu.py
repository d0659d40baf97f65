"""Further refusals of the stand-alone operators: checked before anything is enqueued, so they need no GPU."""
import ctypes

import pytest

import sparsemoe_b200 as sm

FAKE = 1 << 20   # never dereferenced: every call below is refused first


def test_int8_selftest_refusals():
    for ns, written in ((0, FAKE), (-5, FAKE), (10_000_000_001, FAKE), (50_000_000, None), (50_000_000, FAKE + 2)):
        assert sm.lib.moe_selftest_int8_wait_timeout(ns, written, None) == sm.MOE_ERR_INVALID_ARG
        assert b"selftest" in sm.lib.moe_last_error()


@pytest.mark.parametrize("kw", [
    dict(), dict(q=FAKE + 496), dict(q=FAKE - 192), dict(ldx=128, q=FAKE + 112), dict(typ=0, q=FAKE + 512, ldq=256),
    dict(q=FAKE + 4096, s=FAKE + 4096 + 60), dict(q=FAKE + 4096, s=FAKE + 508), dict(q=FAKE + 4096, s=FAKE - 12),
    dict(T=1, q=FAKE + 112), dict(ldx=128, ldq=256, q=FAKE + 64)])
def test_codes_and_scales_in_the_activations_memory(kw):
    """Rows of other blocks are still read where the first codes are written."""
    a = dict(typ=2, T=4, K=64, ldx=64, q=FAKE, ldq=64, s=FAKE + (1 << 16))
    a.update(kw)
    rc = sm.lib.moe_int8_quantize_tokens(FAKE, a["typ"], a["T"], a["K"], a["ldx"], a["q"], a["ldq"], a["s"], None)
    assert rc == sm.MOE_ERR_INVALID_ARG and b"shares memory" in sm.lib.moe_last_error()


@pytest.mark.parametrize("kw", [
    dict(idx=FAKE), dict(w=FAKE), dict(idx=FAKE + 1020), dict(w=FAKE - 92), dict(idx=FAKE + (1 << 16)),
    dict(w=FAKE + (1 << 17) - 92), dict(ld=80, idx=FAKE + 200), dict(bias=FAKE + (1 << 17) + 92),
    dict(bias=FAKE + (1 << 16) - 252), dict(typ=1, w=FAKE + 508), dict(T=1, w=FAKE + 252)])
def test_routes_in_the_logits_memory(kw):
    a = dict(typ=0, T=4, ld=64, bias=None, idx=FAKE + (1 << 17), w=FAKE + (1 << 16))
    a.update(kw)
    r = sm.MoeRouting(0, 1, 1, 1, 1, 1.0)
    rc = sm.lib.moe_route_experts(FAKE, a["typ"], a["T"], 64, a["ld"], 6, ctypes.byref(r), a["bias"], a["idx"], a["w"], None)
    assert rc == sm.MOE_ERR_INVALID_ARG and b"shares memory" in sm.lib.moe_last_error()
