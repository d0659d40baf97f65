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


FAR = [FAKE + (i << 20) for i in range(1, 12)]   # memory apart


def apart(order=0, **kw):
    a = dict(x=FAR[0], out=FAR[1], scratch=FAR[2], w=FAR[3], ws=FAR[4], bias=FAR[5], s=FAR[6])
    a.update(kw)
    return a, sm.MoeInt8Weight(a["w"], 64, a["ws"], order)


@pytest.mark.parametrize("kw", [
    dict(out=FAR[3]), dict(out=FAR[3] + 63 * 64), dict(out=FAR[3] + 63 * 64, order=1), dict(out=FAR[4] + 252),
    dict(out=FAR[5] - 32 * 128 + 2), dict(out=FAR[2]), dict(out=FAR[2] + 32 * 64), dict(x=FAR[2]),
    dict(x=FAR[2] - 32 * 128 + 2)])
def test_linear_outputs_in_an_inputs_memory(kw):
    a, w = apart(**kw)
    rc = sm.lib.moe_int8_linear(a["x"], 2, 32, 64, 64, ctypes.byref(w), 64, a["bias"], a["out"], 2, 64, a["scratch"],
                                1 << 18, None)
    assert rc == sm.MOE_ERR_INVALID_ARG and b"shares memory" in sm.lib.moe_last_error()


@pytest.mark.parametrize("kw", [dict(out=FAR[6]), dict(out=FAR[6] + 124), dict(out=FAR[3] + 64), dict(out=FAR[4]),
                                dict(out=FAR[5] + 252), dict(out=FAR[0] + 31 * 64 + 62)])
def test_matmul_outputs_in_an_inputs_memory(kw):
    a, w = apart(**kw)
    rc = sm.lib.moe_int8_matmul(a["x"], 64, a["s"], 32, 64, ctypes.byref(w), 64, a["bias"], a["out"], 2, 64, None)
    assert rc == sm.MOE_ERR_INVALID_ARG and b"shares memory" in sm.lib.moe_last_error()


@pytest.mark.parametrize("kw", [dict(out=FAR[2]), dict(out=FAR[3]), dict(out=FAR[4]), dict(out=FAR[7]), dict(out=FAR[8] + 252),
                                dict(out=FAR[9] + 64), dict(x=FAR[2] + 64), dict(res=FAR[2]), dict(res=FAR[1] + 2),
                                dict(res=FAR[1], ldr=72)])
def test_shared_expert_outputs_in_an_inputs_memory(kw):
    ldr = kw.pop("ldr", 64)
    a, gate = apart(**kw)
    up, down = sm.MoeInt8Weight(FAR[7], 64, FAR[8], 0), sm.MoeInt8Weight(FAR[9], 64, FAR[10], 0)
    rc = sm.lib.moe_int8_shared_expert(a["x"], 2, 32, 64, 64, ctypes.byref(gate), ctypes.byref(up), ctypes.byref(down), 64,
                                       a.get("res"), ldr, a["out"], 2, 64, a["scratch"], 1 << 18, None)
    assert rc == sm.MOE_ERR_INVALID_ARG and b"shares memory" in sm.lib.moe_last_error()
