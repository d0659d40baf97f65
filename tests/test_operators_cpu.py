"""Refusals of the stand-alone operators, through the C ABI and Python: checked
before anything is enqueued, so they need no GPU."""
import ctypes

import pytest
import torch

import sparsemoe_b200 as sm

FAKE = 1 << 20   # never dereferenced: every call below is refused first


def routing(**kw):
    a = dict(score=0, num_groups=1, groups_kept=1, group_top=1, renormalise=1, scale=1.0)
    a.update(kw)
    return sm.MoeRouting(**a)


def route(r, typ=0, T=4, E=64, ld=64, k=6, x=FAKE, bias=None, idx=FAKE, w=FAKE):
    return sm.lib.moe_route_experts(x, typ, T, E, ld, k, ctypes.byref(r) if r else None, bias, idx, w, None)


@pytest.mark.parametrize("kw, call", [
    (dict(score=2), {}), (dict(num_groups=0), {}), (dict(num_groups=7), {}), (dict(num_groups=8, groups_kept=0), {}),
    (dict(num_groups=8, groups_kept=9), {}), (dict(group_top=3), {}), (dict(group_top=0), {}),
    (dict(scale=float("nan")), {}), (dict(scale=float("inf")), {}),
    ({}, dict(k=0)), ({}, dict(k=33)), ({}, dict(k=7, E=6, ld=6)), ({}, dict(E=0)), ({}, dict(ld=63)), ({}, dict(T=-1)),
    ({}, dict(typ=3)), ({}, dict(x=None)), ({}, dict(idx=None)), ({}, dict(w=None)), ({}, dict(x=FAKE + 2)),
    ({}, dict(idx=FAKE + 1)), ({}, dict(bias=FAKE + 1))])
def test_route_refusals(kw, call):
    assert route(routing(**kw), **call) == sm.MOE_ERR_INVALID_ARG
    assert sm.lib.moe_last_error()


def test_route_limits_and_null_routing():
    assert route(None) == sm.MOE_ERR_INVALID_ARG
    assert route(routing(), E=1025, ld=1025) == sm.MOE_ERR_UNSUPPORTED
    assert route(routing(), T=1 << 32) == sm.MOE_ERR_UNSUPPORTED
    assert route(routing(), T=0, x=None, idx=None, w=None) == sm.MOE_OK   # nothing to do


def weight(w=FAKE, ld=64, scale=FAKE, order=0):
    return sm.MoeInt8Weight(w, ld, scale, order)


def linear(T=32, K=64, N=64, x=FAKE, typ=2, ldx=64, wt=None, bias=None, out=FAKE, otyp=2, ldo=64, scratch=FAKE,
           n=1 << 20):
    wt = weight() if wt is None else wt
    return sm.lib.moe_int8_linear(x, typ, T, K, ldx, ctypes.byref(wt), N, bias, out, otyp, ldo, scratch, n, None)


BAD_LINEAR = [dict(T=-1), dict(K=0), dict(N=0), dict(x=None), dict(typ=3), dict(typ=-1), dict(ldx=63), dict(x=FAKE + 1),
              dict(out=None), dict(otyp=3), dict(ldo=63), dict(out=FAKE + 1), dict(bias=FAKE + 2), dict(scratch=None),
              dict(scratch=FAKE + 16), dict(n=255),
              dict(wt=weight(w=None)), dict(wt=weight(scale=None)), dict(wt=weight(w=FAKE + 8)), dict(wt=weight(ld=65)),
              dict(wt=weight(ld=48)), dict(wt=weight(order=2)), dict(wt=weight(scale=FAKE + 1)),
              dict(wt=weight(order=1, ld=48))]


@pytest.mark.parametrize("kw", BAD_LINEAR)
def test_linear_refusals(kw):
    assert linear(**kw) == sm.MOE_ERR_INVALID_ARG
    assert sm.lib.moe_last_error()


def test_linear_limits():
    assert linear(K=131072, ldx=131072) == sm.MOE_ERR_UNSUPPORTED
    assert linear(T=1 << 31) == sm.MOE_ERR_UNSUPPORTED
    assert linear(T=0, x=None, out=None, scratch=None, n=0) == sm.MOE_OK
    assert sm.lib.moe_int8_linear_scratch_bytes(50, 100, 64) >= 50 * 112 + 50 * 4
    assert sm.lib.moe_int8_linear_scratch_bytes(1, 7168, 8192) == 0    # a few tokens: one kernel, no scratch
    assert sm.lib.moe_int8_linear_scratch_bytes(1, 7168, 65536) > 0    # more CTAs than run at once
    assert sm.lib.moe_int8_linear_scratch_bytes(1, 131071, 64) > 0  # whose codes do not fit its shared memory
    assert sm.lib.moe_int8_linear_scratch_bytes(-1, 100, 64) == 0


@pytest.mark.parametrize("kw", [
    dict(), dict(out=FAKE + 64), dict(out=FAKE + 128, T=2), dict(out=FAKE - 64), dict(out=FAKE + 100, ldx=100, ldo=100),
    dict(T=1, out=FAKE + 126), dict(T=1, out=FAKE - 126), dict(ldx=128, ldo=128, out=FAKE + 126),
    dict(ldx=128, ldo=128, out=FAKE + 130), dict(otyp=0, ldx=256, ldo=128, out=FAKE + 384)])
def test_outputs_in_the_activations_memory(kw):
    assert linear(**kw) == sm.MOE_ERR_INVALID_ARG
    assert b"shares memory" in sm.lib.moe_last_error()


def test_quantize_and_matmul_refusals():
    q = lambda x=FAKE, typ=2, T=4, K=64, ldx=64, out=FAKE, ldq=64, s=FAKE: sm.lib.moe_int8_quantize_tokens(  # noqa: E731
        x, typ, T, K, ldx, out, ldq, s, None)
    for kw in (dict(x=None), dict(typ=5), dict(K=0), dict(ldx=10), dict(out=None), dict(out=FAKE + 8), dict(ldq=72),
               dict(ldq=48), dict(s=None), dict(s=FAKE + 2)):
        assert q(**kw) == sm.MOE_ERR_INVALID_ARG, kw
    wt = weight()
    m = lambda x=FAKE, ldq=64, s=FAKE, K=64, N=64, out=FAKE, ldo=64: sm.lib.moe_int8_matmul(  # noqa: E731
        x, ldq, s, 4, K, ctypes.byref(wt), N, None, out, 0, ldo, None)
    for kw in (dict(x=None), dict(x=FAKE + 4), dict(ldq=60), dict(ldq=48), dict(s=None), dict(K=0), dict(N=65), dict(out=None),
               dict(ldo=10)):
        assert m(**kw) == sm.MOE_ERR_INVALID_ARG, kw


def test_shared_expert_refusals():
    def call(gate=None, up=None, down=None, res=None, ldr=64, d=64, f=64, scratch=FAKE, n=1 << 20, x=FAKE):
        g, u, dn = gate or weight(), up or weight(), down or weight()
        return sm.lib.moe_int8_shared_expert(x, 2, 4, d, 64, ctypes.byref(g), ctypes.byref(u), ctypes.byref(dn), f, res, ldr,
                                             FAKE, 2, 64, scratch, n, None)
    for kw in (dict(gate=weight(order=1)), dict(up=weight(w=None)), dict(down=weight(ld=16)), dict(res=FAKE, ldr=10),
               dict(res=FAKE + 1), dict(scratch=None), dict(n=100), dict(f=0), dict(d=65), dict(x=None)):
        assert call(**kw) == sm.MOE_ERR_INVALID_ARG, kw


def test_python_refusals_on_cpu_tensors():
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    w, s = torch.zeros(64, 64, dtype=torch.int8), torch.ones(64)
    with pytest.raises(ValueError, match="GPU"):
        sm.route_experts(torch.zeros(4, 64), 6)
    with pytest.raises(ValueError, match="GPU"):
        sm.int8_linear(x, w, s)
    with pytest.raises(ValueError, match="GPU"):
        sm.quantize_int8_tokens(x)
    with pytest.raises(ValueError, match="GPU"):
        sm.int8_matmul(w, s, w, s)
    with pytest.raises(ValueError, match="GPU"):
        sm.int8_shared_expert(x, w, s, w, s, w, s)
    with pytest.raises(ValueError, match="score"):
        sm.Routing(score="tanh").struct()


@pytest.mark.parametrize("shape", [(5, 7), (1, 1), (16, 33), (33, 16)])
@pytest.mark.parametrize("order", ["kn", "nk"])
def test_int8_weight_layout(shape, order):
    a = torch.randint(-128, 128, shape, dtype=torch.int8)
    w = a if order == "kn" else a.t().contiguous().t()
    p = sm.int8_weight(w)
    assert torch.equal(p, a)
    wt = sm.operators.weight_struct(p, torch.ones(shape[1]))
    assert wt.row_stride % 16 == 0 and wt.w == p.data_ptr()
    if min(shape) > 1:
        assert wt.order == (0 if order == "kn" else 1)
        assert wt.row_stride >= (shape[1] if order == "kn" else shape[0])
    with pytest.raises(ValueError, match="int8"):
        sm.int8_weight(p.float())
