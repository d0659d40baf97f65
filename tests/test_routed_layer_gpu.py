"""The layer with its own choice of experts (routing, selection bias) and a
shared expert: MoeLayer, the routing stages and ExpertParallelLayer against the
CPU oracle's FFN on the routes that the 64-bit routing restatement gives."""
import ctypes
import os
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

import sparsemoe_b200 as sm
from operator_refs import route_ref
from oracle import oracle as O
from test_int8_linear_gpu import shared_ref

pytestmark = pytest.mark.gpu

SIGMOID = sm.Routing(score="sigmoid", groups=8, kept_groups=4, group_top=2, renormalise=True, scale=2.5)
SOFTMAX = sm.Routing(score="softmax", renormalise=False, scale=16.0)


def bits(t):
    return t.view(torch.int16).cpu().numpy().view(np.uint16)


def shared_weights(d, f, seed=0):
    g = np.random.default_rng(seed)
    out = {}
    for n, (k, m) in (("wg", (d, f)), ("wu", (d, f)), ("wd", (f, d))):
        out["shared_" + n] = g.integers(-127, 128, (k, m)).astype(np.int8)
        out["shared_s" + n[1]] = (g.uniform(0.5, 1.5, m) / (73.0 * np.sqrt(k))).astype(np.float32)
    return out


def slots_of(idx, cfg):
    """Slot of each route in route-id order, -1 where dropped or empty; kept counts [B, E]."""
    cap, slot = cfg.capacity(), np.full(idx.shape, -1, np.int32)
    counts = np.zeros((cfg.num_batches, cfg.num_experts), np.int32)
    for t in range(idx.shape[0]):
        b = t // cfg.tokens
        for l, e in enumerate(idx[t]):
            if e >= 0 and counts[b, e] < cap:
                slot[t, l] = counts[b, e]
                counts[b, e] += 1
    return slot, counts


def reference(cfg, inp, routing, gpu):
    x = inp["x"]
    if inp.get("norm_w") is not None:
        x = O.rmsnorm(x, inp["norm_w"], inp["norm_eps"], cfg.act_bf16)
    r = O.route(x, inp["wr"], inp.get("bias"), cfg.num_batches, cfg.tokens, cfg.d_model, cfg.num_experts, cfg.top_k,
                cfg.capacity(), cfg.act_bf16, cfg.router_f32)
    idx, w = r["idx"], r["w"]
    if routing is not None:
        sb = inp.get("select_bias")
        idx, w = route_ref(torch.from_numpy(r["logits"]), cfg.top_k, routing.score,
                           None if sb is None else torch.from_numpy(sb), routing.groups, routing.kept_groups,
                           routing.group_top, routing.renormalise, routing.scale)
    idx, w = idx.astype(np.int32), w.astype(np.float32)
    slot, counts = slots_of(idx, cfg)
    if cfg.int8ch:
        out = O.ffn_combine_int8ch(x, inp, cfg, idx, w, slot)
    else:
        out = O.ffn_combine(x, inp["wg"], inp["wu"], inp["wd"], cfg.num_batches, cfg.tokens, cfg.d_model, cfg.d_ff,
                            cfg.num_experts, cfg.top_k, cfg.bf16, idx, w, slot)
    t16 = torch.bfloat16 if cfg.act_bf16 else torch.float16
    as16 = lambda a: torch.from_numpy(a.view(np.int16).copy()).view(t16)  # noqa: E731
    if inp.get("residual") is not None:
        out = out + as16(inp["residual"]).float().numpy()
    if inp.get("shared_wg") is not None:
        f = lambda k: torch.from_numpy(inp["shared_" + k])  # noqa: E731
        y, _ = shared_ref(as16(x), f("wg"), f("sg"), f("wu"), f("su"), f("wd"), f("sd"), None)
        out = out + y
    return idx, w, counts, out


def inputs(cfg, seed, select_bias=True, shared=0, norm=False, residual=False):
    inp = sm.make_inputs(cfg, seed)
    g = np.random.default_rng(seed)
    if select_bias:
        inp["select_bias"] = (0.05 * g.standard_normal(cfg.num_experts)).astype(np.float32)
    if shared:
        inp.update(shared_weights(cfg.d_model, shared, seed))
    if norm:
        v = torch.from_numpy((1 + 0.1 * g.standard_normal(cfg.d_model)).astype(np.float32))
        inp["norm_w"], inp["norm_eps"] = bits(v.to(torch.bfloat16 if cfg.act_bf16 else torch.float16)), 1e-5
    if residual:
        inp["residual"] = inp["x"]
    return inp


def check_layer(L, ref, cfg, tol):
    idx, w, counts, out = ref
    np.testing.assert_array_equal(L.idx.cpu().numpy()[: cfg.T], idx)
    np.testing.assert_allclose(L.w.cpu().numpy()[: cfg.T], w, rtol=4e-6, atol=1e-37)
    np.testing.assert_array_equal(L.counts.cpu().numpy()[: cfg.num_batches], counts)
    err = np.abs(L.out.cpu().numpy()[: cfg.T] - out).max() / np.abs(out).max()
    assert err <= tol, err
    if L.out16 is not None:
        assert np.abs(L.out16.float().cpu().numpy()[: cfg.T] - out).max() / np.abs(out).max() <= tol


@pytest.mark.parametrize("dtype, E, k, tol", [(sm.DTYPE_BF16, 64, 6, 1e-2), (sm.DTYPE_F16, 8, 2, 1e-2),
                                              (sm.DTYPE_INT8_CHANNEL, 32, 8, 3e-2)])
@pytest.mark.parametrize("routing", [SIGMOID, SOFTMAX, None], ids=["sigmoid", "softmax", "gate"])
@pytest.mark.parametrize("shared, norm, residual", [(0, False, False), (200, False, True), (384, True, True),
                                                    (96, True, False)])
def test_layer(gpu, dtype, E, k, tol, routing, shared, norm, residual):
    cfg = sm.LayerConfig(2, 150, 512, 256, E, k, 1.0, dtype=dtype, zipf_s=1.0)
    inp = inputs(cfg, E, routing is not None, shared, norm, residual)
    L = sm.MoeLayer(cfg, gpu, routing=routing).load(inp)
    L.forward()
    L.sync_check()
    check_layer(L, reference(cfg, inp, routing, gpu), cfg, tol)


def test_default_routing_equals_the_gate(gpu):
    cfg = sm.LayerConfig(1, 256, 512, 256, 64, 6, 1.25, dtype=sm.DTYPE_BF16, zipf_s=1.0)
    inp = inputs(cfg, 1, select_bias=False)
    a, b = sm.MoeLayer(cfg, gpu).load(inp), sm.MoeLayer(cfg, gpu, routing=sm.Routing()).load(inp)
    a.forward()
    b.forward()
    torch.cuda.synchronize()
    assert torch.equal(a.idx, b.idx) and torch.equal(a.counts, b.counts) and torch.equal(a.logits, b.logits)
    torch.testing.assert_close(a.w, b.w, rtol=2e-6, atol=0)
    torch.testing.assert_close(a.out, b.out, rtol=1e-4, atol=1e-5)


def test_tokens_without_experts(gpu):
    """A bias that masks all but three experts of a top-6 choice: empty slots take no capacity and add nothing."""
    cfg = sm.LayerConfig(1, 100, 256, 128, 64, 6, 1.25, dtype=sm.DTYPE_BF16, cap=-1)
    inp = inputs(cfg, 2)
    inp["select_bias"] = np.full(64, -np.inf, np.float32)
    inp["select_bias"][[5, 17, 40]] = 0.1
    L = sm.MoeLayer(cfg, gpu, routing=SIGMOID).load(inp)
    L.forward()
    L.sync_check()
    assert (L.idx[:100, 3:] == -1).all() and L.counts.sum() == 300
    check_layer(L, reference(cfg, inp, SIGMOID, gpu), cfg, 1e-2)


def test_capture_and_replay(gpu):
    cfg = sm.LayerConfig(1, 64, 512, 256, 64, 6, 1.25, dtype=sm.DTYPE_BF16)
    inp = inputs(cfg, 3, shared=256, residual=True)
    L = sm.MoeLayer(cfg, gpu, routing=SIGMOID).load(inp)
    L.capture()
    x = torch.randn(64, 512, device=gpu).bfloat16()
    L.x[:64].copy_(x)
    L.residual[:64].copy_(x)
    L.replay()
    torch.cuda.synchronize()
    got = L.out.clone()
    L.forward()
    L.sync_check()
    assert torch.equal(got, L.out)


def test_refusals(gpu):
    cfg = sm.LayerConfig(1, 16, 256, 128, 16, 2, 1.25, dtype=sm.DTYPE_BF16)
    inp = inputs(cfg, 4, shared=64)
    with pytest.raises(ValueError, match="routing"):
        sm.MoeLayer(cfg, gpu).load(inp)
    with pytest.raises(ValueError, match="logits"):
        sm.MoeLayer(cfg, gpu, want_logits=False, routing=SOFTMAX)
    with pytest.raises(ValueError, match="shared"):
        sm.MoeLayer(cfg, gpu, routing=SOFTMAX).load({**inp, "shared_wd": inp["shared_wd"][:32]})
    L = sm.MoeLayer(cfg, gpu, routing=sm.Routing(groups=3, kept_groups=2)).load(inp)
    with pytest.raises(sm.MoeError, match="num_groups"):
        L.forward()
    L = sm.MoeLayer(cfg, gpu, routing=SOFTMAX).load(inp)
    st = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    a, dm = L.args(), L.dims()

    def call(fn=sm.lib.moe_solve_v2_ex, args=a, **kw):
        o = L.options()
        for k, v in kw.items():
            setattr(o, k, v)
        return fn(ctypes.byref(args), ctypes.byref(dm), ctypes.byref(o), st)
    b = L.args()
    b.expert_logits = None
    assert call(args=b) == sm.MOE_ERR_INVALID_ARG
    assert call(routing=None) == sm.MOE_ERR_INVALID_ARG            # a bias without a routing
    assert call(fn=sm.lib.moe_stage_route_ex) == sm.MOE_ERR_INVALID_ARG   # a shared expert in a routing stage
    o = L.options()
    o.shared.contents.scratch_bytes = 16
    assert sm.lib.moe_solve_v2_ex(ctypes.byref(a), ctypes.byref(dm), ctypes.byref(o), st) == sm.MOE_ERR_INVALID_ARG
    assert call() == sm.MOE_OK
    L.sync_check()


def test_routing_stages_in_two_phases(gpu):
    """moe_stage_route_counts_ex + _finish leave the tables of moe_solve_v2_ex."""
    cfg = sm.LayerConfig(1, 200, 512, 256, 64, 6, 1.0, dtype=sm.DTYPE_BF16, zipf_s=1.0)
    inp = inputs(cfg, 5)
    L = sm.MoeLayer(cfg, gpu, routing=SIGMOID).load(inp)
    L.forward()
    L.sync_check()
    M = sm.MoeLayer(cfg, gpu, routing=SIGMOID).load(inp)
    raw = torch.zeros(1, 64, dtype=torch.int32, device=gpu)
    a, dm, o = M.args(), M.dims(), M.options()
    st = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    sm.check(sm.lib.moe_stage_route_counts_ex(ctypes.byref(a), ctypes.byref(dm), ctypes.byref(o), raw.data_ptr(), st))
    sm.check(sm.lib.moe_stage_route_finish(ctypes.byref(a), ctypes.byref(dm), st))
    torch.cuda.synchronize()
    assert torch.equal(L.idx, M.idx) and torch.equal(L.w, M.w) and torch.equal(L.counts, M.counts)
    assert raw.sum() == 200 * 6


EP = """
import os, sys, numpy as np, torch, torch.distributed as dist
sys.path[:0] = [{root!r}, {tests!r}]
import sparsemoe_b200 as sm
from sparsemoe_b200.ep import ExpertParallelLayer
from test_routed_layer_gpu import inputs, SIGMOID
os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT={port!r}, NCCL_NVLS_ENABLE="0")
torch.cuda.set_device(0)
from datetime import timedelta
dist.init_process_group("nccl", rank=0, world_size=1, timeout=timedelta(seconds=60), device_id=torch.device("cuda", 0))
cfg = sm.LayerConfig(2, 128, 512, 256, 64, 6, 1.0, dtype=sm.DTYPE_BF16, zipf_s=1.0)
inp = inputs(cfg, 7, shared=200)
single = sm.MoeLayer(cfg, "cuda:0", routing=SIGMOID).load(inp)
want = single.forward().clone()
single.sync_check()
for kw in (dict(), dict(chunks=2), dict(global_batch=True), dict(transport="peer")):
    ep = ExpertParallelLayer(cfg, "cuda:0", routing=SIGMOID, **kw).load(inp)
    out = ep.forward().clone()
    torch.cuda.synchronize()
    assert torch.equal(ep.idx, single.idx) and torch.equal(ep.w, single.w), kw
    assert torch.equal(out[: cfg.T], want[: cfg.T]), kw
    ep.close()
dist.destroy_process_group()
print("ok")
"""


def test_expert_parallel_layer_on_one_rank(gpu):
    root = Path(__file__).resolve().parents[1]
    src = EP.format(root=str(root), tests=str(root / "tests"), port=str(29600 + os.getpid() % 2000))
    r = subprocess.run([sys.executable, "-c", src], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("ok"), r.stdout[-2000:] + r.stderr[-3000:]
