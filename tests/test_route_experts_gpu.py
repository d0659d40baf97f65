"""Expert routing from given logits against a row-by-row 64-bit restatement."""
import math

import numpy as np
import pytest
import torch

import sparsemoe_b200 as sm
from operator_refs import route_ref

pytestmark = pytest.mark.gpu

# Renormalised weights: expf 1 ulp, 1 + e, the division, the sum of k terms
# (k 2^-24), the final division and product: under 16 roundings of 2^-23.
# Unnormalised softmax adds __expf (2 + 1.2 |x - max| ulp, |x - max| <= 20 where
# a term counts) in the sum: under 32 of them.  Both relative; 1e-37 covers the
# subnormal results.
REL = {True: 16 * 2.0 ** -23, False: 32 * 2.0 ** -23}


def check_rows(logits, k, bias=None, score="softmax", groups=1, kept=1, top=1, renorm=True, scale=1.0):
    idx, w = sm.route_experts(logits, k, score=score, bias=bias, groups=groups, kept_groups=kept, group_top=top,
                              renormalise=renorm, scale=scale)
    ri, rw = route_ref(logits, k, score, bias, groups, kept, top, renorm, scale)
    assert idx.dtype == torch.int32 and w.dtype == torch.float32
    np.testing.assert_array_equal(idx.cpu().numpy(), ri)
    np.testing.assert_allclose(w.cpu().double().numpy(), rw, rtol=REL[renorm], atol=1e-37)


def logits_of(T, E, dtype, seed=0, spread=1.6, pad=0):
    g = torch.Generator().manual_seed(seed)
    x = spread * torch.randn(T, E + pad, generator=g) + 0.7 * torch.randn(E + pad, generator=g)
    return x.to(dtype).cuda()[:, :E]


@pytest.mark.parametrize("E, groups, kept, k", [
    (8, 1, 1, 2), (1, 1, 1, 1), (33, 1, 1, 32), (64, 1, 1, 6), (128, 4, 2, 8), (160, 8, 3, 6), (256, 8, 4, 8),
    (256, 16, 5, 8), (244, 4, 2, 7), (255, 5, 2, 9), (96, 32, 9, 4), (288, 36, 3, 6), (512, 8, 8, 10), (1000, 8, 3, 32),
    (1024, 64, 7, 16), (64, 64, 6, 6), (9, 3, 1, 5)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_shapes_types_and_groups(gpu, E, groups, kept, k, score, dtype):
    seed = E * 7 + k
    x = logits_of(37, E, dtype, seed, pad=seed % 9)
    b = 0.1 * torch.randn(E, generator=torch.Generator().manual_seed(seed)).cuda()
    for bias in (None, b):
        for top in (1, 2):
            check_rows(x, k, bias, score, groups, kept, top, renorm=(top == 1) == (bias is None), scale=2.5)


@pytest.mark.parametrize("T", [1, 2, 3, 4, 5, 129])
def test_token_counts(gpu, T):
    check_rows(logits_of(T, 256, torch.float32, T), 8, None, "sigmoid", 8, 4, 2, True, 2.5)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups, kept, top", [(1, 1, 1), (8, 3, 1), (8, 3, 2), (64, 20, 2)])
@pytest.mark.parametrize("with_bias", [False, True])
def test_ties_go_to_the_lower_index(gpu, score, groups, kept, top, with_bias):
    g = torch.Generator().manual_seed(3)
    x = torch.randint(-2, 3, (65, 128), generator=g).float()
    x[0] = 0.0
    x[1, ::2] = -0.0
    x[1, 1::2] = 0.0
    b = (0.25 * torch.randint(-1, 2, (128,), generator=g).float()).cuda() if with_bias else None
    check_rows(x.cuda(), 8, b, score, groups, kept, top, True)
    check_rows(x.bfloat16().cuda(), 8, b, score, groups, kept, top, False)


def test_neighbours_closer_than_f32_scores(gpu):
    """Logits one f32 step apart, whose scores agree in f32, and biases that undo the order of the scores."""
    base = torch.linspace(-6, 6, 40)
    x = torch.stack([base, torch.nextafter(base, torch.tensor(100.0))], 1).reshape(1, 80).repeat(50, 1)
    perm = torch.stack([torch.randperm(80, generator=torch.Generator().manual_seed(i)) for i in range(50)])
    x = x.gather(1, perm).cuda()
    for score in ("softmax", "sigmoid"):
        check_rows(x, 12, None, score)
        check_rows(x, 12, torch.zeros(80).cuda(), score)
        check_rows(x, 12, None, score, 8, 3, 2)
        b = (-torch.sigmoid(x[0].double())).float()       # values near zero, settled by the rounding of the bias
        check_rows(x[:1], 12, b, "sigmoid")
    big = torch.tensor([[30.0, 31.0, 40.0, 50.0, -90.0, -91.0, -200.0, 16.7]]).cuda()   # scores that saturate
    check_rows(big, 8, None, "sigmoid", renorm=False)
    check_rows(big, 3, None, "sigmoid", 4, 2, 1)


MASKS = [float("nan"), -math.inf, -1e20, torch.finfo(torch.float32).min]


@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups, kept, top", [(1, 1, 1), (8, 2, 2), (64, 3, 2)])
@pytest.mark.parametrize("renorm", [True, False])
def test_masks(gpu, mask, score, groups, kept, top, renorm):
    x = logits_of(33, 128, torch.float32, 5)
    hide = torch.rand(33, 128, generator=torch.Generator().manual_seed(1)).cuda() < 0.6
    x[hide] = mask
    x[3] = mask                         # nothing left
    x[4] = mask
    x[4, 77] = -3.0                     # one left
    x[5, : 64] = mask                   # whole groups gone
    b = 0.1 * torch.randn(128, generator=torch.Generator().manual_seed(2)).cuda()
    for bias in (None, b):
        check_rows(x, 8, bias, score, groups, kept, top, renorm)
    idx, w = sm.route_experts(x, 8, score=score)
    assert (idx[3] == -1).all() and (w[3] == 0).all()
    assert idx[4].tolist() == [77] + [-1] * 7


def test_lowest_value_of_each_type_is_a_mask(gpu):
    for dtype in (torch.float16, torch.bfloat16, torch.float32):
        x = logits_of(4, 40, dtype, 6)
        x[:, 10:] = torch.finfo(dtype).min
        check_rows(x, 16, None, "softmax")
        check_rows(x, 16, torch.zeros(40).cuda(), "sigmoid", 4, 2, 2)
        assert (sm.route_experts(x, 16)[0][:, 10:] == -1).all()


def test_infinite_and_extreme_logits(gpu):
    x = logits_of(6, 64, torch.float32, 7)
    x[0, 5] = math.inf
    x[1, 5] = x[1, 60] = math.inf
    x[2] = -300.0 + torch.arange(64).cuda() * 0.5      # every sigmoid below 1e-100
    x[3] = 3e38
    x[4] = -9e19
    for score in ("softmax", "sigmoid"):
        for renorm in (True, False):
            check_rows(x, 6, None, score, renorm=renorm)
            check_rows(x, 6, 0.1 * torch.ones(64).cuda(), score, renorm=renorm)


def test_masking_and_forcing_biases(gpu):
    x = logits_of(9, 64, torch.bfloat16, 8)
    b = torch.zeros(64).cuda()
    b[3], b[4], b[5] = -math.inf, math.nan, -1e20
    b[40] = b[41] = math.inf
    b[50] = 1e30
    for score in ("softmax", "sigmoid"):
        check_rows(x, 8, b, score)
        check_rows(x, 8, b, score, 8, 3, 2)
    idx = sm.route_experts(x, 8, score="sigmoid", bias=b)[0]
    assert (idx[:, 0] == 40).all() and (idx[:, 1] == 41).all() and (idx[:, 2] == 50).all()
    assert not torch.isin(idx, torch.tensor([3, 4, 5], dtype=torch.int32, device=idx.device)).any()


def test_strided_and_misaligned_rows(gpu):
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        store = logits_of(21, 300, dtype, 9)
        for off, E in ((0, 256), (1, 256), (3, 64), (7, 250)):
            x = store[:, off: off + E]
            a = sm.route_experts(x, 6, score="sigmoid", groups=2, kept_groups=1, group_top=2)
            b = sm.route_experts(x.contiguous(), 6, score="sigmoid", groups=2, kept_groups=1, group_top=2)
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        one = store[4:5, :256]
        assert torch.equal(sm.route_experts(one, 4)[0], sm.route_experts(one.clone(), 4)[0])


def test_empty_batch_out_and_refusals(gpu):
    idx, w = sm.route_experts(torch.empty(0, 64, device=gpu), 4)
    assert idx.shape == (0, 4) and w.shape == (0, 4)
    x = logits_of(10, 64, torch.float32)
    guard_i = torch.full((14, 4), 99, dtype=torch.int32, device=gpu)
    guard_w = torch.full((14, 4), 99.0, device=gpu)
    sm.route_experts(x, 4, out=(guard_i[2:12], guard_w[2:12]))
    a, b = sm.route_experts(x, 4)
    assert torch.equal(guard_i[2:12], a) and torch.equal(guard_w[2:12], b)
    assert (guard_i[:2] == 99).all() and (guard_i[12:] == 99).all() and (guard_w[:2] == 99).all() and (guard_w[12:] == 99).all()
    with pytest.raises(sm.MoeError):
        sm.route_experts(x, 65)
    with pytest.raises(sm.MoeError):
        sm.route_experts(x, 4, groups=5)
    for bad in (dict(bias=torch.zeros(63, device=gpu)), dict(bias=torch.zeros(64, dtype=torch.float16, device=gpu)),
                dict(bias=torch.zeros(64)), dict(out=(a[:5], b[:5])), dict(out=(b, a)), dict(score="other")):
        with pytest.raises(ValueError):
            sm.route_experts(x, 4, **bad)
    with pytest.raises(ValueError):
        sm.route_experts(x.t(), 4)
    with pytest.raises(ValueError):
        sm.route_experts(x[0].expand(10, 64), 4)
    with pytest.raises(ValueError):
        sm.route_experts(x.double(), 4)


def test_default_is_the_layers_gate(gpu):
    """softmax over the top-k logits: the same indices, weights within f32 rounding."""
    cfg = sm.LayerConfig(1, 300, 512, 256, 64, 6, 1.25, dtype=sm.DTYPE_BF16)
    layer = sm.MoeLayer(cfg, gpu).load(sm.make_inputs(cfg, 0))
    layer.forward()
    layer.sync_check()
    idx, w = sm.route_experts(layer.logits[: cfg.T], 6)
    assert torch.equal(idx, layer.idx[: cfg.T])
    # the gate divides by (sum + 1e-10), sum >= 1
    torch.testing.assert_close(w, layer.w[: cfg.T], rtol=2e-6, atol=0)


def special_rows(E, dtype):
    """Ties, close neighbours, masked and infinite logits, and ordinary rows between them."""
    x = logits_of(4105 if E <= 64 else 16393, E, torch.float32, E, spread=2.0)   # (four a warp from 4096 or 16384 on)
    g = torch.Generator().manual_seed(E)
    x[10:200] = torch.randint(-2, 3, (190, E), generator=g).float().cuda()
    x[200:230] = 0.0
    x[230:260] = (torch.randint(0, 40, (30, E), generator=g).float() * 2.0 ** -22 + 1.0).cuda()
    x[260:300, ::2] = -math.inf
    x[300:320] = math.nan
    x[320:330, 1:] = -1e20
    x[330] = torch.finfo(torch.float32).min
    x[331, 3] = math.inf
    x[332, [3, E - 1]] = math.inf
    x[333] = -300.0 + torch.arange(E).cuda() * 0.25
    x[-9:] = x[230:239]
    return x.to(dtype)


@pytest.mark.parametrize("E, groups, kept", [(8, 1, 1), (32, 1, 1), (64, 1, 1), (64, 8, 2), (96, 8, 5), (128, 1, 1), (160, 8, 3),
                                             (256, 1, 1), (256, 8, 4)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_large_batches_equal_small_ones(gpu, E, groups, kept, score, dtype):
    """Batches large enough for four tokens a warp choose as the small ones do (which the tests above hold to the definition)."""
    x = special_rows(E, dtype)
    tied = torch.round(torch.randn(E, generator=torch.Generator().manual_seed(9)) * 2) / 16
    for bias in (None, tied.cuda(), (0.1 * torch.randn(E, generator=torch.Generator().manual_seed(1))).cuda()):
        for top in (1, 2):
            for k in (1, min(E, 6), 8):
                kw = dict(score=score, bias=bias, groups=groups, kept_groups=kept, group_top=top, renormalise=top == 1,
                          scale=2.5)
                idx, w = sm.route_experts(x, k, **kw)
                parts = [sm.route_experts(x[i: i + 1500], k, **kw) for i in range(0, x.shape[0], 1500)]
                assert torch.equal(idx, torch.cat([p[0] for p in parts]))
                torch.testing.assert_close(w, torch.cat([p[1] for p in parts]), rtol=2 * REL[top == 1], atol=1e-37)
    # and a sample of the rows against the definition
    rows = torch.tensor([0, 1, 10, 50, 200, 230, 231, 259, 260, 300, 320, 330, 331, 332, 333, 4095, 4100, 4104])
    bias = (0.1 * torch.randn(E, generator=torch.Generator().manual_seed(1))).cuda()
    idx, w = sm.route_experts(x, min(E, 8), score=score, bias=bias, groups=groups, kept_groups=kept, group_top=2)
    ri, rw = route_ref(x[rows.cuda()], min(E, 8), score, bias, groups, kept, 2, True, 1.0)
    np.testing.assert_array_equal(idx[rows.cuda()].cpu().numpy(), ri)
    np.testing.assert_allclose(w[rows.cuda()].cpu().double().numpy(), rw, rtol=REL[True], atol=1e-37)


@pytest.mark.parametrize("groups, kept", [(1, 1), (8, 1), (8, 2)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("k", [5, 6, 7, 8])
def test_large_batches_with_all_choices_in_one_part(gpu, groups, kept, score, k):
    """The best experts neighbours of each other, closer than f32 scores tell apart: the border behind the last
    choice lies within them."""
    x = logits_of(16800, 256, torch.float32, 21)
    g = torch.Generator().manual_seed(k)
    close = (torch.rand(16800, 32, generator=g).argsort(1).float() * 2.0 ** -22 + 4.0).cuda()
    x[:, 64:96] = close                        # one part of 32 holds every choice
    x[2000:3000, 96:98] = 4.0                  # and ties with it in the next
    b = (torch.round(torch.randn(256, generator=g) * 2) / 64).cuda()
    b[64:96] = 0.25
    for bias in (None, b, torch.zeros(256).cuda()):
        for top in (1, 2):
            kw = dict(score=score, bias=bias, groups=groups, kept_groups=kept, group_top=top)
            idx, w = sm.route_experts(x, k, **kw)
            parts = [sm.route_experts(x[i: i + 8400], k, **kw) for i in (0, 8400)]
            assert torch.equal(idx, torch.cat([p[0] for p in parts]))
            ri, _ = route_ref(x[1995:2005], k, score, bias, groups, kept, top, True, 1.0)
            np.testing.assert_array_equal(idx[1995:2005].cpu().numpy(), ri)


def test_streams_and_graphs(gpu):
    x = logits_of(500, 256, torch.float32, 11)
    kw = dict(score="sigmoid", groups=8, kept_groups=4, group_top=2, bias=torch.zeros(256, device=gpu), scale=2.5)
    want = sm.route_experts(x, 8, **kw)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        y = x.clone()
        got = sm.route_experts(y, 8, **kw)
    st.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    buf = x.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = sm.route_experts(buf, 8, **kw)
    buf.copy_(x.flip(0))
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out[0], want[0].flip(0)) and torch.equal(out[1], want[1].flip(0))
