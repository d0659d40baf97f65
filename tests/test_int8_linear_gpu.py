"""Per-token quantiser, int8 products and the shared expert against 64-bit restatements."""
import math

import numpy as np
import pytest
import torch

import sparsemoe_b200 as sm
from operator_refs import half_step, int8_matrix, matmul_ref, quantize_ref, tiny

pytestmark = pytest.mark.gpu


def tokens(T, K, dtype, seed=0, pad=0, off=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, K + pad + off, generator=g)
    x[:, torch.randint(0, K + pad + off, (max(1, K // 100),), generator=g)] *= 12
    return x.to(dtype).cuda()[:, off: off + K]


# ---- quantiser ---------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T, K", [(1, 1), (3, 7), (5, 64), (9, 1001), (8, 1024), (7, 1032), (4, 4096), (3, 4099), (2, 7168),
                                  (2, 8193), (1, 20000), (700, 96)])
def test_codes_and_scales_are_exact(gpu, dtype, T, K):
    for pad, off in ((0, 0), (8, 8), (3, 1)):
        x = tokens(T, K, dtype, T + K, pad, off)
        q, s = sm.quantize_int8_tokens(x)
        rq, rs = quantize_ref(x)
        np.testing.assert_array_equal(s.cpu().numpy(), rs)
        np.testing.assert_array_equal(q.cpu().numpy(), rq)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_values_on_rounding_borders(gpu, dtype):
    """amax 127 makes s = 1 and the halves ties; other scales put values next to a border."""
    n = torch.arange(-126, 127).double() + 0.5
    near = [n, torch.nextafter(n.float(), torch.tensor(1e9)).double(), torch.nextafter(n.float(), torch.tensor(-1e9)).double()]
    rows = []
    for m in near:
        for scale in (1.0, 2.0 ** -9, 3.0, 1.0 / 3.0, 0.7310585):
            rows.append(torch.cat([m * scale, torch.tensor([127.0 * scale], dtype=torch.float64)]))
    x = torch.stack(rows).to(dtype).cuda()
    q, s = sm.quantize_int8_tokens(x)
    rq, rs = quantize_ref(x)
    np.testing.assert_array_equal(s.cpu().numpy(), rs)
    np.testing.assert_array_equal(q.cpu().numpy(), rq)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [1e-45, 1e-43, 3e-40, 1e-38, 1e-30, 1e-19, 1e19, 1e30, 3e38])
def test_tiny_and_huge_rows(gpu, dtype, size):
    x = (torch.linspace(-1, 1, 255).double() * size).to(dtype).repeat(3, 1).cuda()
    q, s = sm.quantize_int8_tokens(x)
    rq, rs = quantize_ref(x)
    np.testing.assert_array_equal(s.cpu().numpy(), rs)
    np.testing.assert_array_equal(q.cpu().numpy(), rq)


def test_zero_and_broken_rows(gpu):
    x = tokens(6, 300, torch.bfloat16)
    x[1] = 0
    x[2, 17] = math.nan
    x[3, 299] = -math.inf
    q, s = sm.quantize_int8_tokens(x)
    assert s[1] == 1 and (q[1] == 0).all()
    assert torch.isnan(s[2]) and torch.isnan(s[3]) and torch.isfinite(s[[0, 1, 4, 5]]).all()
    w, ws = int8_matrix(torch.Generator().manual_seed(0), 300, 40, "kn", gpu)
    y = sm.int8_linear(x, w, ws)
    assert torch.isnan(y[2:4]).all() and torch.isfinite(y[[0, 1, 4, 5]]).all() and (y[1] == 0).all()


def test_quantiser_writes_its_rows_only(gpu):
    x = tokens(5, 13, torch.bfloat16)
    q = torch.full((7, 32), 55, dtype=torch.int8, device=gpu)
    s = torch.full((7,), 5.0, device=gpu)
    sm.check(sm.lib.moe_int8_quantize_tokens(x.data_ptr(), 2, 5, 13, x.stride(0), q[1:].data_ptr(), 32, s[1:].data_ptr(),
                                             torch.cuda.current_stream().cuda_stream))
    rq, _ = quantize_ref(x)
    np.testing.assert_array_equal(q[1:6, :13].cpu().numpy(), rq)
    assert (q[:, 13:] == 55).all() and (q[0] == 55).all() and (q[6] == 55).all() and s[0] == 5 and s[6] == 5


# ---- product -------------------------------------------------------------------------


def check_linear(x, w, ws, bias, out_dtype, y):
    """Roundings after the exact sum: s32 to f32, two products, the bias sum
    (2^-24 each, of the product's and the bias's magnitudes), the output's half step."""
    rq, rs = quantize_ref(x)
    ref, mag = matmul_ref(rq, rs, w, ws, bias)
    tol = half_step(out_dtype) * np.abs(ref) * 1.01 + 5 * 2.0 ** -24 * mag + tiny(out_dtype)
    err = np.abs(y.cpu().double().numpy() - ref)
    assert y.dtype == out_dtype and y.shape == ref.shape
    assert (err <= tol).all(), f"worst {np.max(err / tol)} of the tolerance"


@pytest.mark.parametrize("order", ["kn", "nk"])
@pytest.mark.parametrize("T, K, N", [
    (1, 1, 1), (1, 16, 16), (1, 7168, 256), (2, 300, 100), (5, 1, 9), (7, 128, 128), (8, 129, 127), (17, 512, 1000),
    (33, 2048, 130), (64, 1000, 64), (127, 256, 300), (128, 384, 512), (129, 100, 257), (200, 1024, 1408),
    (300, 700, 2500), (1000, 260, 700), (2100, 136, 3001)])
def test_shapes(gpu, T, K, N, order):
    g = torch.Generator().manual_seed(T + K + N)
    x = tokens(T, K, torch.bfloat16, T + N)
    w, ws = int8_matrix(g, K, N, order, gpu)
    check_linear(x, w, ws, None, torch.bfloat16, sm.int8_linear(x, w, ws))
    b = torch.randn(N, generator=g).cuda()
    check_linear(x, w, ws, b, torch.float32, sm.int8_linear(x, w, ws, bias=b, out_dtype=torch.float32))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T", [3, 150, 1100])
def test_types(gpu, dtype, out_dtype, T):
    g = torch.Generator().manual_seed(1)
    x = tokens(T, 777, dtype, 2, pad=5, off=3)
    w, ws = int8_matrix(g, 777, 1033, "kn", gpu)
    check_linear(x, w, ws, None, out_dtype, sm.int8_linear(x, w, ws, out_dtype=out_dtype))


def test_sums_at_the_limit_of_s32(gpu):
    """K at its largest with codes and weights at their extremes: |sum| = 127 * 128 * 131071 < 2^31."""
    K = 131071
    x = torch.ones(2, K, dtype=torch.bfloat16, device=gpu)
    x[1] = -1
    store = torch.full((K, 32), -128, dtype=torch.int8, device=gpu)
    w, ws = store[:, :20], torch.ones(20, device=gpu)
    y = sm.int8_linear(x, w, ws, out_dtype=torch.float32)
    check_linear(x, w, ws, None, torch.float32, y)


def test_matmul_takes_codes(gpu):
    g = torch.Generator().manual_seed(4)
    x = tokens(70, 500, torch.float16, 5)
    w, ws = int8_matrix(g, 500, 333, "nk", gpu)
    q, s = sm.quantize_int8_tokens(x)
    a = sm.int8_matmul(q, s, w, ws, out_dtype=torch.float16)
    assert torch.equal(a, sm.int8_linear(x, w, ws))
    q = torch.randint(-128, 128, (70, 512), dtype=torch.int8, device=gpu)[:, :500]   # every code, -128 too
    y = sm.int8_matmul(q, s, w, ws, out_dtype=torch.float32)
    ref, mag = matmul_ref(q.cpu().double().numpy(), s.cpu().numpy(), w, ws)
    assert (np.abs(y.cpu().double().numpy() - ref) <= 5 * 2.0 ** -24 * mag).all()
    one = sm.int8_matmul(q[:1], s[:1], w, ws, out_dtype=torch.float32)
    assert torch.equal(one, y[:1])


@pytest.mark.parametrize("order", ["kn", "nk"])
@pytest.mark.parametrize("K, N", [(7168, 2048), (2048, 7168), (14336, 400), (1000, 2100), (9001, 4300), (129, 40000)])
def test_a_few_tokens(gpu, K, N, order):
    """Every way that few tokens take (rows short and long, K split or not, more tiles than run at once) agrees with
    the codes' product and, bit for bit, with the rows of a large batch."""
    g = torch.Generator().manual_seed(K + N)
    x = tokens(140, K, torch.bfloat16, 11)
    w, ws = int8_matrix(g, K, N, order, gpu)
    b = torch.randn(N, generator=g).cuda()
    whole = sm.int8_linear(x, w, ws, bias=b, out_dtype=torch.float32)
    check_linear(x[:16], w, ws, b, torch.float32, whole[:16])
    q, s = sm.quantize_int8_tokens(x)
    for n in (1, 2, 3, 4, 5, 8, 9, 15, 16, 17):
        assert torch.equal(sm.int8_linear(x[:n], w, ws, bias=b, out_dtype=torch.float32), whole[:n])
        assert torch.equal(sm.int8_matmul(q[:n], s[:n], w, ws, bias=b, out_dtype=torch.float32), whole[:n])


def test_rows_do_not_depend_on_the_batch(gpu):
    """Exact sums: a token's output is the same bits in any batch, tile or split."""
    g = torch.Generator().manual_seed(6)
    x = tokens(3000, 1500, torch.bfloat16, 7)
    w, ws = int8_matrix(g, 1500, 900, "kn", gpu)
    y = sm.int8_linear(x, w, ws, out_dtype=torch.float32)
    for n in (1, 2, 100, 129, 700):
        assert torch.equal(sm.int8_linear(x[:n], w, ws, out_dtype=torch.float32), y[:n])
    assert torch.equal(sm.int8_linear(x, sm.int8_weight(w.t().contiguous().t()), ws, out_dtype=torch.float32), y)


@pytest.mark.parametrize("T", [5, 300, 2500])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("off, ld", [(0, 1024), (8, 1024), (1, 1001), (3, 1024)])
def test_strided_outputs_keep_their_surroundings(gpu, T, out_dtype, off, ld):
    g = torch.Generator().manual_seed(8)
    x = tokens(T, 200, torch.bfloat16, 9)
    w, ws = int8_matrix(g, 200, 900, "kn", gpu)
    want = sm.int8_linear(x, w, ws, out_dtype=out_dtype)
    store = torch.full((T + 2, ld), 7.0, dtype=out_dtype, device=gpu)
    y = sm.int8_linear(x, w, ws, out=store[1: T + 1, off: off + 900])
    assert y.data_ptr() == store[1:, off:].data_ptr() and torch.equal(y, want)
    store[1: T + 1, off: off + 900] = 7.0
    assert (store == 7.0).all()


def test_linear_refusals_on_the_gpu(gpu):
    x = tokens(4, 64, torch.bfloat16)
    w, ws = int8_matrix(torch.Generator().manual_seed(0), 64, 48, "kn", gpu)
    assert sm.int8_linear(x[:0], w, ws).shape == (0, 48)
    bad = torch.zeros(64, 50, dtype=torch.int8, device=gpu)
    for call in (lambda: sm.int8_linear(x, bad, torch.ones(50, device=gpu)),
                 lambda: sm.int8_linear(x, w[:32], ws), lambda: sm.int8_linear(x, w, ws[:40]),
                 lambda: sm.int8_linear(x, w.float(), ws), lambda: sm.int8_linear(x, w.cpu(), ws),
                 lambda: sm.int8_linear(x, w, ws, bias=torch.zeros(3, device=gpu)),
                 lambda: sm.int8_linear(x, w, ws, out_dtype=torch.int32),
                 lambda: sm.int8_linear(x.double(), w, ws), lambda: sm.int8_linear(x[0], w, ws),
                 lambda: sm.int8_linear(x.t().contiguous().t(), w, ws),
                 lambda: sm.int8_linear(x, w, ws, out=torch.empty(4, 47, device=gpu)),
                 lambda: sm.int8_linear(x, w[:, ::2], ws[:24])):
        with pytest.raises(ValueError):
            call()


def test_streams_and_graphs(gpu):
    g = torch.Generator().manual_seed(10)
    w, ws = int8_matrix(g, 2048, 1024, "kn", gpu)
    for T in (1, 64, 2048):
        x = tokens(T, 2048, torch.bfloat16, T)
        want = sm.int8_linear(x, w, ws)
        streams = [torch.cuda.Stream() for _ in range(3)]
        outs = []
        for st in streams:                      # calls that overlap share nothing
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                outs.append([sm.int8_linear(x, w, ws) for _ in range(5)])
        torch.cuda.synchronize()
        assert all(torch.equal(y, want) for o in outs for y in o)
        buf = x.clone()
        graphs = []
        for _ in range(2):
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr):
                y = sm.int8_linear(buf, w, ws)
            graphs.append((gr, y))
        buf.copy_(x.flip(0))
        for gr, _ in graphs:
            gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(y, want.flip(0)) for _, y in graphs)
    sm.check(sm.lib.moe_check_device_status(torch.cuda.current_stream().cuda_stream))


# ---- shared expert -------------------------------------------------------------------


def shared_ref(x, wg, sg, wu, su, wd, sd, residual):
    """f64 shared expert and the tolerance of an f32 one before its output's rounding.

    h carries a relative error of at most (10 + 5 |g|) 2^-23: the roundings of g
    and u (3 each of 2^-24), of silu (an error of g is amplified by at most
    1 + |g|, __expf adds 2 + 1.2 |g| ulp) and of the product.  A code may fall on
    the other side of a border it is nearer to than that error (its own and the
    scale's, which is the largest element's); each such code moves y by one
    step of its weight."""
    q, s = quantize_ref(x)
    g, _ = matmul_ref(q, s, wg, sg)
    u, _ = matmul_ref(q, s, wu, su)
    with np.errstate(over="ignore"):
        h = u * g / (1.0 + np.exp(-g))
    rel = (10 + 5 * np.abs(g)) * 2.0 ** -23
    amax = np.abs(h).max(1, keepdims=True)
    rel_s = np.take_along_axis(rel, np.abs(h).argmax(1)[:, None], 1) + 2.0 ** -24
    sh = np.where(amax > 0, amax / 127.0, 1.0)
    r = h / sh
    qh = np.rint(r)
    loose = np.abs(np.abs(r - np.floor(r)) - 0.5) <= np.abs(r) * (rel + rel_s)
    w = wd.double().cpu().numpy()
    scale = sh * sd.double().cpu().numpy()
    y = (qh @ w) * scale
    tol = (loose.astype(np.float64) @ np.abs(w)) * scale + np.abs(y) * (rel_s + 5 * 2.0 ** -24)
    if residual is not None:
        y = y + residual.double().cpu().numpy()
    return y, tol + 2.0 ** -23 * np.abs(y)


@pytest.mark.parametrize("order", ["kn", "nk"])
@pytest.mark.parametrize("T, d, f", [(1, 512, 256), (1, 33, 7), (3, 100, 130), (64, 256, 1408), (130, 300, 200),
                                     (257, 128, 96), (1500, 256, 1411), (4000, 200, 512)])
def test_shared_expert(gpu, T, d, f, order):
    gen = torch.Generator().manual_seed(T + d + f)
    wg, sg = int8_matrix(gen, d, f, order, gpu)
    wu, su = int8_matrix(gen, d, f, order, gpu)
    wd, sd = int8_matrix(gen, f, d, order, gpu)
    sg, su = sg / math.sqrt(d), su / math.sqrt(d)
    for dtype, with_residual in ((torch.bfloat16, True), (torch.float16, False), (torch.float32, True)):
        x = tokens(T, d, dtype, T)
        r = tokens(T, d, dtype, T + 1) if with_residual else None
        y = sm.int8_shared_expert(x, wg, sg, wu, su, wd, sd, residual=r)
        ref, tol = shared_ref(x, wg, sg, wu, su, wd, sd, r)
        tol = tol + half_step(dtype) * 1.01 * np.abs(ref) + half_step(dtype) * tol + tiny(dtype)
        err = np.abs(y.cpu().double().numpy() - ref)
        assert y.dtype == dtype and (err <= tol).all(), f"worst {np.max(err / tol)} of the tolerance"
        if r is not None:                       # the residual may be the output
            z = r.clone()
            assert torch.equal(sm.int8_shared_expert(x, wg, sg, wu, su, wd, sd, residual=z, out=z), y)


@pytest.mark.parametrize("K", [96, 4096, 7168])
def test_broken_rows_among_a_few(gpu, K):
    x = tokens(16, K, torch.bfloat16, 1)
    x[0, K - 1], x[1], x[2, 17], x[3, K // 2] = math.inf, 0, math.nan, -math.inf
    w, ws = int8_matrix(torch.Generator().manual_seed(0), K, 200, "kn", gpu)
    whole = sm.int8_linear(torch.cat([x, x, x]), w, ws)[:16]
    q, s = sm.quantize_int8_tokens(x)
    for n in (1, 4, 5, 16):
        for y in (sm.int8_linear(x[:n], w, ws), sm.int8_matmul(q[:n], s[:n], w, ws)):
            bad = [t for t in (0, 2, 3) if t < n]
            good = [t for t in range(n) if t not in bad]
            assert torch.isnan(y[bad]).all() and torch.equal(y[good], whole[:n][good])
            assert n < 2 or (y[1] == 0).all()


def test_outputs_beside_and_in_the_inputs(gpu):
    w, ws = int8_matrix(torch.Generator().manual_seed(0), 256, 256, "kn", gpu)
    for T in (1, 3, 16, 200):
        wide = torch.zeros(T, 512, dtype=torch.bfloat16, device=gpu)
        x = wide[:, :256]
        x.copy_(tokens(T, 256, torch.bfloat16, T))
        want = sm.int8_linear(x.clone(), w, ws)
        assert torch.equal(sm.int8_linear(x, w, ws, out=wide[:, 256:]), want)   # the other half of the rows
        for bad in (x, wide[:, 128:384]):
            with pytest.raises(sm.MoeError, match="shares memory"):
                sm.int8_linear(x, w, ws, out=bad)
        ref = sm.int8_shared_expert(x, w, ws, w, ws, w, ws, residual=x.clone())
        with pytest.raises(sm.MoeError, match="shares memory"):
            sm.int8_shared_expert(x, w, ws, w, ws, w, ws, residual=wide[:, 128:384], out=wide[:, 256:])
        assert torch.equal(sm.int8_shared_expert(x, w, ws, w, ws, w, ws, residual=x, out=x), ref)


@pytest.mark.parametrize("d, f", [(2048, 1408), (7168, 600), (300, 9000)])
def test_shared_expert_of_a_few_tokens(gpu, d, f):
    gen = torch.Generator().manual_seed(d + f)
    wg, sg = int8_matrix(gen, d, f, "kn", gpu)
    wu, su = int8_matrix(gen, d, f, "kn", gpu)
    wd, sd = int8_matrix(gen, f, d, "kn", gpu)
    sg, su = sg / math.sqrt(d), su / math.sqrt(d)
    x = tokens(17, d, torch.bfloat16, 3)
    for n in (1, 4, 5, 8, 9, 16, 17):
        y = sm.int8_shared_expert(x[:n], wg, sg, wu, su, wd, sd)
        ref, tol = shared_ref(x[:n], wg, sg, wu, su, wd, sd, None)
        tol = tol + half_step(x.dtype) * (1.01 * np.abs(ref) + tol) + tiny(x.dtype)
        err = np.abs(y.cpu().double().numpy() - ref)
        assert (err <= tol).all(), f"{n} tokens: worst {np.max(err / tol)} of the tolerance"


def test_calls_in_a_row_on_forked_streams(gpu):
    """Kernels that start early: each call reads what the one before it, or another stream's, has just written, in the
    order of the streams; eager and captured, the scratch and outputs reused at once."""
    gen = torch.Generator().manual_seed(8)
    w, ws = int8_matrix(gen, 1024, 1024, "kn", gpu)
    w2, ws2 = int8_matrix(gen, 1024, 1024, "nk", gpu)
    logits_w, logits_s = int8_matrix(gen, 1024, 64, "kn", gpu)
    side = torch.cuda.Stream()

    def run(x, out):
        main = torch.cuda.current_stream()
        a = sm.int8_linear(x, w, ws)
        for _ in range(3):                      # a chain, each link on what the last has written
            a = sm.int8_linear(a, w2, ws2, out=out)
            a = sm.int8_linear(a, w, ws)
        side.wait_stream(main)
        with torch.cuda.stream(side):
            b = sm.int8_linear(a, w2, ws2)
            b = sm.int8_linear(b, w, ws)
        c = sm.int8_linear(a, w, ws)
        main.wait_stream(side)
        lg = sm.int8_linear(b + c, logits_w, logits_s, out_dtype=torch.float32)
        idx, wt = sm.route_experts(lg, 6, score="sigmoid")
        b.record_stream(main)
        return a, b, c, lg, idx, wt

    for T in (1, 4, 12, 40, 700):
        x = tokens(T, 1024, torch.bfloat16, T)
        out = torch.empty(T, 1024, dtype=torch.bfloat16, device=gpu)
        q = lambda a, m, s: sm.int8_linear(a, m, s)  # noqa: E731
        steps = [q(x, w, ws)]
        torch.cuda.synchronize()
        for _ in range(3):
            for m, s in ((w2, ws2), (w, ws)):
                steps.append(q(steps[-1], m, s))
                torch.cuda.synchronize()        # one at a time
        a = steps[-1]
        want = [a, q(q(a, w2, ws2), w, ws), q(a, w, ws)]
        torch.cuda.synchronize()
        want.append(sm.int8_linear(want[1] + want[2], logits_w, logits_s, out_dtype=torch.float32))
        torch.cuda.synchronize()
        want += sm.route_experts(want[3], 6, score="sigmoid")
        torch.cuda.synchronize()
        for _ in range(20):
            got = run(x, out)
        torch.cuda.synchronize()
        assert all(torch.equal(g, h) for g, h in zip(got, want))
        buf = torch.zeros_like(x)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            got = run(buf, out)
        for _ in range(5):
            buf.copy_(x)
            gr.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(g, h) for g, h in zip(got, want))
            buf.zero_()


def test_behind_copies_and_fills(gpu):
    """The kernel before may be none: copies and fills, eager and in a graph."""
    gen = torch.Generator().manual_seed(9)
    w, ws = int8_matrix(gen, 512, 512, "kn", gpu)
    for T in (1, 10, 300):
        x = tokens(T, 512, torch.bfloat16, T)
        want, lg = sm.int8_linear(x, w, ws), tokens(T, 64, torch.float32, 1)
        ridx, rw = sm.route_experts(lg, 4)
        a, b, lb = torch.empty_like(x), torch.empty_like(x), torch.empty_like(lg)

        def run():
            b.zero_()
            a.copy_(x)
            y = sm.int8_linear(a, w, ws)
            b.copy_(y)
            z = sm.int8_matmul(*sm.quantize_int8_tokens(b), w, ws)
            lb.zero_()
            lb.copy_(lg)
            return y, z, *sm.route_experts(lb, 4)

        ref = want, sm.int8_linear(want, w, ws), ridx, rw
        for _ in range(10):
            got = run()
        assert all(torch.equal(g, r) for g, r in zip(got, ref))
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            got = run()
        for _ in range(3):
            gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(g, r) for g, r in zip(got, ref))


def test_calls_from_two_threads(gpu):
    from concurrent.futures import ThreadPoolExecutor
    gen = torch.Generator().manual_seed(12)
    w, ws = int8_matrix(gen, 4096, 900, "kn", gpu)
    xs = [tokens(T, 4096, torch.bfloat16, T) for T in (1, 4, 11, 130)]
    want = [sm.int8_linear(x, w, ws) for x in xs]
    torch.cuda.synchronize()

    def work(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            out = [sm.int8_linear(xs[(i + k) % 4], w, ws) for i in range(40)]
            torch.cuda.current_stream().synchronize()
        return all(torch.equal(y, want[(i + k) % 4]) for i, y in enumerate(out))

    with ThreadPoolExecutor(3) as pool:
        assert all(pool.map(work, range(3)))


def test_shared_expert_refusals_and_graph(gpu):
    gen = torch.Generator().manual_seed(0)
    wg, sg = int8_matrix(gen, 96, 64, "kn", gpu)
    wd, sd = int8_matrix(gen, 64, 96, "kn", gpu)
    x = tokens(9, 96, torch.bfloat16)
    want = sm.int8_shared_expert(x, wg, sg, wg, sg, wd, sd)
    assert sm.int8_shared_expert(x[:0], wg, sg, wg, sg, wd, sd).shape == (0, 96)
    for call in (lambda: sm.int8_shared_expert(x, wg, sg, wg[:, :48], sg[:48], wd, sd),
                 lambda: sm.int8_shared_expert(x, wg, sg, wg, sg, wg, sg),
                 lambda: sm.int8_shared_expert(x, wg, sg, wg, sg, wd, sd, residual=x[:4]),
                 lambda: sm.int8_shared_expert(x, wg, sg, wg, sg, wd, sd, residual=x.float())):
        with pytest.raises(ValueError):
            call()
    nk = sm.int8_weight(wg.t().contiguous().t())
    with pytest.raises(sm.MoeError, match="order"):
        sm.int8_shared_expert(x, wg, sg, nk, sg, wd, sd)
    buf = x.clone()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        y = sm.int8_shared_expert(buf, wg, sg, wg, sg, wd, sd)
    buf.copy_(x.flip(0))
    gr.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want.flip(0))
    sm.check(sm.lib.moe_check_device_status(torch.cuda.current_stream().cuda_stream))
