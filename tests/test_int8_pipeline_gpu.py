"""The pipelines of the int8 products from start to end: K of fewer and more blocks than there are stages, tiles of
one CTA, of clusters and of CTA pairs, launch behind launch, so that a stage whose last release is missed or waited
for in the wrong phase shows as a wait that runs out or as a wrong sum."""
import pytest
import torch

import sparsemoe_b200 as sm

pytestmark = pytest.mark.gpu


def codes(gen, T, K, N, gpu):
    """Codes, weights whose sums stay below 2^24 (so that f32 holds them), and scales of one."""
    q = torch.randint(-127, 128, (T, (K + 15) // 16 * 16), generator=gen, dtype=torch.int8, device=gpu)[:, :K]
    w = sm.int8_weight(torch.randint(-8, 9, (K, N), generator=gen, dtype=torch.int8, device=gpu))
    return q, w, torch.ones(T, device=gpu), torch.ones(N, device=gpu)


# few tokens, one tile a CTA, clusters that split K, several tiles a CTA, CTA pairs (from 2 blocks of K on at this size)
@pytest.mark.parametrize("T, N", [(3, 600), (16, 600), (130, 300), (700, 2000), (16384, 4097)])
def test_every_number_of_blocks(gpu, T, N):
    gen = torch.Generator(device=gpu).manual_seed(T)
    side = torch.cuda.Stream()
    for K in [128 * b - 37 for b in range(1, 14)]:
        q, w, s, ws = codes(gen, T, K, N, gpu)
        want = q.float() @ w.float()
        side.wait_stream(torch.cuda.current_stream())
        outs = [sm.int8_matmul(q, s, w, ws, out_dtype=torch.float32) for _ in range(4)]
        with torch.cuda.stream(side):
            outs += [sm.int8_matmul(q, s, w, ws, out_dtype=torch.float32) for _ in range(4)]
        torch.cuda.synchronize()
        for y in outs:
            assert torch.equal(y, want), K
        del outs
    sm.check(sm.lib.moe_check_device_status(torch.cuda.current_stream().cuda_stream))


def test_fused_gate_and_up_of_every_number_of_blocks(gpu):
    """The gate and up columns of a pair's tile: the same rows from a large batch and from one without pairs."""
    gen = torch.Generator(device=gpu).manual_seed(1)
    f = 2048
    for K in [128 * b - 37 for b in range(1, 14)]:
        x = torch.randn(8192, K, generator=gen, device=gpu).bfloat16()
        wg, wu = (sm.int8_weight(torch.randint(-127, 128, (K, f), generator=gen, dtype=torch.int8, device=gpu)) for _ in "gu")
        wd = sm.int8_weight(torch.randint(-127, 128, (f, K), generator=gen, dtype=torch.int8, device=gpu))
        sg, sd = torch.full((f,), 1e-3, device=gpu), torch.full((K,), 1e-3, device=gpu)
        y = [sm.int8_shared_expert(x, wg, sg, wu, sg, wd, sd) for _ in range(3)]
        part = sm.int8_shared_expert(x[:300], wg, sg, wu, sg, wd, sd)
        assert all(torch.equal(z, y[0]) for z in y[1:])
        assert torch.equal(y[0][:300], part), K
    sm.check(sm.lib.moe_check_device_status(torch.cuda.current_stream().cuda_stream))


def test_a_wait_that_ran_out_stops_no_other_call(gpu):
    """A cluster whose wait runs out after 50 ms leaves a report for the host: products behind it, of every kind of
    tile, are not touched by it, and the report comes once."""
    gen = torch.Generator(device=gpu).manual_seed(2)
    sm.sync_check()
    cases = []
    for T, K, N in ((3, 7168, 600), (16, 900, 600), (130, 131071, 300), (700, 2048, 2000), (16384, 1024, 4097)):
        q, w, s, ws = codes(gen, T, K, N, gpu)
        cases.append((q, s, w, ws, sm.int8_matmul(q, s, w, ws, out_dtype=torch.float32)))
    sm.sync_check()
    written = torch.zeros(2, dtype=torch.int32, device=gpu)
    sm.check(sm.lib.moe_selftest_int8_wait_timeout(50_000_000, written.data_ptr(),
                                                   torch.cuda.current_stream().cuda_stream))
    got = [sm.int8_matmul(q, s, w, ws, out_dtype=torch.float32) for q, s, w, ws, _ in cases]
    with pytest.raises(sm.MoeError, match="int8 product"):
        sm.sync_check()
    assert all(torch.equal(y, c[-1]) for y, c in zip(got, cases))
    sm.sync_check(gpu)
    y = sm.int8_matmul(*cases[0][:4], out_dtype=torch.float32)
    sm.sync_check("cuda:0")
    assert torch.equal(y, cases[0][-1])


def test_no_cta_of_a_cluster_writes_behind_a_wait_that_ran_out(gpu):
    """The CTA that sums up the parts of a cluster learns that another one has given up."""
    written = torch.zeros(2, dtype=torch.int32, device=gpu)
    sm.check(sm.lib.moe_selftest_int8_wait_timeout(20_000_000, written.data_ptr(),
                                                   torch.cuda.current_stream().cuda_stream))
    with pytest.raises(sm.MoeError, match="int8 product"):
        sm.sync_check()
    assert written.tolist() == [0, 0]
