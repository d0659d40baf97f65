"""Weights of chosen experts whose scores lie many orders of magnitude apart, against 64-bit arithmetic."""
import numpy as np
import pytest
import torch

import sparsemoe_b200 as sm

pytestmark = pytest.mark.gpu

# 16 roundings of 2^-23 (expf, 1 + e, the reciprocal, a product, the sum of up to 8, the division, the scale); d 2^-24
# more where the ratio is the exp of a rounded difference d of logits; and 2 ulp of subnormal scores over the smallest
# sum that they are divided by, 2^-26: 2^-148 2^26 2.5 < 1e-36.
ATOL = 1e-36


@pytest.mark.parametrize("E, T", [(16, 500), (64, 5000), (256, 17000)])
@pytest.mark.parametrize("mean, spread", [(-40.0, 20.0), (-75.0, 10.0), (-80.0, 30.0), (-17.0, 2.0), (0.0, 40.0)])
def test_renormalised_sigmoids_far_apart(gpu, E, T, mean, spread):
    g = torch.Generator().manual_seed(E)
    x = mean + spread * torch.randn(T, E, generator=g)
    pick = torch.randn(E, generator=g)
    for bias in (None, 10.0 * pick):             # by the logits, and by a bias alone, the score of any size
        idx, w = sm.route_experts(x.cuda(), 8, score="sigmoid", bias=None if bias is None else bias.cuda(), scale=2.5)
        idx, w = idx.cpu().numpy(), w.cpu().double().numpy()
        lx = np.take_along_axis(x.double().numpy(), idx, 1)
        ls = np.minimum(lx, 0.0) - np.log1p(np.exp(-np.abs(lx)))     # log sigmoid
        d = ls.max(1, keepdims=True) - ls
        want = 2.5 * np.exp(-d) / np.exp(-d).sum(1, keepdims=True)
        worst = (np.abs(w - want) / (want * (16 + d / 2) * 2.0 ** -23 + ATOL)).max()
        assert worst <= 1, worst
