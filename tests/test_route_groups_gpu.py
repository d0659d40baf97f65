"""The order of expert groups against 64-bit arithmetic where f32 scores cannot tell it: biases that cancel in a group,
scores far below one, sums that are equal.  Batches below and above the sizes from which a warp takes four tokens."""
import numpy as np
import pytest
import torch

import sparsemoe_b200 as sm

pytestmark = pytest.mark.gpu


def chosen(x, b, score, groups, kept, top, k):
    """Indices [T, k] of finite logits from the definition, all rows at once: f64 scores, sums of the `top` largest of
    each group; equal are sums that agree to 2^-49 of what they are summed from."""
    T, E = x.shape
    per = E // groups
    with np.errstate(over="ignore"):
        if score == "sigmoid":
            s = 1.0 / (1.0 + np.exp(-x))
        else:
            e = np.exp(x - x.max(1, keepdims=True))
            s = e / e.sum(1, keepdims=True)
    value = x if b is None else s + b
    member = (s if b is None else value).reshape(T, groups, per)
    at = np.argsort(-member, axis=2, kind="stable")[:, :, :top]
    best = np.take_along_axis(member, at, 2)
    marks = best.sum(2)
    size = np.abs(best)
    if b is not None:
        size = size + np.abs(np.take_along_axis(np.broadcast_to(b.reshape(1, groups, per), member.shape), at, 2))
    tie = 2.0 ** -49 * size.sum(2) if top == 2 else np.zeros((T, groups))
    stay = np.zeros((T, groups), bool)
    for _ in range(kept):
        left = np.where(stay, -np.inf, marks)
        m = left.argmax(1)
        rows = np.arange(T)
        reach = np.where(stay, -np.inf, marks + tie) >= (marks[rows, m] - tie[rows, m])[:, None]
        stay[rows, reach.argmax(1)] = True
    value = np.where(np.repeat(stay, per, axis=1), value, -np.inf)
    return np.argsort(-value, axis=1, kind="stable")[:, :k]


def check(x, b, score, groups, kept, top, k, parts=4000):
    """The whole batch, and its rows in batches of a warp a token."""
    want = chosen(x.double().cpu().numpy(), None if b is None else b.double().cpu().numpy(), score, groups, kept, top, k)
    kw = dict(score=score, bias=b, groups=groups, kept_groups=kept, group_top=top)
    for step in (x.shape[0], parts):
        idx = torch.cat([sm.route_experts(x[i: i + step], k, **kw)[0] for i in range(0, x.shape[0], step)]).cpu().numpy()
        wrong = (idx != want).any(1)
        assert not wrong.any(), f"{wrong.sum()} of {len(wrong)} rows, {(idx[wrong] < 0).any(1).sum()} of them with empty slots"


@pytest.mark.parametrize("size", [1e3, 1e4, 1e6])
@pytest.mark.parametrize("E, T", [(16, 20000), (32, 20000), (256, 20000)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_biases_that_cancel_in_a_group(gpu, size, E, T, score):
    """One expert of each group forced, the others forbidden: sums of two near zero whose members' f32 steps are larger."""
    g = torch.Generator().manual_seed(E)
    x = (1.6 * torch.randn(T, E, generator=g)).cuda()
    b = torch.full((8, E // 8), -size)
    b[torch.arange(8), torch.randint(0, E // 8, (8,), generator=g)] = size
    check(x, b.flatten().cuda(), score, 8, 4, 2, 4)
    check(x, (b.flatten() + 0.1 * torch.randn(E, generator=g)).cuda(), score, 8, 3, 2, 4)
    check(x, b.flatten().cuda(), score, 8, 4, 1, 4)


# (experts, groups, tokens): groups of whole lanes, groups inside lanes and across them, more than 32 groups, groups of one
SHAPES = [(256, 8, 17000), (64, 8, 6000), (32, 8, 6000), (160, 8, 17000), (256, 4, 3000), (244, 4, 3000), (96, 32, 3000),
          (288, 36, 1000), (1024, 64, 300), (8, 8, 3000)]


@pytest.mark.parametrize("E, groups, T", SHAPES)
@pytest.mark.parametrize("mean", [-30.0, -40.0, -300.0])
def test_small_sigmoids(gpu, E, groups, T, mean):
    """Scores far below one, whose sums differ by far less than 2^-49."""
    g = torch.Generator().manual_seed(E)
    x = (1.6 * torch.randn(T, E, generator=g) + mean).cuda()
    zero = torch.zeros(E, device=gpu)
    for kept in sorted({1, groups // 2, groups - 1} - {0}):
        k = min(8, kept * (E // groups))
        check(x, None, "sigmoid", groups, kept, 2, k)
    check(x, zero, "sigmoid", groups, 1, 2, 1)
    check(x, (1e-14 * torch.randn(E, generator=g)).cuda(), "sigmoid", groups, 1, 2, 1)


@pytest.mark.parametrize("E, groups, T", SHAPES)
@pytest.mark.parametrize("spread", [16.0, 80.0])
def test_softmax_of_wide_logits(gpu, E, groups, T, spread):
    g = torch.Generator().manual_seed(E)
    x = (spread * torch.randn(T, E, generator=g)).cuda()
    for kept in sorted({1, groups // 2, groups - 1} - {0}):
        k = min(8, kept * (E // groups))
        check(x, None, "softmax", groups, kept, 2, k)
    check(x, torch.zeros(E, device=gpu), "softmax", groups, 1, 2, 1)


@pytest.mark.parametrize("E, groups, T", [(32, 8, 4200), (64, 16, 50), (320, 40, 50)])
def test_sums_each_equal_to_the_next(gpu, E, groups, T):
    """Group sums 1 + 3 j 2^-50 in any order: neighbours are equal, others are not.  As many groups stay as are asked for."""
    x = torch.zeros(T, E, device=gpu)
    for seed in range(6):
        order = torch.randperm(groups, generator=torch.Generator().manual_seed(seed))
        b = torch.full((groups, E // groups), -1.0)
        b[:, 0] = 0.0
        b[:, 1] = 3.0 * order * 2.0 ** -50
        b = b[:, torch.randperm(E // groups, generator=torch.Generator().manual_seed(seed))].flatten().cuda()
        for kept in (1, 2, 5, groups - 1):
            check(x, b, "sigmoid", groups, kept, 2, min(2 * kept, 8), parts=40)


@pytest.mark.parametrize("E, groups, T", SHAPES[:-1])
def test_mirrored_sigmoids_are_equal(gpu, E, groups, T):
    """sigmoid(x) + sigmoid(-x) is one for every x: the first groups stay."""
    g = torch.Generator().manual_seed(E)
    half = 5.0 * torch.rand(T, groups, 1, generator=g) + 0.1
    x = torch.cat([half, -half, torch.full((T, groups, E // groups - 2), -7.0)], 2).reshape(T, E).cuda()
    kept = groups // 2
    want = chosen(x.double().cpu().numpy(), None, "sigmoid", groups, kept, 2, kept)
    assert (want // (E // groups) < kept).all()
    check(x, None, "sigmoid", groups, kept, 2, min(kept, 8))


@pytest.mark.parametrize("E, part, T", [(1024, 32, 200), (1024, 32, 3), (256, 32, 17000), (512, 16, 100)])
def test_sums_that_round_one_way(gpu, E, part, T):
    """Softmax sums of 1 + 2^-24 + 2^-24 + .., every addition of a lane rounded up by nearly half a step, and biases
    that leave values of the size of that error."""
    x = torch.full((E // part, part), -16.6353)     # exp: 2^-24 (1 + 2^-12)
    x[:, 0] = 0.0
    x[: E // part // 2, 1] = -16.0
    x = x.flatten().repeat(T, 1)
    s = torch.softmax(x[0].double(), 0)
    for seed in range(4):
        g = torch.Generator().manual_seed(seed)
        b = (-s + 40 * 2.0 ** -23 * s.max() * torch.randn(E, generator=g, dtype=torch.float64)).float()
        for kept, groups, top in ((1, 1, 1), (3, 8, 1), (3, 8, 2)):
            check(x.cuda(), b.cuda(), "softmax", groups, kept, top, 8)
