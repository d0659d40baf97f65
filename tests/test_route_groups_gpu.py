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
