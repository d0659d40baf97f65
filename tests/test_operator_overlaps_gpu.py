"""Outputs beside the inputs, in one allocation with them, are taken; in their memory they are refused."""
import pytest
import torch

import sparsemoe_b200 as sm

pytestmark = pytest.mark.gpu


def stream():
    return torch.cuda.current_stream().cuda_stream


@pytest.mark.parametrize("T", [1, 5, 300])
def test_codes_beside_the_activations(gpu, T):
    """Codes and scales behind the activations, and codes in the same rows behind each row's values."""
    x = torch.randn(T, 64, device=gpu).bfloat16()
    q, s = sm.quantize_int8_tokens(x)
    flat = torch.zeros(T * 128 + T * 64 + T * 4, dtype=torch.uint8, device=gpu)
    a, c, d = flat[: T * 128], flat[T * 128: T * 192], flat[T * 192:]
    a.view(torch.bfloat16).copy_(x.flatten())
    sm.check(sm.lib.moe_int8_quantize_tokens(a.data_ptr(), 2, T, 64, 64, c.data_ptr(), 64, d.data_ptr(), stream()))
    assert torch.equal(c.view(torch.int8).view(T, 64), q) and torch.equal(d.view(torch.float32), s)
    wide = torch.zeros(T, 192, dtype=torch.uint8, device=gpu)
    wide[:, :128] = x.view(torch.uint8)
    sm.check(sm.lib.moe_int8_quantize_tokens(wide.data_ptr(), 2, T, 64, 96, wide.data_ptr() + 128, 192, d.data_ptr(),
                                             stream()))
    assert torch.equal(wide[:, 128:].view(torch.int8), q) and torch.equal(wide[:, :128], x.view(torch.uint8))


@pytest.mark.parametrize("T", [1, 7, 5000])
def test_routes_beside_the_logits(gpu, T):
    """The outputs behind the logits in one allocation; in the logits, or one in the other, they are refused."""
    x = torch.randn(T, 64, device=gpu)
    b = 0.1 * torch.randn(64, device=gpu)
    want = sm.route_experts(x, 6, bias=b)
    flat = torch.empty(T * 64 + 2 * T * 6, device=gpu)
    y, i, w = flat[: T * 64].view(T, 64), flat[T * 64: T * 70].view(torch.int32).view(T, 6), flat[T * 70:].view(T, 6)
    y.copy_(x)
    sm.route_experts(y, 6, bias=b, out=(i, w))
    assert torch.equal(i, want[0]) and torch.equal(w, want[1]) and torch.equal(y, x)
    inside = flat[T * 64 - 1: T * 70 - 1].view(T, 6)
    for out in ((inside.view(torch.int32), w), (i, inside), (i, i.view(torch.float32))):
        with pytest.raises(sm.MoeError, match="shares memory"):
            sm.route_experts(y, 6, bias=b, out=out)
