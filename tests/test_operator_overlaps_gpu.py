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
