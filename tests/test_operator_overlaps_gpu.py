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


@pytest.mark.parametrize("T", [1, 6, 12, 300])
def test_products_in_one_allocation(gpu, T):
    """Everything a call reads and writes in one buffer, side by side; one element into a neighbour is refused."""
    K = N = 128
    x = torch.randn(T, K, device=gpu).bfloat16()
    w = torch.randint(-127, 128, (K, N), dtype=torch.int8, device=gpu)
    s, b = torch.rand(N, device=gpu) * 0.01, torch.randn(N, device=gpu)
    want, plain = sm.int8_linear(x, w, s, bias=b), sm.int8_shared_expert(x, w, s, w, s, w, s)
    flat = torch.zeros(2 * T * K * 2 + K * N + 2 * N * 4 + 64, dtype=torch.uint8, device=gpu)
    at = 0

    def place(t):
        nonlocal at
        v = flat[at: at + t.numel() * t.element_size()].view(t.dtype).view(t.shape)
        at += v.numel() * v.element_size()
        return v.copy_(t)

    fx, fw, fs, fo, fb = place(x), place(w), place(s), place(torch.zeros_like(x)), place(b)
    assert torch.equal(sm.int8_linear(fx, fw, fs, bias=fb, out=fo), want)
    q, sq = sm.quantize_int8_tokens(fx)
    assert torch.equal(sm.int8_matmul(q, sq, fw, fs, bias=fb, out=fo), want)
    assert torch.equal(sm.int8_shared_expert(fx, fw, fs, fw, fs, fw, fs, out=fo), plain)
    half = flat.view(torch.bfloat16)
    first = (fo.data_ptr() - flat.data_ptr()) // 2
    for off in (-1, 1):                          # into the scales before it, the bias behind it
        out = half[first + off: first + off + T * N].view(T, N)
        for call in (lambda: sm.int8_linear(fx, fw, fs, bias=fb, out=out),
                     lambda: sm.int8_matmul(q, sq, fw, fs, bias=fb, out=out)):
            with pytest.raises(sm.MoeError, match="shares memory"):
                call()
    with pytest.raises(sm.MoeError, match="shares memory"):
        sm.int8_shared_expert(fx, fw, fs, fw, fs, fw, fs, out=half[first - 1: first - 1 + T * N].view(T, N))
    # the activations' own memory: they have been read by the time the output is written
    assert torch.equal(sm.int8_shared_expert(fx, fw, fs, fw, fs, fw, fs, out=fx), plain)
