"""Stand-alone operators next to the layer: expert routing from given logits,
int8 products with token and channel scales, and the int8 shared expert.

Every call runs on torch's current stream of the tensors' device, allocates its
outputs and scratch from torch's allocator (so calls may overlap on several
streams and be captured into CUDA graphs), does not synchronise, and has no
gradient: the library serves models, it does not train them.  Wrong arguments
raise ValueError, failures of the library MoeError.  The waits inside the int8
products are bounded: a product that gives up returns like any other, its
outputs undefined, and the next sync_check() raises.
"""
from __future__ import annotations

import ctypes
import dataclasses
import functools

import torch

from . import _PKG, check, lib
from .config import MOE_SCORES, MOE_WEIGHT_KN, MOE_WEIGHT_NK, MoeInt8Weight, MoeRouting


class _Missing:
    """In the place of a native entry that cannot be loaded: the layer and the C API's mirror work without it, an
    operator's call raises."""

    def __init__(self, reason: ImportError):
        self._reason = reason

    def __getattr__(self, name):
        raise ImportError(f"{_PKG / '_operators.so'}, the entry of the stand-alone operators, cannot be loaded "
                          f"({self._reason}): build it with `python sparsemoe_b200/build.py`") from self._reason


try:
    from . import _operators
    _operators.bind(check, *(ctypes.cast(f, ctypes.c_void_p).value for f in (
        lib.moe_route_experts, lib.moe_int8_quantize_tokens, lib.moe_int8_matmul, lib.moe_int8_linear,
        lib.moe_int8_linear_scratch_bytes, lib.moe_int8_shared_expert, lib.moe_int8_shared_expert_scratch_bytes)))
except ImportError as e:
    _operators = _Missing(e)


def sync_check(device: torch.device | str | int | None = None) -> None:
    """Waits for torch's current stream on `device` (default: the current one) and raises MoeError if a wait inside
    an int8 product has run out on that device since the last check, on any stream (reported once; other calls'
    outputs are not affected), or in the last layer call there."""
    with torch.cuda.device(device):
        check(lib.moe_check_device_status(ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)))


# ---- routing ---------------------------------------------------------------------


@dataclasses.dataclass(frozen=True)
class Routing:
    """How experts are chosen from the logits (MoeRouting in the C API).

    The default is the layer's own gate: the softmax over the top-k logits.
    `score`: "softmax" or "sigmoid"; `groups` / `kept_groups` / `group_top`:
    only experts of the `kept_groups` best of `groups` groups of neighbours,
    a group scored by its largest value or the sum of its two largest;
    `renormalise`: the chosen weights add up to `scale`.
    """

    score: str = "softmax"
    groups: int = 1
    kept_groups: int = 1
    group_top: int = 1
    renormalise: bool = True
    scale: float = 1.0

    def struct(self) -> MoeRouting:
        return _routing(self.score, self.groups, self.kept_groups, self.group_top, self.renormalise, self.scale)


@functools.lru_cache(maxsize=512)
def _routing(score, groups, kept_groups, group_top, renormalise, scale) -> MoeRouting:
    if score not in MOE_SCORES:
        raise ValueError(f"score must be one of {sorted(MOE_SCORES)}, got {score!r}")
    return MoeRouting(MOE_SCORES[score], groups, kept_groups, group_top, 1 if renormalise else 0, scale)


def route_experts(logits: torch.Tensor, top_k: int, *, score: str = "softmax", bias: torch.Tensor | None = None,
                  groups: int = 1, kept_groups: int = 1, group_top: int = 1, renormalise: bool = True,
                  scale: float = 1.0, out: tuple[torch.Tensor, torch.Tensor] | None = None):
    """Experts and weights of each token from its router logits [T, E] (f32,
    f16 or bf16; rows may be strided; E <= 1024, top_k <= 32).

    Returns (indices int32 [T, top_k], weights f32 [T, top_k]), in descending
    order of the experts' values (score + `bias`, a selection bias [E] f32 that
    leaves the weights alone; without one the logits), equal values by the
    lower index, as f64 arithmetic on the logits orders them.  Experts masked
    by a logit that is NaN, -inf, <= -1e20 or f16's lowest value, or by such a
    bias, are never chosen; slots left empty hold (-1, 0).  `out`: the two contiguous
    tensors to write instead.
    """
    spec = _routing(score, groups, kept_groups, group_top, renormalise, scale)
    return _operators.route(logits, top_k, ctypes.addressof(spec), bias, out)


# ---- int8 products ---------------------------------------------------------------


def weight_struct(w: torch.Tensor, scale: torch.Tensor) -> MoeInt8Weight:
    """The C image of an int8 matrix [K, N] that int8_weight() has laid out, and its scales."""
    order, ld = (MOE_WEIGHT_KN, w.stride(0)) if w.stride(1) == 1 else (MOE_WEIGHT_NK, w.stride(1))
    return MoeInt8Weight(w.data_ptr(), (ld + 15) // 16 * 16, scale.data_ptr(), order)


def int8_weight(w: torch.Tensor) -> torch.Tensor:
    """A copy of the int8 matrix w [K, N] in its own axis order whose rows start
    on 16-byte boundaries: what the products take for any K and N (done once,
    when weights are loaded)."""
    if w.dtype != torch.int8 or w.dim() != 2:
        raise ValueError("w must be a 2-D int8 matrix")
    if w.stride(0) == 1 and w.stride(1) != 1:
        return int8_weight(w.t()).t()
    store = torch.zeros(w.shape[0], (w.shape[1] + 15) // 16 * 16, dtype=torch.int8, device=w.device)
    store[:, : w.shape[1]] = w
    return store[:, : w.shape[1]]


def quantize_int8_tokens(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Per-token symmetric int8 of x [T, K]: (q [T, K] int8 with rows on 16-byte
    boundaries, scale [T] f32 = max|x| / 127 -- times f32(1/127) -- or 1 where
    that is zero; q = round-half-even of the exact x / scale).  A row with a NaN
    or an infinity gets a NaN scale."""
    return _operators.quantize(x)


def int8_matmul(q: torch.Tensor, scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, *,
                bias: torch.Tensor | None = None, out_dtype: torch.dtype | None = None,
                out: torch.Tensor | None = None) -> torch.Tensor:
    """(q @ w) * scale[:, None] * w_scale + bias for int8 q [T, K] (rows on
    16-byte boundaries, as quantize_int8_tokens makes them) and w [K, N]
    (either axis contiguous, the other's stride a multiple of 16): s32 sums,
    f32 after them, one rounding to the output type (bf16 by default)."""
    return _operators.matmul(q, scale, w, w_scale, bias, out_dtype, out)


def int8_linear(x: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, *, bias: torch.Tensor | None = None,
                out_dtype: torch.dtype | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """x [T, K] (f32, f16, bf16) times the int8 matrix w [K, N] with f32 scales
    w_scale [N], the tokens quantised on the fly (quantize_int8_tokens, then
    int8_matmul); the output has x's type unless out_dtype or out says otherwise;
    out must share memory with no input."""
    return _operators.linear(x, w, w_scale, bias, out_dtype, out)


def int8_shared_expert(x: torch.Tensor, w_gate: torch.Tensor, s_gate: torch.Tensor, w_up: torch.Tensor,
                       s_up: torch.Tensor, w_down: torch.Tensor, s_down: torch.Tensor, *,
                       residual: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """The shared expert of an MoE layer, an int8 SwiGLU FFN that every token
    takes: h = silu(x Wg) * (x Wu) in f32, y = h Wd (+ residual [T, d] of x's
    type), x and h quantised per token.  Weights as for int8_linear: gate and
    up [d, f] in one axis order, down [f, d].  The output has x's type unless
    `out` (which may be the residual) has another."""
    return _operators.shared(x, w_gate, s_gate, w_up, s_up, w_down, s_down, residual, out)
