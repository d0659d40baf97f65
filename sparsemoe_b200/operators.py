"""Stand-alone operators next to the layer: expert routing from given logits,
int8 products with token and channel scales, and the int8 shared expert.

Every call runs on torch's current stream of the tensors' device, allocates its
outputs and scratch from torch's allocator (so calls may overlap on several
streams and be captured into CUDA graphs), does not synchronise, and has no
gradient: the library serves models, it does not train them.  Wrong arguments
raise ValueError, failures of the library MoeError.
"""
from __future__ import annotations

import ctypes
import dataclasses
import functools

import torch

from . import check, lib
from .config import (MOE_SCORES, MOE_TYPE_BF16, MOE_TYPE_F16, MOE_TYPE_F32, MOE_WEIGHT_KN, MOE_WEIGHT_NK,
                     MoeInt8Weight, MoeRouting)

_TYPE = {torch.float32: MOE_TYPE_F32, torch.float16: MOE_TYPE_F16, torch.bfloat16: MOE_TYPE_BF16}
_ref = ctypes.byref
_empty = torch.empty        # (sizes are given one by one: a tuple of them takes torch's parser longer)
_i32, _f32, _i8, _u8 = torch.int32, torch.float32, torch.int8, torch.uint8
_device = torch.cuda.current_device
_raw_stream = torch._C._cuda_getCurrentRawStream   # the handle alone: current_stream() builds an object first
_route_fn, _linear_fn, _shared_fn = lib.moe_route_experts, lib.moe_int8_linear, lib.moe_int8_shared_expert
_linear_scratch = functools.lru_cache(maxsize=4096)(lib.moe_int8_linear_scratch_bytes)
_shared_scratch = functools.lru_cache(maxsize=4096)(lib.moe_int8_shared_expert_scratch_bytes)


def _call(index: int, fn, *args) -> None:
    """fn(*args, stream) on device `index` and torch's current stream there."""
    if _device() == index:
        rc = fn(*args, _raw_stream(index))
        if rc:
            check(rc)
        return
    prev = _device()
    torch.cuda.set_device(index)
    try:
        check(fn(*args, _raw_stream(index)))
    finally:
        torch.cuda.set_device(prev)


def _rows(t: torch.Tensor, name: str) -> tuple[int, int, int]:
    """(rows, columns, row stride) of a 2-D tensor whose rows are contiguous."""
    if t.dim() != 2:
        raise ValueError(f"{name} must be 2-D, got shape {tuple(t.shape)}")
    rows, cols = t.shape
    ld, step = t.stride()
    if step != 1 and cols > 1:
        raise ValueError(f"{name}: the elements of a row must be contiguous")
    if ld < cols:
        if rows > 1:
            raise ValueError(f"{name}: rows overlap (stride {ld} for {cols} columns)")
        ld = cols
    return rows, cols, ld


def _vector(t, n: int, name: str, index: int):
    if t is None:
        return None
    if t.dtype != torch.float32 or t.shape != (n,) or (n > 1 and t.stride(0) != 1) or t.get_device() != index:
        raise ValueError(f"{name} must be a contiguous f32 vector of {n} on cuda:{index}")
    return t.data_ptr()


def _output(out, rows: int, cols: int, dtype, like: torch.Tensor):
    """(tensor, MOE_TYPE_*, row stride) of the output: `out`, or a new tensor of `dtype`."""
    if out is None:
        kind = _TYPE.get(dtype)
        if kind is None:
            raise ValueError(f"the output must be f32, f16 or bf16, not {dtype}")
        return _empty(rows, cols, dtype=dtype, device=like.device), kind, cols
    kind = _TYPE.get(out.dtype)
    if kind is None or out.shape != (rows, cols) or out.get_device() != like.get_device() or \
            (dtype is not None and out.dtype != dtype):
        raise ValueError(f"out must be f32, f16 or bf16 of shape {(rows, cols)} on {like.device}"
                         + (f" and {dtype}" if dtype is not None else ""))
    return out, kind, _rows(out, "out")[2]


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


@functools.lru_cache(maxsize=512)
def _routing_ref(*spec):
    return _ref(_routing(*spec))


def route_experts(logits: torch.Tensor, top_k: int, *, score: str = "softmax", bias: torch.Tensor | None = None,
                  groups: int = 1, kept_groups: int = 1, group_top: int = 1, renormalise: bool = True,
                  scale: float = 1.0, out: tuple[torch.Tensor, torch.Tensor] | None = None):
    """Experts and weights of each token from its router logits [T, E] (f32,
    f16 or bf16; rows may be strided; E <= 1024, top_k <= 32).

    Returns (indices int32 [T, top_k], weights f32 [T, top_k]), in descending
    order of the experts' values (score + `bias`, a selection bias [E] f32 that
    leaves the weights alone; without one the logits), equal values by the
    lower index, as f64 arithmetic on the logits orders them.  Experts masked by a logit
    that is NaN, -inf, <= -1e20 or f16's lowest value, or by such a bias, are
    never chosen; slots left empty hold (-1, 0).  `out`: the two contiguous
    tensors to write instead.
    """
    kind = _TYPE.get(logits.dtype)
    index = logits.get_device()
    if kind is None or index < 0:
        raise ValueError("logits must be f32, f16 or bf16 on a GPU")
    T, E, ld = _rows(logits, "logits")
    r = _routing_ref(score, groups, kept_groups, group_top, renormalise, scale)
    b = _vector(bias, E, "bias", index)
    if out is None:
        dev = logits.device
        idx = _empty(T, top_k, dtype=_i32, device=dev)
        w = _empty(T, top_k, dtype=_f32, device=dev)
    else:
        idx, w = out
        for t, dt in ((idx, torch.int32), (w, torch.float32)):
            if t.shape != (T, top_k) or t.dtype != dt or not t.is_contiguous() or t.get_device() != index:
                raise ValueError(f"out must be contiguous int32 and f32 tensors of shape {(T, top_k)} on cuda:{index}")
    _call(index, _route_fn, logits.data_ptr(), kind, T, E, ld, top_k, r, b, idx.data_ptr(), w.data_ptr())
    return idx, w


# ---- int8 products ---------------------------------------------------------------


def _weight(w: torch.Tensor, scale: torch.Tensor, name: str, K: int, index: int) -> tuple[MoeInt8Weight, int]:
    """The C image of an int8 matrix [K, N] and N."""
    if w.dtype != torch.int8 or w.dim() != 2 or w.shape[0] != K or w.get_device() != index:
        raise ValueError(f"{name} must be int8 [K={K}, N] on cuda:{index}, got {w.dtype} {tuple(w.shape)} on {w.device}")
    N = w.shape[1]
    sk, sn = w.stride()
    # the stride of an axis of one element says nothing
    if sn == 1 and (sk % 16 == 0 and sk >= N or K == 1):
        order, ld = MOE_WEIGHT_KN, sk if K > 1 else (N + 15) // 16 * 16
    elif sk == 1 and (sn % 16 == 0 and sn >= K or N == 1):
        order, ld = MOE_WEIGHT_NK, sn if N > 1 else (K + 15) // 16 * 16
    else:
        raise ValueError(f"{name}: one axis must be contiguous and the other's stride a multiple of 16 bytes, got strides "
                         f"{(sk, sn)}; int8_weight() lays a matrix out so")
    return MoeInt8Weight(w.data_ptr(), ld, _vector(scale, N, name + "'s scale", index), order), N


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


def _x(x: torch.Tensor) -> tuple[int, int, int, int, int]:
    """(MOE_TYPE_*, device index, tokens, K, row stride) of activations."""
    kind = _TYPE.get(x.dtype)
    index = x.get_device()
    if kind is None or index < 0:
        raise ValueError("x must be f32, f16 or bf16 on a GPU")
    return (kind, index, *_rows(x, "x"))


def quantize_int8_tokens(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Per-token symmetric int8 of x [T, K]: (q [T, K] int8 with rows on 16-byte
    boundaries, scale [T] f32 = max|x| / 127 -- times f32(1/127) -- or 1 where
    that is zero; q = round-half-even of the exact x / scale).  A row with a NaN
    or an infinity gets a NaN scale."""
    kind, index, T, K, ld = _x(x)
    kp = (K + 15) // 16 * 16
    q = _empty(T, kp, dtype=_i8, device=x.device)
    s = _empty(T, dtype=_f32, device=x.device)
    _call(index, lib.moe_int8_quantize_tokens, x.data_ptr(), kind, T, K, ld, q.data_ptr(), kp, s.data_ptr())
    return q[:, :K], s


def int8_matmul(q: torch.Tensor, scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, *,
                bias: torch.Tensor | None = None, out_dtype: torch.dtype | None = None,
                out: torch.Tensor | None = None) -> torch.Tensor:
    """(q @ w) * scale[:, None] * w_scale + bias for int8 q [T, K] (rows on
    16-byte boundaries, as quantize_int8_tokens makes them) and w [K, N]
    (either axis contiguous, the other's stride a multiple of 16): s32 sums,
    f32 after them, one rounding to the output type (bf16 by default)."""
    index = q.get_device()
    if q.dtype != torch.int8 or index < 0:
        raise ValueError("q must be int8 on a GPU")
    T, K, ld = _rows(q, "q")
    if T <= 1:
        ld = (ld + 15) // 16 * 16
    wt, N = _weight(w, w_scale, "w", K, index)
    b = _vector(bias, N, "bias", index)
    s = _vector(scale, T, "scale", index)
    out, kind, ldo = _output(out, T, N, out_dtype if out is not None or out_dtype is not None else torch.bfloat16, q)
    _call(index, lib.moe_int8_matmul, q.data_ptr(), ld, s, T, K, _ref(wt), N, b, out.data_ptr(), kind, ldo)
    return out


def int8_linear(x: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, *, bias: torch.Tensor | None = None,
                out_dtype: torch.dtype | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """x [T, K] (f32, f16, bf16) times the int8 matrix w [K, N] with f32 scales
    w_scale [N], the tokens quantised on the fly (quantize_int8_tokens, then
    int8_matmul); the output has x's type unless out_dtype or out says otherwise."""
    kind, index, T, K, ld = _x(x)
    wt, N = _weight(w, w_scale, "w", K, index)
    b = _vector(bias, N, "bias", index)
    out, okind, ldo = _output(out, T, N, x.dtype if out is None and out_dtype is None else out_dtype, x)
    n = _linear_scratch(T, K)
    scratch = _empty(n, dtype=_u8, device=x.device) if n else None
    _call(index, _linear_fn, x.data_ptr(), kind, T, K, ld, _ref(wt), N, b, out.data_ptr(), okind, ldo,
          scratch.data_ptr() if n else None, n)
    return out


def int8_shared_expert(x: torch.Tensor, w_gate: torch.Tensor, s_gate: torch.Tensor, w_up: torch.Tensor,
                       s_up: torch.Tensor, w_down: torch.Tensor, s_down: torch.Tensor, *,
                       residual: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """The shared expert of an MoE layer, an int8 SwiGLU FFN that every token
    takes: h = silu(x Wg) * (x Wu) in f32, y = h Wd (+ residual [T, d] of x's
    type), x and h quantised per token.  Weights as for int8_linear: gate and
    up [d, f] in one axis order, down [f, d].  The output has x's type unless
    `out` (which may be the residual) has another."""
    kind, index, T, d, ld = _x(x)
    g, f = _weight(w_gate, s_gate, "w_gate", d, index)
    u, fu = _weight(w_up, s_up, "w_up", d, index)
    dn, do = _weight(w_down, s_down, "w_down", f, index)
    if fu != f or do != d:
        raise ValueError(f"w_up must be [{d}, {f}] and w_down [{f}, {d}]")
    res, ld_res = None, 0
    if residual is not None:
        if residual.shape != x.shape or residual.dtype != x.dtype or residual.get_device() != index:
            raise ValueError("residual must have x's shape, type and device")
        ld_res = _rows(residual, "residual")[2]
        res = residual.data_ptr()
    out, okind, ldo = _output(out, T, d, x.dtype if out is None else None, x)
    n = _shared_scratch(T, d, f)
    scratch = _empty(n, dtype=_u8, device=x.device)
    _call(index, _shared_fn, x.data_ptr(), kind, T, d, ld, _ref(g), _ref(u), _ref(dn), f, res, ld_res, out.data_ptr(),
          okind, ldo, scratch.data_ptr(), n)
    return out
