"""RMS norm of every query and key head and the position rotation, in one pass (no counterpart under this name in
hipEngine, whose runner composes the two steps).

``y = x / sqrt(mean(x^2) + eps) * weight`` per head, then pairs ``(a, b) -> rope_scale * (a cos t - b sin t, b cos t +
a sin t)`` with ``t = position * inv_freq[i]`` over the first ``rotary_dim`` values: pairs ``(i, i + rotary_dim / 2)``, or
``(2i, 2i + 1)`` where ``interleaved``. Statistics in float32, angles in float64, one rounding at the end.
"""

from __future__ import annotations

import ctypes

from hipengine_amd.core.hip import HipRuntime
from hipengine_amd.kernels.hip_gfx950 import _launch
from hipengine_amd.kernels.hip_gfx950._launch import I32, I64, VOID, check_launch, entry, validate_pointers
from hipengine_amd.kernels.hip_gfx950.attention._args import (
    F32,
    HEAD_DIMS,
    KINDS,
    are_pointers,
    check_head_dim,
    check_positive,
    check_rotation,
    check_stride,
    kind_of,
)
from hipengine_amd.kernels.registry import KernelKey, register

_ARGS = [VOID] * 8 + [I32] * 2 + [I64] * 9 + [F32, F32, I32, VOID]


def qk_norm_rope(q_ptr: int | None, k_ptr: int | None, q_out_ptr: int | None, k_out_ptr: int | None, tokens: int,
                 q_heads: int, kv_heads: int, head_dim: int, *, q_weight_ptr: int | None = None,
                 k_weight_ptr: int | None = None, positions_ptr: int | None = None, inv_freq_ptr: int | None = None,
                 rotary_dim: int = 0, interleaved: bool = False, in_kind: str = "bf16", out_kind: str = "bf16",
                 q_stride: int = 0, k_stride: int = 0, q_out_stride: int = 0, k_out_stride: int = 0, eps: float = 1e-6,
                 rope_scale: float = 1.0, stream: int = 0, library: ctypes.CDLL | None = None,
                 runtime: HipRuntime | None = None) -> None:
    """q ``[tokens, q_heads, head_dim]`` and k ``[tokens, kv_heads, head_dim]`` into their outputs. A null weight skips
    the norm, a null ``inv_freq_ptr`` the rotation, 0 heads one of the two tensors. Strides count elements from one
    token to the next (0: packed), so q and k may be columns of one projection's output. An output may be its input
    where kind and stride agree."""
    q_width, k_width = q_heads * head_dim, kv_heads * head_dim
    if _launch.VALIDATE and not (
            0 < tokens <= 4194303 and 0 <= q_heads <= 4096 and 0 <= kv_heads <= 4096 and q_heads + kv_heads > 0
            and head_dim in HEAD_DIMS and in_kind in KINDS and out_kind in KINDS and eps >= 0.0
            and (16 <= rotary_dim <= head_dim and rotary_dim & 15 == 0 and are_pointers(positions_ptr) if inv_freq_ptr
                 else rotary_dim == 0)
            and (q_heads == 0 or are_pointers(q_ptr, q_out_ptr)) and (kv_heads == 0 or are_pointers(k_ptr, k_out_ptr))
            and (q_stride == 0 or q_stride >= q_width) and (q_out_stride == 0 or q_out_stride >= q_width)
            and (k_stride == 0 or k_stride >= k_width) and (k_out_stride == 0 or k_out_stride >= k_width)
            and (q_heads == 0 or q_ptr != q_out_ptr) and (kv_heads == 0 or k_ptr != k_out_ptr)):
        check_positive(tokens=tokens)
        if tokens > 4194303:
            raise ValueError("tokens must be at most 4194303")
        if q_heads < 0 or kv_heads < 0 or q_heads + kv_heads == 0 or q_heads > 4096 or kv_heads > 4096:
            raise ValueError("q_heads and kv_heads must be 0 .. 4096, not both 0")
        check_head_dim(head_dim)
        kind_of(in_kind, "in_kind")
        kind_of(out_kind, "out_kind")
        check_rotation(inv_freq_ptr, rotary_dim, head_dim)
        if not eps >= 0.0:
            raise ValueError("eps must not be negative")
        if q_heads:
            validate_pointers(q_ptr=q_ptr, q_out_ptr=q_out_ptr)
        if kv_heads:
            validate_pointers(k_ptr=k_ptr, k_out_ptr=k_out_ptr)
        if inv_freq_ptr:
            validate_pointers(positions_ptr=positions_ptr)
        for name, stride, heads in (("q_stride", q_stride, q_heads), ("q_out_stride", q_out_stride, q_heads),
                                    ("k_stride", k_stride, kv_heads), ("k_out_stride", k_out_stride, kv_heads)):
            check_stride(name, stride, heads * head_dim)
        for name, heads, src, dst, a, b in (("q", q_heads, q_ptr, q_out_ptr, q_stride, q_out_stride),
                                            ("k", kv_heads, k_ptr, k_out_ptr, k_stride, k_out_stride)):
            packed = heads * head_dim
            if heads and src == dst and (in_kind != out_kind or (a or packed) != (b or packed)):
                raise ValueError(f"{name} in place needs equal kinds and strides")
    check_launch(entry("hipengine_gfx950_qk_norm_rope", _ARGS, library)(
        q_ptr, k_ptr, q_weight_ptr, k_weight_ptr, positions_ptr, inv_freq_ptr, q_out_ptr, k_out_ptr, KINDS[in_kind],
        KINDS[out_kind], tokens, q_heads, kv_heads, head_dim, rotary_dim, q_stride, k_stride, q_out_stride, k_out_stride,
        eps, rope_scale, 1 if interleaved else 0, stream), runtime)


def register_kernels(backend: str = "hip_gfx950", *, replace: bool = False) -> None:
    register(KernelKey(backend, "qk_norm+rope", "f32_weight"), qk_norm_rope, replace=replace)
