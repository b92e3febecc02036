"""Attention of ragged queries over the 8-bit paged KV cache of :mod:`kv_cache_q8`: single tokens, drafts of a few and
prompts, causal, grouped query heads, optionally within a sliding window.

``out = softmax(scale * q K^T) V``; the query in row i of a sequence's n is at place ``kv_lens[b] - n + i`` and sees the
places up to its own, with ``window > 0`` the last ``window`` of them. A query that sees nothing gives zeros.
"""

from __future__ import annotations

import ctypes
import functools
import math

from hipengine_amd.core.hip import HipRuntime
from hipengine_amd.kernels.hip_gfx950 import _launch
from hipengine_amd.kernels.hip_gfx950._launch import I32, I64, VOID, check_launch, entry, validate_pointers
from hipengine_amd.kernels.hip_gfx950.attention._args import (
    F32,
    KINDS,
    are_pointers,
    check_batch,
    check_head_dim,
    check_positive,
    check_stride,
    kind_of,
)
from hipengine_amd.kernels.hip_gfx950.attention.kv_cache_q8 import KVCacheQ8
from hipengine_amd.kernels.registry import KernelKey, register

_ARGS = [VOID, VOID, I32, I64, I64] + [VOID] * 5 + [I64] + [VOID] * 2 + [I64] * 9 + [F32, I64, VOID, I64, VOID]
_WORKSPACE_ARGS = [I64] * 7 + [ctypes.POINTER(I64)]

_MOST_ROWS = 65535 * 128            # of a sequence and KV head; twice as many of head_dim 256


def _rows_fit(tokens: int, max_q_len: int, q_heads: int, kv_heads: int, head_dim: int) -> bool:
    return min(max_q_len, tokens) * (q_heads // kv_heads) <= (2 * _MOST_ROWS if head_dim == 256 else _MOST_ROWS)


def _check_shape(tokens: int, batch: int, max_q_len: int, max_kv_len: int, q_heads: int, kv_heads: int, head_dim: int) -> None:
    check_positive(tokens=tokens, batch=batch, max_q_len=max_q_len, q_heads=q_heads, kv_heads=kv_heads)
    check_batch(batch)
    if tokens > 1 << 26:
        raise ValueError("tokens must be at most 2^26")
    if max_kv_len < 0 or max_kv_len > 1 << 30:
        raise ValueError("max_kv_len must be 0 .. 2^30")
    if q_heads % kv_heads != 0 or q_heads > 4096:
        raise ValueError("q_heads must be a multiple of kv_heads, at most 4096")
    check_head_dim(head_dim)
    if not _rows_fit(tokens, max_q_len, q_heads, kv_heads, head_dim):
        raise ValueError("a sequence may have at most 65535 * 128 rows (tokens * query heads) for each KV head, "
                         "65535 * 256 of head_dim 256: attend to a longer prompt in chunks")


def paged_attention_q8_workspace_bytes(tokens: int, batch: int, max_q_len: int, max_kv_len: int, q_heads: int,
                                       kv_heads: int, head_dim: int, *, library: ctypes.CDLL | None = None) -> int:
    """Bytes of scratch that a call of these sizes needs, whatever its window; 0 where it needs none."""
    if library is not None:
        return _workspace_bytes(tokens, batch, max_q_len, max_kv_len, q_heads, kv_heads, head_dim, library)
    return _default_workspace_bytes(tokens, batch, max_q_len, max_kv_len, q_heads, kv_heads, head_dim)


def _workspace_bytes(tokens: int, batch: int, max_q_len: int, max_kv_len: int, q_heads: int, kv_heads: int, head_dim: int,
                     library: ctypes.CDLL | None) -> int:
    _check_shape(tokens, batch, max_q_len, max_kv_len, q_heads, kv_heads, head_dim)
    out = I64(0)
    check_launch(entry("hipengine_gfx950_paged_attention_q8_workspace_bytes", _WORKSPACE_ARGS, library)(
        tokens, batch, max_q_len, max_kv_len, q_heads, kv_heads, head_dim, ctypes.byref(out)), None)
    return int(out.value)


@functools.lru_cache(maxsize=64)   # a function of the sizes alone, asked for at every step of a decode loop
def _default_workspace_bytes(tokens: int, batch: int, max_q_len: int, max_kv_len: int, q_heads: int, kv_heads: int,
                             head_dim: int) -> int:
    return _workspace_bytes(tokens, batch, max_q_len, max_kv_len, q_heads, kv_heads, head_dim, None)


def paged_attention_q8(cache: KVCacheQ8, q_ptr: int, out_ptr: int, page_table_ptr: int, table_stride: int,
                       q_start_ptr: int, kv_lens_ptr: int, tokens: int, batch: int, max_q_len: int, max_kv_len: int,
                       q_heads: int, *, workspace_ptr: int | None = None, workspace_bytes: int = 0,
                       scale: float | None = None, window: int = 0, kind: str = "bf16", q_stride: int = 0,
                       out_stride: int = 0, stream: int = 0, library: ctypes.CDLL | None = None,
                       runtime: HipRuntime | None = None) -> None:
    """q and out ``[tokens, q_heads, head_dim]`` (bf16 or fp16 bits, both of one kind). ``max_q_len`` and ``max_kv_len``
    are at least the longest sequence's; ``scale`` defaults to ``head_dim ** -0.5``. The workspace (16-byte aligned) is
    scratch of the size ``paged_attention_q8_workspace_bytes`` gives; calls that overlap in time need one each."""
    kv_heads, head_dim = cache.kv_heads, cache.head_dim
    width = q_heads * head_dim
    if _launch.VALIDATE and not (
            0 < tokens <= 1 << 26 and 0 < batch <= 65535 and max_q_len > 0 and 0 <= max_kv_len <= 1 << 30
            and 0 < q_heads <= 4096 and q_heads % kv_heads == 0 and table_stride > 0 and (kind == "bf16" or kind == "fp16")
            and (scale is None or 0.0 < scale < math.inf) and 0 <= window <= 1 << 30
            and (q_stride == 0 or q_stride >= width) and (out_stride == 0 or out_stride >= width) and q_ptr != out_ptr
            and (tokens * q_heads <= _MOST_ROWS or _rows_fit(tokens, max_q_len, q_heads, kv_heads, head_dim))
            and are_pointers(q_ptr, out_ptr, page_table_ptr, q_start_ptr, kv_lens_ptr)):
        _check_shape(tokens, batch, max_q_len, max_kv_len, q_heads, kv_heads, head_dim)
        check_positive(table_stride=table_stride)
        kind_of(kind, "kind", ("bf16", "fp16"))
        if scale is not None and not 0.0 < scale < math.inf:
            raise ValueError("scale must be positive and finite")
        if window < 0 or window > 1 << 30:
            raise ValueError("window must be 0 (none) .. 2^30")
        check_stride("q_stride", q_stride, width)
        check_stride("out_stride", out_stride, width)
        validate_pointers(q_ptr=q_ptr, out_ptr=out_ptr, page_table_ptr=page_table_ptr, q_start_ptr=q_start_ptr,
                          kv_lens_ptr=kv_lens_ptr)
        if q_ptr == out_ptr:
            raise ValueError("out_ptr must not be q_ptr")
    check_launch(entry("hipengine_gfx950_paged_attention_q8", _ARGS, library)(
        q_ptr, out_ptr, KINDS[kind], q_stride, out_stride, cache.k_ptr, cache.v_ptr, cache.k_scale_ptr, cache.v_scale_ptr,
        page_table_ptr, table_stride, q_start_ptr, kv_lens_ptr, tokens, batch, max_q_len, max_kv_len, q_heads,
        kv_heads, head_dim, cache.pages, cache.page_size, head_dim ** -0.5 if scale is None else scale,
        window, workspace_ptr, workspace_bytes, stream), runtime)


def register_kernels(backend: str = "hip_gfx950", *, replace: bool = False) -> None:
    register(KernelKey(backend, "attention", "q8_block32", "paged"), paged_attention_q8, replace=replace)
