"""The paged KV cache held in 8 bits, one float32 scale for each block of 32 tokens and KV head: appending keys (normed
and rotated on the way, if asked) and values, and reading tokens back.

Buffers of a cache (raw device pointers; the caller owns them):

* ``k``, ``v``: uint8 ``[pages, kv_heads, page_size / 32, head_dim * 32]``, bytes ``128 + q`` with q in -127..127;
  a K block is ``[head_dim / 16][32 tokens][16]``, a V block ``[head_dim][32]`` with token t at place ``v_place(t)``
  (the operand order of the attention kernel's matrix instructions);
* ``k_scale``, ``v_scale``: float32 ``[pages, kv_heads, page_size / 32]``; a value is ``q * scale``.

``page_table`` is int32 ``[batch, table_stride]``, ``q_start`` int32 ``[batch + 1]`` (rows of sequence b are ``q_start[b]``
to ``q_start[b + 1] - 1``) and ``kv_lens`` int32 ``[batch]`` the tokens of each sequence in the cache, this call's rows
included; :mod:`paged_attention_q8` takes the same arrays.
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
    check_batch,
    check_head_dim,
    check_positive,
    check_rotation,
    check_stride,
    kind_of,
)
from hipengine_amd.kernels.registry import KernelKey, register

BLOCK_TOKENS = 32
_PAGE_SIZES = frozenset(1 << i for i in range(5, 21))

_APPEND_ARGS = [VOID, VOID, I32, I64, I64, VOID, VOID, VOID, I64, I32, F32, F32] + [VOID] * 5 + [I64] + [VOID] * 2 + [I64] * 7 + [VOID]
_READ_ARGS = [VOID] * 5 + [I64] + [VOID] * 4 + [I32] + [I64] * 8 + [VOID]


def v_place(token: int) -> int:
    """Place of a block's token 0..31 in the rows of a V block."""
    return (token & 3) | ((token >> 3 & 3) << 2) | ((token >> 2 & 1) << 4)


class KVCacheQ8:
    """The buffers and sizes of one layer's cache, checked once when it is made."""

    __slots__ = ("k_ptr", "v_ptr", "k_scale_ptr", "v_scale_ptr", "pages", "page_size", "kv_heads", "head_dim")

    def __init__(self, k_ptr: int, v_ptr: int, k_scale_ptr: int, v_scale_ptr: int, pages: int, page_size: int,
                 kv_heads: int, head_dim: int) -> None:
        if not (0 < pages < 1 << 31 and 0 < kv_heads <= 65535 and page_size in _PAGE_SIZES and head_dim in HEAD_DIMS
                and are_pointers(k_ptr, v_ptr, k_scale_ptr, v_scale_ptr) and (k_ptr | v_ptr) & 15 == 0):
            check_positive(pages=pages, kv_heads=kv_heads)
            if pages > 2**31 - 1 or kv_heads > 65535:
                raise ValueError("pages must fit int32 page numbers and kv_heads be at most 65535")
            if page_size not in _PAGE_SIZES:
                raise ValueError("page_size must be a power of two, 32 .. 2^20")
            check_head_dim(head_dim)
            validate_pointers(k_ptr=k_ptr, v_ptr=v_ptr, k_scale_ptr=k_scale_ptr, v_scale_ptr=v_scale_ptr)
            raise ValueError("k_ptr and v_ptr must be 16-byte aligned")
        self.k_ptr, self.v_ptr, self.k_scale_ptr, self.v_scale_ptr = k_ptr, v_ptr, k_scale_ptr, v_scale_ptr
        self.pages, self.page_size, self.kv_heads, self.head_dim = pages, page_size, kv_heads, head_dim

    @staticmethod
    def value_bytes(pages: int, page_size: int, kv_heads: int, head_dim: int) -> int:
        """Bytes of each of ``k`` and ``v``."""
        return pages * page_size * kv_heads * head_dim

    @staticmethod
    def scale_bytes(pages: int, page_size: int, kv_heads: int) -> int:
        """Bytes of each of ``k_scale`` and ``v_scale``."""
        return pages * (page_size // BLOCK_TOKENS) * kv_heads * 4


def kv_append_q8(cache: KVCacheQ8, k_ptr: int, v_ptr: int, page_table_ptr: int, table_stride: int, q_start_ptr: int,
                 kv_lens_ptr: int, tokens: int, batch: int, max_q_len: int, *, k_weight_ptr: int | None = None,
                 positions_ptr: int | None = None, inv_freq_ptr: int | None = None, rotary_dim: int = 0,
                 interleaved: bool = False, in_kind: str = "bf16", k_stride: int = 0, v_stride: int = 0, eps: float = 1e-6,
                 rope_scale: float = 1.0, stream: int = 0, library: ctypes.CDLL | None = None,
                 runtime: HipRuntime | None = None) -> None:
    """Append k and v ``[tokens, kv_heads, head_dim]`` at the end of their sequences.

    ``k_weight_ptr`` (float32 ``[head_dim]``) norms every key head, ``inv_freq_ptr`` rotates it at ``positions_ptr``
    (int64 ``[tokens]``; None: a token's place in its sequence). A block's scale grows to hold the new tokens, and its
    earlier tokens are rescaled then; a block whose first token is appended starts anew; bytes behind the new tokens
    stay. A NaN or infinity makes its block's scale NaN until the block starts anew. No block may be appended to under two
    names in one call (two sequences, or a page twice in one table)."""
    width = cache.kv_heads * cache.head_dim
    if _launch.VALIDATE and not (
            tokens > 0 and 0 < batch <= 65535 and max_q_len > 0 and table_stride > 0 and in_kind in KINDS and eps >= 0.0
            and (k_stride == 0 or k_stride >= width) and (v_stride == 0 or v_stride >= width)
            and (16 <= rotary_dim <= cache.head_dim and rotary_dim & 15 == 0 if inv_freq_ptr else rotary_dim == 0)
            and are_pointers(k_ptr, v_ptr, page_table_ptr, q_start_ptr, kv_lens_ptr)):
        check_positive(tokens=tokens, batch=batch, max_q_len=max_q_len, table_stride=table_stride)
        check_batch(batch)
        kind_of(in_kind, "in_kind")
        check_rotation(inv_freq_ptr, rotary_dim, cache.head_dim)
        check_stride("k_stride", k_stride, width)
        check_stride("v_stride", v_stride, width)
        if not eps >= 0.0:
            raise ValueError("eps must not be negative")
        validate_pointers(k_ptr=k_ptr, v_ptr=v_ptr, page_table_ptr=page_table_ptr, q_start_ptr=q_start_ptr,
                          kv_lens_ptr=kv_lens_ptr)
    check_launch(entry("hipengine_gfx950_kv_append_q8", _APPEND_ARGS, library)(
        k_ptr, v_ptr, KINDS[in_kind], k_stride, v_stride, k_weight_ptr, positions_ptr, inv_freq_ptr, rotary_dim,
        1 if interleaved else 0, eps, rope_scale, cache.k_ptr, cache.v_ptr, cache.k_scale_ptr, cache.v_scale_ptr,
        page_table_ptr, table_stride, q_start_ptr, kv_lens_ptr, tokens, batch, max_q_len, cache.pages, cache.page_size,
        cache.kv_heads, cache.head_dim, stream), runtime)


def kv_read_q8(cache: KVCacheQ8, k_out_ptr: int | None, v_out_ptr: int | None, page_table_ptr: int, table_stride: int,
               row_start_ptr: int, kv_lens_ptr: int, tokens: int, batch: int, *, out_kind: str = "bf16",
               k_out_stride: int = 0, v_out_stride: int = 0, stream: int = 0, library: ctypes.CDLL | None = None,
               runtime: HipRuntime | None = None) -> None:
    """Read the last ``row_start[b + 1] - row_start[b]`` cached tokens of every sequence b into rows ``row_start[b]`` ..
    of the outputs ``[tokens, kv_heads, head_dim]``. One of the outputs may be None. Tokens on a page that is not in the
    cache read as zeros."""
    width = cache.kv_heads * cache.head_dim
    if _launch.VALIDATE and not (
            tokens > 0 and 0 < batch <= 65535 and table_stride > 0 and out_kind in KINDS and (k_out_ptr or v_out_ptr)
            and (k_out_stride == 0 or k_out_stride >= width) and (v_out_stride == 0 or v_out_stride >= width)
            and are_pointers(page_table_ptr, row_start_ptr, kv_lens_ptr)):
        check_positive(tokens=tokens, batch=batch, table_stride=table_stride)
        check_batch(batch)
        kind_of(out_kind, "out_kind")
        check_stride("k_out_stride", k_out_stride, width)
        check_stride("v_out_stride", v_out_stride, width)
        if not k_out_ptr and not v_out_ptr:
            raise ValueError("k_out_ptr or v_out_ptr must be a non-null device pointer")
        validate_pointers(page_table_ptr=page_table_ptr, row_start_ptr=row_start_ptr, kv_lens_ptr=kv_lens_ptr)
    check_launch(entry("hipengine_gfx950_kv_read_q8", _READ_ARGS, library)(
        cache.k_ptr, cache.v_ptr, cache.k_scale_ptr, cache.v_scale_ptr, page_table_ptr, table_stride, row_start_ptr,
        kv_lens_ptr, k_out_ptr, v_out_ptr, KINDS[out_kind], k_out_stride, v_out_stride, tokens, batch, cache.pages,
        cache.page_size, cache.kv_heads, cache.head_dim, stream), runtime)


def register_kernels(backend: str = "hip_gfx950", *, replace: bool = False) -> None:
    register(KernelKey(backend, "kv_cache", "q8_block32", "append"), kv_append_q8, replace=replace)
    register(KernelKey(backend, "kv_cache", "q8_block32", "read"), kv_read_q8, replace=replace)
