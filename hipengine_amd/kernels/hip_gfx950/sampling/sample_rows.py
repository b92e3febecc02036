"""Sampling one token of every row of float32 logits from given uniform numbers: temperature, top-k, top-p, min-p (the
greedy choice alone is ``linear.lm_head.argmax_f32_rows_i32``).

Tokens are ordered by logit, highest first, equal ones by index; with ``w = exp((l - l_max) / temperature)`` top-k keeps
the first k, top-p of those the shortest prefix that holds ``top_p`` of their weight, min-p drops ``w < min_p``. The token
is the first one, by index, up to which the kept weights sum to more than ``uniform`` times their total.
"""

from __future__ import annotations

import ctypes
import functools

from hipengine_amd.core.hip import HipRuntime
from hipengine_amd.kernels.hip_gfx950 import _launch
from hipengine_amd.kernels.hip_gfx950._launch import I64, VOID, check_launch, entry, validate_pointers
from hipengine_amd.kernels.registry import KernelKey, register

MAX_VOCAB = 1 << 22

_ARGS = [VOID, I64] + [VOID] * 7 + [I64, I64, VOID, I64, VOID]
_WORKSPACE_ARGS = [I64, I64, ctypes.POINTER(I64)]


def _check_shape(rows: int, vocab_size: int) -> None:
    if rows <= 0 or rows > 65535:
        raise ValueError("rows must be 1 .. 65535")
    if vocab_size <= 0 or vocab_size > MAX_VOCAB:
        raise ValueError(f"vocab_size must be 1 .. {MAX_VOCAB}")


def sample_workspace_bytes(rows: int, vocab_size: int, *, library: ctypes.CDLL | None = None) -> int:
    """Bytes of scratch that a call of these sizes needs."""
    return _default_workspace_bytes(rows, vocab_size) if library is None else _workspace_bytes(rows, vocab_size, library)


def _workspace_bytes(rows: int, vocab_size: int, library: ctypes.CDLL | None) -> int:
    _check_shape(rows, vocab_size)
    out = I64(0)
    check_launch(entry("hipengine_gfx950_sample_f32_rows_i32_workspace_bytes", _WORKSPACE_ARGS, library)(
        rows, vocab_size, ctypes.byref(out)), None)
    return int(out.value)


@functools.lru_cache(maxsize=64)   # a function of the sizes alone, asked for at every step of a decode loop
def _default_workspace_bytes(rows: int, vocab_size: int) -> int:
    return _workspace_bytes(rows, vocab_size, None)


def sample_f32_rows_i32(logits_ptr: int, uniform_ptr: int, out_ids_ptr: int, rows: int, vocab_size: int, *,
                        workspace_ptr: int, workspace_bytes: int, temperature_ptr: int | None = None,
                        top_k_ptr: int | None = None, top_p_ptr: int | None = None, min_p_ptr: int | None = None,
                        out_logprobs_ptr: int | None = None, logits_stride: int = 0, stream: int = 0,
                        library: ctypes.CDLL | None = None, runtime: HipRuntime | None = None) -> None:
    """``logits`` float32 ``[rows, vocab_size]`` (0: packed rows), ``uniform`` float32 ``[rows]`` in 0 <= u < 1, int32
    ``out_ids`` and optionally float32 ``out_logprobs`` ``[rows]``. Settings are arrays ``[rows]`` (float32, ``top_k``
    int32), each of which may be None; a temperature of 0 or less takes the highest logit, one above 0 counts as at least
    2^-124. A log-probability is that of the kept tokens' distribution, which the token was drawn from. A row with nothing
    but -infinity and NaN gives -1. The workspace (8-byte aligned) is scratch of the size ``sample_workspace_bytes`` gives;
    calls that overlap in time need one each."""
    if _launch.VALIDATE:
        _check_shape(rows, vocab_size)
        if logits_stride != 0 and logits_stride < vocab_size:
            raise ValueError("logits_stride must be 0 or at least vocab_size")
        validate_pointers(logits_ptr=logits_ptr, uniform_ptr=uniform_ptr, out_ids_ptr=out_ids_ptr, workspace_ptr=workspace_ptr)
    check_launch(entry("hipengine_gfx950_sample_f32_rows_i32", _ARGS, library)(
        logits_ptr, logits_stride, uniform_ptr, temperature_ptr, top_k_ptr, top_p_ptr, min_p_ptr, out_ids_ptr,
        out_logprobs_ptr, rows, vocab_size, workspace_ptr, workspace_bytes, stream), runtime)


def register_kernels(backend: str = "hip_gfx950", *, replace: bool = False) -> None:
    register(KernelKey(backend, "sample", "f32", "rows_i32"), sample_f32_rows_i32, replace=replace)
