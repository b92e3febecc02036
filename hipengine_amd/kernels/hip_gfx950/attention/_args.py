"""Argument checks shared by the attention wrappers."""

from __future__ import annotations

import ctypes

from hipengine_amd.kernels.hip_gfx950._launch import KIND_BF16, KIND_F16, KIND_F32

F32 = ctypes.c_float
KINDS = {"f32": KIND_F32, "bf16": KIND_BF16, "fp16": KIND_F16}
HEAD_DIMS = frozenset({64, 128, 256})


# The wrappers test their arguments in one expression and take the argument by argument checks below only where it fails,
# for the message: a launch of a few microseconds is not to wait for its own checks.
def are_pointers(*values: int | None) -> bool:
    for value in values:
        if type(value) is not int or value <= 0:
            return False
    return True


def kind_of(name: str, argument: str, allowed: tuple[str, ...] = ("f32", "bf16", "fp16")) -> int:
    if name not in allowed:
        raise ValueError(f"{argument} must be one of {', '.join(allowed)}")
    return KINDS[name]


def check_positive(**values: int) -> None:
    for name, value in values.items():
        if value <= 0:
            raise ValueError(f"{name} must be positive")


def check_batch(batch: int) -> None:
    if batch > 65535:
        raise ValueError("batch must be at most 65535")


def check_head_dim(head_dim: int) -> None:
    if head_dim not in HEAD_DIMS:
        raise ValueError("head_dim must be 64, 128 or 256")


def check_rotation(inv_freq_ptr: int | None, rotary_dim: int, head_dim: int) -> None:
    if not inv_freq_ptr:
        if rotary_dim != 0:
            raise ValueError("rotary_dim needs inv_freq_ptr")
    elif rotary_dim < 16 or rotary_dim > head_dim or rotary_dim % 16 != 0:
        raise ValueError("rotary_dim must be a multiple of 16, at most head_dim")


def check_stride(name: str, stride: int, width: int) -> None:
    """0 stands for packed rows."""
    if stride != 0 and stride < width:
        raise ValueError(f"{name} must be 0 or at least heads * head_dim")
