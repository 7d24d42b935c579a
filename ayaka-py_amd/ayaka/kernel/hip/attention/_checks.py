"""Argument checks shared by the attention operators."""

from __future__ import annotations

import math

import torch

ATTENTION_DTYPES = (torch.float16, torch.bfloat16)
MAX_HEAD_DIM = 256


def on_device_of(first: torch.Tensor, *others: torch.Tensor) -> bool:
    """All tensors on one CUDA device (the detailed checks name the one that is not)."""
    index = first.get_device()
    for t in others:
        if t.get_device() != index:
            return False
    return first.is_cuda


def check_window(window: int, sinks: int) -> None:
    if type(window) is int and type(sinks) is int and window >= 0 and sinks >= 0:
        return
    for name, value in (("window", window), ("sinks", sinks)):
        if isinstance(value, bool) or not isinstance(value, int):
            raise TypeError(f"{name} must be an integer")
        if value < 0:
            raise ValueError(f"{name} must not be negative")


def check_scale(scale: float, name: str = "softmax_scale") -> None:
    if not math.isfinite(scale):
        raise ValueError(f"{name} must be finite")


def check_heads(heads: int, kv_heads: int, dim: int) -> None:
    if kv_heads < 1 or heads < 1 or heads % kv_heads:
        raise ValueError(f"query heads ({heads}) must be a positive multiple of the key/value heads ({kv_heads})")
    if not 1 <= dim <= MAX_HEAD_DIM:
        raise ValueError(f"head_dim must be between 1 and {MAX_HEAD_DIM}, got {dim}")


def rows_of_heads(t: torch.Tensor) -> torch.Tensor:
    """``[rows, heads, dim]`` with unit stride along ``dim`` (a copy only where it has another)."""
    return t if t.stride(2) == 1 or t.shape[2] == 1 else t.contiguous()


def new_output(query: torch.Tensor) -> torch.Tensor:
    """A contiguous tensor of the query's shape and dtype."""
    return torch.empty_like(query, memory_format=torch.contiguous_format)
