"""A KV cache in 4 bits: appends (with or without position rotation) and rows read back, on the
gfx950 kernels of ``csrc/rope_kv.hip``.

A plane is two uint8 tensors, ``codes [pages, kv_heads, page_size, head_dim / 2]`` and ``scales
[pages, kv_heads, page_size, head_dim / 32]``. Codes are OCP e2m1, the even dim in the low half
of a byte; every 32 dims of a row share one UE8M0 scale, the least power of two under which
none of them exceeds 6 (as ``per_token_group_quant_mxfp8`` scales its groups, for a largest code
of 448). So there is no calibrated scale, and a cached element takes 4.25 bits. A group that
holds an infinity or NaN is NaN as a whole; magnitudes over 1.5 * 2^127 count as that. Scale code
``s`` stands for 2^(s - 127) from 0 on and 255 for NaN; a group of zeros is written with scale code 0 and
codes of zero. (The mxfp8 products take scale code 0 for a factor of 0 instead.)

The planes are head-major, unlike the 16-bit and fp8 caches: a head's rows of a page are
consecutive, as its attention reads them. No counterpart in the reference. There is no CPU path.
"""

from __future__ import annotations

import torch

from ayaka.kernel.hip import _lib
from ayaka.kernel.hip._host import require_dtype
from ayaka.kernel.hip.attention._checks import MAX_HEAD_DIM, on_device_of
from ayaka.kernel.hip.cache.rope_cache import (
    check_devices,
    check_payload,
    check_result,
    check_rotation,
    packed_rows,
)
from ayaka.kernel.ops import custom_op

__all__ = ["gather_cache_mxfp4", "rope_write_kv_mxfp4", "write_kv_mxfp4"]

GROUP = 32
_PAYLOAD_DTYPES = (torch.float32, torch.float16, torch.bfloat16)


def check_plane(codes: torch.Tensor, scales: torch.Tensor, name: str) -> tuple[int, int, int, int]:
    """``(pages, kv_heads, page_size, head_dim)`` of a 4-bit plane."""
    if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
        require_dtype(codes, f"{name}_codes", (torch.uint8,))
        require_dtype(scales, f"{name}_scales", (torch.uint8,))
    if codes.ndim != 4 or scales.ndim != 4:
        raise ValueError(f"{name}_codes and {name}_scales must be [pages, kv_heads, page_size, head_dim / 2] and [..., head_dim / 32]")
    pages, kv_heads, page_size, half = codes.shape
    their_pages, their_heads, their_size, groups = scales.shape
    if their_pages != pages or their_heads != kv_heads or their_size != page_size:
        raise ValueError(f"{name}_codes and {name}_scales must be [pages, kv_heads, page_size, head_dim / 2] and [..., head_dim / 32]")
    dim = 2 * half
    if dim % GROUP or not GROUP <= dim <= MAX_HEAD_DIM or groups * GROUP != dim:
        raise ValueError(f"the head_dim of a 4-bit cache must be a multiple of {GROUP} up to {MAX_HEAD_DIM}, with a scale for every "
                         f"{GROUP} dims; got {dim} dims and {groups} scales")
    if kv_heads < 1 or page_size < 8 or page_size % 8:
        raise ValueError(f"a 4-bit cache needs kv_heads and a page_size that is a multiple of 8, got {kv_heads} and {page_size}")
    _check_memory(codes, scales, name)
    return pages, kv_heads, page_size, dim


def _check_memory(codes, scales, name) -> None:
    if not codes.is_contiguous() or not scales.is_contiguous():
        raise ValueError("KV cache pages must be contiguous")
    if (codes.data_ptr() | scales.data_ptr()) & 15:
        raise ValueError(f"{name}_codes and {name}_scales must be 16-byte aligned")


def check_planes(key_codes, key_scales, value_codes, value_scales) -> tuple[int, int, int, int]:
    """Those of K and V; V's geometry needs no look of its own where it is K's."""
    geometry = check_plane(key_codes, key_scales, "key")
    same = value_codes.shape == key_codes.shape and value_scales.shape == key_scales.shape
    if same and value_codes.dtype == value_scales.dtype == torch.uint8:
        _check_memory(value_codes, value_scales, "value")
    elif check_plane(value_codes, value_scales, "value") != geometry:
        raise ValueError("KV cache planes must share geometry")
    return geometry


def _write(query, heads, key, value, rows, positions, cos_sin, planes, slots, query_out, key_out, interleaved) -> None:
    pages, kv_heads, page_size, dim = check_planes(*planes)
    if rows[1] != kv_heads or rows[2] != dim:
        raise ValueError(f"key and value rows {tuple(rows[1:])} do not match a cache of {kv_heads} heads of {dim}")
    tokens = rows[0]
    if tokens == 0:
        return
    # (the tensors stay referenced: a copy's memory must not be handed out before the launch)
    query, *q = packed_rows(query)
    key, *k = packed_rows(key)
    value, *v = packed_rows(value)
    slots = slots.contiguous()
    positions = None if positions is None else positions.contiguous()
    with _lib.on_device(key):
        _lib.call("ayk_rope_kv_write_mxfp4", *q, *k, *v, _lib.dtype_code(key.dtype), tokens, heads, kv_heads, dim,
                  _lib.ptr(positions), _lib.ptr(cos_sin), *((0, 0) if cos_sin is None else cos_sin.shape), int(interleaved),
                  *packed_rows(query_out)[1:], *packed_rows(key_out)[1:], *[p.data_ptr() for p in planes], pages, page_size,
                  slots.data_ptr(), _lib.stream_of(key))


def _rope_write_kv_mxfp4_fake(query, key, value, positions, cos_sin, key_codes, key_scales, value_codes, value_scales, slots,
                              query_out, key_out=None, interleaved=False) -> None:
    return None


@custom_op(name="rope_write_kv_mxfp4", fake_impl=_rope_write_kv_mxfp4_fake,
           mutates_args=["key_codes", "key_scales", "value_codes", "value_scales", "query_out", "key_out"])
def rope_write_kv_mxfp4(
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    positions: torch.Tensor,
    cos_sin: torch.Tensor,
    key_codes: torch.Tensor,
    key_scales: torch.Tensor,
    value_codes: torch.Tensor,
    value_scales: torch.Tensor,
    slots: torch.Tensor,
    query_out: torch.Tensor,
    key_out: torch.Tensor | None = None,
    interleaved: bool = False,
) -> None:
    """``rope_write_kv`` into a 4-bit cache: the arguments, and what becomes of padding tokens,
    are that operator's, but for the planes (see the module) and the static scales, which a
    4-bit cache does not have."""
    if not on_device_of(query, key, value, positions, cos_sin, key_codes, key_scales, value_codes, value_scales, slots,
                        query_out, query if key_out is None else key_out):
        check_devices(query, "query", key=key, value=value, positions=positions, cos_sin=cos_sin, key_codes=key_codes,
                      key_scales=key_scales, value_codes=value_codes, value_scales=value_scales, slots=slots,
                      query_out=query_out, key_out=query if key_out is None else key_out)
    rows = check_payload(key, value, slots)
    shape = check_rotation(query, key, rows, positions, cos_sin)
    check_result(query_out, "query_out", query, shape)
    if key_out is not None:
        check_result(key_out, "key_out", key, rows)
    _write(query, shape[1], key, value, rows, positions, cos_sin, (key_codes, key_scales, value_codes, value_scales), slots,
           query_out, key_out, interleaved)


def _write_kv_mxfp4_fake(key, value, key_codes, key_scales, value_codes, value_scales, slots) -> None:
    return None


@custom_op(name="cache_write_kv_mxfp4", fake_impl=_write_kv_mxfp4_fake,
           mutates_args=["key_codes", "key_scales", "value_codes", "value_scales"])
def write_kv_mxfp4(
    key: torch.Tensor,
    value: torch.Tensor,
    key_codes: torch.Tensor,
    key_scales: torch.Tensor,
    value_codes: torch.Tensor,
    value_scales: torch.Tensor,
    slots: torch.Tensor,
) -> None:
    """Write keys and values as they are: ``write_kv`` into a 4-bit cache.

    Args:
        key, value: ``[tokens, kv_heads, head_dim]`` fp16/bf16, row and head strides free.
        key_codes, key_scales, value_codes, value_scales: the planes (see the module).
        slots: int64 ``[tokens]``; those outside the cache are skipped, and none may come twice.
    """
    check_devices(key, "key", value=value, key_codes=key_codes, key_scales=key_scales, value_codes=value_codes,
                  value_scales=value_scales, slots=slots)
    rows = check_payload(key, value, slots)
    _write(None, 0, key, value, rows, None, None, (key_codes, key_scales, value_codes, value_scales), slots, None, None, False)


def _gather_cache_mxfp4_fake(codes, scales, slots, destination) -> None:
    return None


@custom_op(name="cache_gather_mxfp4", fake_impl=_gather_cache_mxfp4_fake, mutates_args=["destination"])
def gather_cache_mxfp4(codes: torch.Tensor, scales: torch.Tensor, slots: torch.Tensor, destination: torch.Tensor) -> None:
    """Rows of one 4-bit plane by slot, as values.

    Args:
        codes, scales: one plane (see the module).
        slots: int64 ``[n]``, repeats allowed; a slot outside the plane gives a zero row.
        destination: contiguous fp32/fp16/bf16 of ``n * kv_heads * head_dim`` elements, ``[n,
            kv_heads, head_dim]`` as ``varlen_attention`` takes keys and values.

    Every value of a cache is exact in fp32 and bf16. fp16 rounds, and has no value for what is held as 65536 or
    more: it comes back infinite. Of rows that were fp16 when they were written these are the magnitudes
    from 57344 on.
    """
    check_devices(codes, "codes", scales=scales, slots=slots, destination=destination)
    pages, kv_heads, page_size, dim = check_plane(codes, scales, "cache")
    if slots.ndim != 1 or slots.dtype != torch.int64:
        raise ValueError("gather slots must be a rank-1 int64 tensor")
    if destination.dtype not in _PAYLOAD_DTYPES:
        require_dtype(destination, "destination", _PAYLOAD_DTYPES)
    rows = slots.numel()
    if destination.numel() != rows * kv_heads * dim:
        raise ValueError("gather destination must hold one cache row per slot")
    if not destination.is_contiguous():
        raise ValueError("gather needs a contiguous destination")
    if rows == 0:
        return
    slots = slots.contiguous()
    with _lib.on_device(codes):
        _lib.call("ayk_kv_gather_mxfp4", codes.data_ptr(), scales.data_ptr(), pages, page_size, kv_heads, dim, slots.data_ptr(),
                  rows, destination.data_ptr(), _lib.dtype_code(destination.dtype), _lib.stream_of(codes))
