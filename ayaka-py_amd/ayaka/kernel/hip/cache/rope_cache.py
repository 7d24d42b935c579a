"""Position rotation of queries and keys with the append to the paged KV cache, on the gfx950
kernels of ``csrc/rope_kv.hip``.

``rope_write_kv`` fills the caches that ``write_kv`` fills and ``paged_decode_attention``
reads, with the same rounding of every value. The reference rotates in its model code and
then calls ``write_kv``; the fused operator has no counterpart there. There is no CPU path.
"""

from __future__ import annotations

import torch

from ayaka.kernel.hip import _lib
from ayaka.kernel.hip._host import require_cuda, require_dtype, require_same_device, require_shape
from ayaka.kernel.hip.attention._checks import ATTENTION_DTYPES, MAX_HEAD_DIM, check_heads, on_device_of
from ayaka.kernel.hip.cache.cache_ops import _check_scale
from ayaka.kernel.ops import custom_op

__all__ = ["rope_write_kv"]

_FP8_DTYPES = (torch.float8_e4m3fn, torch.float8_e5m2)


def check_payload(key, value, slots) -> torch.Size:
    """Keys and values of one step and their slots; their shape."""
    if key.dtype not in ATTENTION_DTYPES or value.dtype != key.dtype:
        require_dtype(key, "key", ATTENTION_DTYPES)
        require_dtype(value, "value", (key.dtype,))
    shape = key.shape
    if len(shape) != 3 or shape != value.shape:
        raise ValueError("key and value must be [tokens, kv_heads, head_dim] of one shape")
    tokens, kv_heads, dim = shape
    if kv_heads < 1 or not 1 <= dim <= MAX_HEAD_DIM:
        raise ValueError(f"key and value must have heads, and a head_dim between 1 and {MAX_HEAD_DIM}")
    check_index(slots, "slots", tokens)
    return shape


def check_index(index, name, tokens) -> None:
    if index.dtype != torch.int64:
        require_dtype(index, name, (torch.int64,))
    if index.shape != (tokens,):
        require_shape(index, name, (tokens,))


def check_rotation(query, key, shape, positions, cos_sin) -> torch.Size:
    """Queries beside their keys (of that shape), and the table that rotates both; the queries' shape."""
    if query.dtype != key.dtype:
        require_dtype(query, "query", (key.dtype,))
    queries, (tokens, kv_heads, dim) = query.shape, shape
    if len(queries) != 3 or queries[0] != tokens or queries[2] != dim:
        raise ValueError("query must be [tokens, heads, head_dim] with the key's tokens and head_dim")
    check_heads(queries[1], kv_heads, dim)
    check_index(positions, "positions", tokens)
    if cos_sin.dtype != torch.float32:
        require_dtype(cos_sin, "cos_sin", (torch.float32,))
    if cos_sin.ndim != 2 or cos_sin.shape[0] < 1 or not cos_sin.is_contiguous():
        raise ValueError("cos_sin must be a contiguous [positions, rotary_dim] table")
    rotary = cos_sin.shape[1]
    if rotary < 2 or rotary % 2 or rotary > dim:
        raise ValueError(f"rotary_dim must be even, at least 2 and at most head_dim {dim}, got {rotary}")
    return queries


def check_result(out, name, like, shape) -> None:
    """A caller's buffer for rotated rows: any row and head stride, elements side by side."""
    if out.dtype != like.dtype:
        require_dtype(out, name, (like.dtype,))
    if out.shape != shape:
        require_shape(out, name, tuple(shape))
    row, head, unit = out.stride()
    if unit != 1 and shape[2] > 1:
        raise ValueError(f"{name} must have stride(2) == 1")
    if (row == 0 and shape[0] > 1) or (head == 0 and shape[1] > 1):
        raise ValueError(f"{name} must not overlap itself")


def check_devices(first, first_name, **others) -> None:
    """All operands on one CUDA device, named where one is not."""
    if not on_device_of(first, *others.values()):
        require_cuda(first, first_name)
        for name, t in others.items():
            require_cuda(t, name)
            require_same_device(t, name, first, first_name)


def packed_rows(t: torch.Tensor | None) -> tuple:
    """``[tokens, heads, dim]`` rows with unit stride along ``dim`` (a copy only where it has another): the
    tensor, its address, its row and head strides."""
    if t is None:
        return None, None, 0, 0
    row, head, unit = t.stride()
    if unit != 1 and t.shape[2] != 1:
        t = t.contiguous()
        row, head, _ = t.stride()
    return t, t.data_ptr(), row, head


def _rope_write_kv_fake(query, key, value, positions, cos_sin, key_cache, value_cache, slots, k_inverse, v_inverse, query_out,
                        key_out=None, interleaved=False) -> None:
    return None


@custom_op(name="rope_write_kv", fake_impl=_rope_write_kv_fake,
           mutates_args=["key_cache", "value_cache", "query_out", "key_out"])
def rope_write_kv(
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    positions: torch.Tensor,
    cos_sin: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    slots: torch.Tensor,
    k_inverse: float,
    v_inverse: float,
    query_out: torch.Tensor,
    key_out: torch.Tensor | None = None,
    interleaved: bool = False,
) -> None:
    """Rotate a step's queries and keys and write keys and values to the paged cache.

    Args:
        query: ``[tokens, heads, head_dim]`` fp16/bf16, ``head_dim`` at most 256. Row and head
            strides are free, here and below (a slice of a fused projection is read in place).
        key, value: ``[tokens, kv_heads, head_dim]`` of the query's dtype; ``heads`` is a
            multiple of ``kv_heads``.
        positions: int64 ``[tokens]``, rows of ``cos_sin``.
        cos_sin: contiguous fp32 ``[positions, rotary_dim]``: the cosines of a position's
            ``rotary_dim / 2`` angles, then their sines. Dims from ``rotary_dim`` on pass through.
        key_cache, value_cache: contiguous ``[pages, page_size, kv_heads, head_dim]``, e4m3fn /
            e5m2 or the query's dtype.
        slots: int64 ``[tokens]``, ``page * page_size + offset``. A token with a slot outside the
            cache (padding: a negative one) is rotated, and not written. No slot may come twice.
        k_inverse, v_inverse: inverse static scales of an fp8 cache, as in ``write_kv``.
        query_out: ``[tokens, heads, head_dim]`` of the query's dtype, the rotated queries. May be
            ``query`` itself; no other overlap of an output with an input is allowed.
        key_out: optional ``[tokens, kv_heads, head_dim]``, the rotated keys in 16 bits, for
            attention over the step's own rows. May be ``key`` itself.
        interleaved: the pairs are dims ``(2 i, 2 i + 1)`` instead of ``(i, i + rotary_dim / 2)``.

    A token whose position is outside the table gives zero rows and is not written.
    """
    # (a dictionary of names only where an operand is refused)
    if not on_device_of(query, key, value, positions, cos_sin, key_cache, value_cache, slots, query_out,
                        query if key_out is None else key_out):
        check_devices(query, "query", key=key, value=value, positions=positions, cos_sin=cos_sin, key_cache=key_cache,
                      value_cache=value_cache, slots=slots, query_out=query_out, key_out=query if key_out is None else key_out)
    _check_scale(k_inverse, v_inverse)
    rows = check_payload(key, value, slots)
    shape = check_rotation(query, key, rows, positions, cos_sin)
    tokens, kv_heads, dim = rows
    cache, kind = key_cache.shape, key_cache.dtype
    if kind not in _FP8_DTYPES and kind != key.dtype:
        require_dtype(key_cache, "key_cache", (*_FP8_DTYPES, key.dtype))
    if len(cache) != 4 or cache != value_cache.shape or value_cache.dtype != kind or cache[2] != kv_heads or cache[3] != dim:
        raise ValueError("key_cache and value_cache must be [pages, page_size, kv_heads, head_dim] of one dtype, for the key's heads")
    if not key_cache.is_contiguous() or not value_cache.is_contiguous():
        raise ValueError("KV cache pages must be contiguous")
    check_result(query_out, "query_out", query, shape)
    if key_out is not None:
        check_result(key_out, "key_out", key, rows)
    if tokens == 0:
        return
    # (the tensors stay referenced: a copy's memory must not be handed out before the launch)
    query, *q = packed_rows(query)
    key, *k = packed_rows(key)
    value, *v = packed_rows(value)
    positions, slots = positions.contiguous(), slots.contiguous()
    with _lib.on_device(query):
        _lib.call("ayk_rope_kv_write", *q, *k, *v, _lib.dtype_code(query.dtype), tokens, shape[1], kv_heads, dim,
                  positions.data_ptr(), cos_sin.data_ptr(), *cos_sin.shape, int(interleaved), *packed_rows(query_out)[1:],
                  *packed_rows(key_out)[1:], key_cache.data_ptr(), value_cache.data_ptr(), _lib.dtype_code(kind),
                  cache[0] * cache[1], slots.data_ptr(), k_inverse, v_inverse, _lib.stream_of(query))
