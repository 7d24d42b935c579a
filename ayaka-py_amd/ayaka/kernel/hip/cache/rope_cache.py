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
from ayaka.kernel.hip.attention._checks import ATTENTION_DTYPES, MAX_HEAD_DIM, check_heads, on_device_of, rows_of_heads
from ayaka.kernel.hip.cache.cache_ops import _check_scale
from ayaka.kernel.ops import custom_op

__all__ = ["rope_write_kv"]

_FP8_DTYPES = (torch.float8_e4m3fn, torch.float8_e5m2)


def check_payload(key, value, slots) -> None:
    """Keys and values of one step and their slots."""
    if key.dtype not in ATTENTION_DTYPES or value.dtype != key.dtype:
        require_dtype(key, "key", ATTENTION_DTYPES)
        require_dtype(value, "value", (key.dtype,))
    if key.ndim != 3 or key.shape != value.shape:
        raise ValueError("key and value must be [tokens, kv_heads, head_dim] of one shape")
    if key.shape[1] < 1 or not 1 <= key.shape[2] <= MAX_HEAD_DIM:
        raise ValueError(f"key and value must have heads, and a head_dim between 1 and {MAX_HEAD_DIM}")
    check_index(slots, "slots", key.shape[0])


def check_index(index, name, tokens) -> None:
    if index.dtype != torch.int64:
        require_dtype(index, name, (torch.int64,))
    if index.shape != (tokens,):
        require_shape(index, name, (tokens,))


def check_rotation(query, key, positions, cos_sin) -> None:
    """Queries beside their keys, and the table that rotates both."""
    if query.dtype != key.dtype:
        require_dtype(query, "query", (key.dtype,))
    if query.ndim != 3 or query.shape[0] != key.shape[0] or query.shape[2] != key.shape[2]:
        raise ValueError("query must be [tokens, heads, head_dim] with the key's tokens and head_dim")
    check_heads(query.shape[1], key.shape[1], key.shape[2])
    check_index(positions, "positions", key.shape[0])
    if cos_sin.dtype != torch.float32:
        require_dtype(cos_sin, "cos_sin", (torch.float32,))
    if cos_sin.ndim != 2 or cos_sin.shape[0] < 1 or not cos_sin.is_contiguous():
        raise ValueError("cos_sin must be a contiguous [positions, rotary_dim] table")
    rotary = cos_sin.shape[1]
    if rotary < 2 or rotary % 2 or rotary > key.shape[2]:
        raise ValueError(f"rotary_dim must be even, at least 2 and at most head_dim {key.shape[2]}, got {rotary}")


def check_result(out, name, like, like_name) -> None:
    """A caller's buffer for rotated rows: any row and head stride, elements side by side."""
    if out.dtype != like.dtype:
        require_dtype(out, name, (like.dtype,))
    if out.shape != like.shape:
        require_shape(out, name, tuple(like.shape))
    require_same_device(out, name, like, like_name)
    if out.shape[2] > 1 and out.stride(2) != 1:
        raise ValueError(f"{name} must have stride(2) == 1")
    if any(n > 1 and s == 0 for n, s in zip(out.shape, out.stride())):
        raise ValueError(f"{name} must not overlap itself")


def check_devices(first, first_name, **others) -> None:
    """All operands on one CUDA device, named where one is not."""
    if not on_device_of(first, *others.values()):
        require_cuda(first, first_name)
        for name, t in others.items():
            require_cuda(t, name)
            require_same_device(t, name, first, first_name)


def rows_and_strides(t: torch.Tensor | None) -> tuple:
    """Address and the row and head strides of ``[tokens, heads, dim]`` rows."""
    return (None, 0, 0) if t is None else (t.data_ptr(), t.stride(0), t.stride(1))


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
    others = {"key": key, "value": value, "positions": positions, "cos_sin": cos_sin, "key_cache": key_cache,
              "value_cache": value_cache, "slots": slots, "query_out": query_out}
    if key_out is not None:
        others["key_out"] = key_out
    check_devices(query, "query", **others)
    _check_scale(k_inverse, v_inverse)
    check_payload(key, value, slots)
    check_rotation(query, key, positions, cos_sin)
    tokens, heads, dim = query.shape
    kv_heads, cache = key.shape[1], key_cache.shape
    if key_cache.dtype not in _FP8_DTYPES and key_cache.dtype != key.dtype:
        require_dtype(key_cache, "key_cache", (*_FP8_DTYPES, key.dtype))
    if len(cache) != 4 or cache != value_cache.shape or value_cache.dtype != key_cache.dtype or cache[2:] != key.shape[1:]:
        raise ValueError("key_cache and value_cache must be [pages, page_size, kv_heads, head_dim] of one dtype, for the key's heads")
    if not key_cache.is_contiguous() or not value_cache.is_contiguous():
        raise ValueError("KV cache pages must be contiguous")
    check_result(query_out, "query_out", query, "query")
    if key_out is not None:
        check_result(key_out, "key_out", key, "key")
    if tokens == 0:
        return
    query, key, value = rows_of_heads(query), rows_of_heads(key), rows_of_heads(value)
    positions, slots = positions.contiguous(), slots.contiguous()
    with _lib.on_device(query):
        _lib.call("ayk_rope_kv_write", *rows_and_strides(query), *rows_and_strides(key), *rows_and_strides(value),
                  _lib.dtype_code(query.dtype), tokens, heads, kv_heads, dim, positions.data_ptr(), cos_sin.data_ptr(),
                  cos_sin.shape[0], cos_sin.shape[1], int(interleaved), *rows_and_strides(query_out), *rows_and_strides(key_out),
                  key_cache.data_ptr(), value_cache.data_ptr(), _lib.dtype_code(key_cache.dtype), cache[0] * cache[1],
                  slots.data_ptr(), k_inverse, v_inverse, _lib.stream_of(query))
