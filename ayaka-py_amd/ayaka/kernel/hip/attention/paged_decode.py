"""Attention of one new token per sequence over the paged KV cache, on the gfx950 kernels of
``csrc/paged_decode.hip``.

The cache is the one ``write_kv`` fills: ``[pages, page_size, kv_heads, head_dim]``, fp8 with
one static scale per plane or the query's own 16-bit dtype. Position ``j`` of row ``b`` lies
at slot ``block_tables[b, j // page_size] * page_size + j % page_size``. The reference's FP8
path ends at the cache; this operator has no counterpart there. There is no CPU path.
"""

from __future__ import annotations

import math

import torch

from ayaka.kernel.hip import _lib
from ayaka.kernel.hip._host import prepare_output, require_cuda, require_dtype, require_same_device
from ayaka.kernel.hip.attention._checks import (
    ATTENTION_DTYPES,
    check_heads,
    check_scale,
    check_window,
    new_output,
    on_device_of,
    rows_of_heads,
)
from ayaka.kernel.ops import custom_op

__all__ = ["paged_decode_attention"]

_FP8_DTYPES = (torch.float8_e4m3fn, torch.float8_e5m2)


def _paged_decode_attention_fake(query, key_cache, value_cache, block_tables, seq_lens, softmax_scale, k_scale=1.0,
                                 v_scale=1.0, window=0, sinks=0, out=None):
    return torch.empty(query.shape, dtype=query.dtype, device=query.device) if out is None else out


def _check(query, key_cache, value_cache, block_tables, seq_lens) -> None:
    if not on_device_of(query, key_cache, value_cache, block_tables, seq_lens):
        for t, name in ((query, "query"), (key_cache, "key_cache"), (value_cache, "value_cache"),
                        (block_tables, "block_tables"), (seq_lens, "seq_lens")):
            require_cuda(t, name)
            require_same_device(t, name, query, "query")
    dtype = query.dtype
    if dtype not in ATTENTION_DTYPES:
        require_dtype(query, "query", ATTENTION_DTYPES)
    if key_cache.dtype not in _FP8_DTYPES and key_cache.dtype != dtype:
        require_dtype(key_cache, "key_cache", (*_FP8_DTYPES, dtype))
    shape, cache = query.shape, key_cache.shape
    if len(shape) != 3:
        raise ValueError("query must be [batch, heads, head_dim]")
    if len(cache) != 4 or cache != value_cache.shape or key_cache.dtype != value_cache.dtype:
        raise ValueError("key_cache and value_cache must be [pages, page_size, kv_heads, head_dim] of one shape and dtype")
    if not key_cache.is_contiguous() or not value_cache.is_contiguous():
        raise ValueError("KV cache pages must be contiguous")
    batch, heads, dim = shape
    if cache[1] < 1 or cache[3] != dim:
        raise ValueError(f"cache {tuple(cache)} does not match a query of head_dim {dim}")
    check_heads(heads, cache[2], dim)
    if block_tables.dtype != torch.int32 or seq_lens.dtype != torch.int32:
        require_dtype(block_tables, "block_tables", (torch.int32,))
        require_dtype(seq_lens, "seq_lens", (torch.int32,))
    table = block_tables.shape
    if len(table) != 2 or table[0] != batch or (table[1] > 1 and block_tables.stride(1) != 1):
        raise ValueError("block_tables must be [batch, pages] with stride(1) == 1")
    if seq_lens.shape != (batch,) or not seq_lens.is_contiguous():
        raise ValueError("seq_lens must be a contiguous [batch] vector")


@custom_op(name="paged_decode_attention", fake_impl=_paged_decode_attention_fake, mutates_args=["out"])
def paged_decode_attention(
    query: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    block_tables: torch.Tensor,
    seq_lens: torch.Tensor,
    softmax_scale: float,
    k_scale: float = 1.0,
    v_scale: float = 1.0,
    window: int = 0,
    sinks: int = 0,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Softmax attention of one query token per sequence over its cached positions.

    Args:
        query: ``[batch, heads, head_dim]`` fp16/bf16, ``head_dim`` at most 256; the token at
            position ``seq_lens[b] - 1``, whose key and value the cache already holds.
        key_cache, value_cache: contiguous ``[pages, page_size, kv_heads, head_dim]``,
            e4m3fn / e5m2 or the query's dtype; ``heads`` is a multiple of ``kv_heads``.
        block_tables: int32 ``[batch, max_pages]``; entries past a sequence's last page are
            not read, and the positions of a page outside the cache count as hidden. The launch
            is chosen from the width: short sequences through a table for long ones take up
            to 5 us more than through one of their own width.
        seq_lens: int32 ``[batch]``; 0 (padding rows) gives a zero output.
        softmax_scale: factor of the scores, ``head_dim ** -0.5`` as a rule.
        k_scale, v_scale: dequantization scales of an fp8 cache (the inverses of what
            ``write_kv`` was given).
        window: positions a token sees, itself included; 0 for all.
        sinks: first positions that stay visible outside the window.
        out: optional contiguous ``[batch, heads, head_dim]`` of the query's dtype.

    Lengths and tables are read on the device only: the operator can be captured in a graph
    and replayed with new contents.
    """
    _check(query, key_cache, value_cache, block_tables, seq_lens)
    check_window(window, sinks)
    check_scale(softmax_scale)
    if not (0.0 < k_scale < math.inf and 0.0 < v_scale < math.inf):
        raise ValueError("KV scales must be finite and positive")
    if out is None:
        result = new_output(query)
    else:
        result = prepare_output(query, out, like_name="query")
        if not result.is_contiguous():
            raise ValueError("out must be contiguous")
    batch, heads, dim = query.shape
    if batch == 0:
        return result
    query = rows_of_heads(query)
    pages, page_size, kv_heads, _ = key_cache.shape
    width = block_tables.shape[1]
    cache_code = _lib.dtype_code(key_cache.dtype)
    need = _lib.query("ayk_paged_decode_attention_split_bytes", batch, heads, kv_heads, dim, cache_code, width * page_size,
                      window, sinks)
    workspace = torch.empty(need, dtype=torch.uint8, device=query.device) if need else None
    _lib.call("ayk_paged_decode_attention", query.data_ptr(), _lib.dtype_code(query.dtype), query.stride(0), query.stride(1),
              key_cache.data_ptr(), value_cache.data_ptr(), cache_code, pages, page_size, block_tables.data_ptr(),
              block_tables.stride(0), width, seq_lens.data_ptr(), batch, heads, kv_heads, dim, softmax_scale, k_scale, v_scale,
              window, sinks, result.data_ptr(), _lib.ptr(workspace), need, _lib.stream_of(query))
    return result
