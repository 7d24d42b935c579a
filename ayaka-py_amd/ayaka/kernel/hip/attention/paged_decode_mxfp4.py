"""Attention of one new token per sequence over a KV cache in 4 bits, on the gfx950 kernels of
``csrc/paged_decode_mxfp4.hip``.

The cache is the one that ``rope_write_kv_mxfp4`` and ``write_kv_mxfp4`` fill (e2m1 codes and a
UE8M0 scale for every 32 dims, head-major planes); tables, lengths and masks are those of
``paged_decode_attention``. No counterpart in the reference. There is no CPU path.
"""

from __future__ import annotations

import torch

from ayaka.kernel.hip import _lib
from ayaka.kernel.hip._host import prepare_output, require_dtype
from ayaka.kernel.hip.attention._checks import (
    ATTENTION_DTYPES,
    check_heads,
    check_scale,
    check_window,
    new_output,
    on_device_of,
    rows_of_heads,
)
from ayaka.kernel.hip.cache.mxfp4_cache import check_planes
from ayaka.kernel.hip.cache.rope_cache import check_devices
from ayaka.kernel.ops import custom_op

__all__ = ["paged_decode_attention_mxfp4"]


def _paged_decode_attention_mxfp4_fake(query, key_codes, key_scales, value_codes, value_scales, block_tables, seq_lens,
                                       softmax_scale, window=0, sinks=0, out=None):
    return torch.empty(query.shape, dtype=query.dtype, device=query.device) if out is None else out


@custom_op(name="paged_decode_attention_mxfp4", fake_impl=_paged_decode_attention_mxfp4_fake, mutates_args=["out"])
def paged_decode_attention_mxfp4(
    query: torch.Tensor,
    key_codes: torch.Tensor,
    key_scales: torch.Tensor,
    value_codes: torch.Tensor,
    value_scales: torch.Tensor,
    block_tables: torch.Tensor,
    seq_lens: torch.Tensor,
    softmax_scale: float,
    window: int = 0,
    sinks: int = 0,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Softmax attention of one query token per sequence over its positions in a 4-bit cache.

    Args:
        query: ``[batch, heads, head_dim]`` fp16/bf16; the token at position ``seq_lens[b] - 1``,
            whose key and value the cache already holds. Row and head strides are free.
        key_codes, value_codes: uint8 ``[pages, kv_heads, page_size, head_dim / 2]``, contiguous;
            ``head_dim`` a multiple of 32 up to 256, ``page_size`` a multiple of 8, ``heads`` a
            multiple of ``kv_heads``.
        key_scales, value_scales: uint8 ``[pages, kv_heads, page_size, head_dim / 32]``.
        block_tables: int32 ``[batch, max_pages]``; entries past a sequence's last page are
            not read, and the positions of a page outside the cache count as hidden.
        seq_lens: int32 ``[batch]``; 0 (padding rows) gives a zero output.
        softmax_scale: factor of the scores, ``head_dim ** -0.5`` as a rule.
        window: positions a token sees, itself included; 0 for all.
        sinks: first positions that stay visible outside the window.
        out: optional contiguous ``[batch, heads, head_dim]`` of the query's dtype.

    Lengths and tables are read on the device only: the operator can be captured in a graph
    and replayed with new contents.
    """
    if not on_device_of(query, key_codes, key_scales, value_codes, value_scales, block_tables, seq_lens):
        check_devices(query, "query", key_codes=key_codes, key_scales=key_scales, value_codes=value_codes,
                      value_scales=value_scales, block_tables=block_tables, seq_lens=seq_lens)
    if query.dtype not in ATTENTION_DTYPES:
        require_dtype(query, "query", ATTENTION_DTYPES)
    if query.ndim != 3:
        raise ValueError("query must be [batch, heads, head_dim]")
    pages, kv_heads, page_size, cache_dim = check_planes(key_codes, key_scales, value_codes, value_scales)
    batch, heads, dim = query.shape
    if cache_dim != dim:
        raise ValueError(f"a cache of head_dim {cache_dim} does not match a query of head_dim {dim}")
    check_heads(heads, kv_heads, dim)
    if block_tables.dtype != torch.int32 or seq_lens.dtype != torch.int32:
        require_dtype(block_tables, "block_tables", (torch.int32,))
        require_dtype(seq_lens, "seq_lens", (torch.int32,))
    table = block_tables.shape
    if len(table) != 2 or table[0] != batch or (table[1] > 1 and block_tables.stride(1) != 1):
        raise ValueError("block_tables must be [batch, pages] with stride(1) == 1")
    if seq_lens.shape != (batch,) or not seq_lens.is_contiguous():
        raise ValueError("seq_lens must be a contiguous [batch] vector")
    check_window(window, sinks)
    check_scale(softmax_scale)
    if out is None:
        result = new_output(query)
    else:
        result = prepare_output(query, out, like_name="query")
        if not result.is_contiguous() or result.data_ptr() % 16:
            raise ValueError("out must be contiguous and 16-byte aligned")
    if batch == 0:
        return result
    query = rows_of_heads(query)
    width = table[1]
    need = _lib.query("ayk_paged_decode_attention_mxfp4_split_bytes", batch, heads, kv_heads, dim, width * page_size, window,
                      sinks)
    with _lib.on_device(query):
        workspace = torch.empty(need, dtype=torch.uint8, device=query.device) if need else None
        _lib.call("ayk_paged_decode_attention_mxfp4", query.data_ptr(), _lib.dtype_code(query.dtype), query.stride(0),
                  query.stride(1), key_codes.data_ptr(), key_scales.data_ptr(), value_codes.data_ptr(), value_scales.data_ptr(),
                  pages, page_size, block_tables.data_ptr(), block_tables.stride(0), width, seq_lens.data_ptr(), batch, heads,
                  kv_heads, dim, softmax_scale, window, sinks, result.data_ptr(), _lib.ptr(workspace), need,
                  _lib.stream_of(query))
    return result
