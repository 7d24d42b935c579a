"""Attention of packed sequences (prompts, chunks of prompts) with grouped heads, a sliding
window and first tokens that stay visible, on the gfx950 kernels of
``csrc/varlen_attention.hip``.

No counterpart in the reference's FP8 path. Keys and values are rows as the projections
give them, or as ``gather_cache`` reads them back from an fp8 cache for a chunk of a longer
prompt. There is no CPU path, and no backward: the package serves, it does not train.
"""

from __future__ import annotations

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

__all__ = ["varlen_attention"]


def _varlen_attention_fake(query, key, value, cu_seqlens_q, cu_seqlens_k, softmax_scale, causal=True, window=0, sinks=0,
                           out=None):
    return torch.empty(query.shape, dtype=query.dtype, device=query.device) if out is None else out


def _check(query, key, value, cu_seqlens_q, cu_seqlens_k) -> None:
    if not on_device_of(query, key, value, cu_seqlens_q, cu_seqlens_k):
        for t, name in ((query, "query"), (key, "key"), (value, "value"), (cu_seqlens_q, "cu_seqlens_q"),
                        (cu_seqlens_k, "cu_seqlens_k")):
            require_cuda(t, name)
            require_same_device(t, name, query, "query")
    dtype = query.dtype
    if dtype not in ATTENTION_DTYPES or key.dtype != dtype or value.dtype != dtype:
        require_dtype(query, "query", ATTENTION_DTYPES)
        require_dtype(key, "key", (dtype,))
        require_dtype(value, "value", (dtype,))
    shape, keys = query.shape, key.shape
    if len(shape) != 3:
        raise ValueError("query must be [tokens, heads, head_dim]")
    if len(keys) != 3 or keys != value.shape or keys[2] != shape[2]:
        raise ValueError("key and value must be [tokens, kv_heads, head_dim] of one shape, with the query's head_dim")
    check_heads(shape[1], keys[1], shape[2])
    for t, name in ((cu_seqlens_q, "cu_seqlens_q"), (cu_seqlens_k, "cu_seqlens_k")):
        if t.dtype != torch.int32:
            require_dtype(t, name, (torch.int32,))
        if t.ndim != 1 or t.shape[0] < 1 or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous [sequences + 1] vector")
    if cu_seqlens_q.shape != cu_seqlens_k.shape:
        raise ValueError("cu_seqlens_q and cu_seqlens_k must name the same sequences")


@custom_op(name="varlen_attention", fake_impl=_varlen_attention_fake, mutates_args=["out"])
def varlen_attention(
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    cu_seqlens_q: torch.Tensor,
    cu_seqlens_k: torch.Tensor,
    softmax_scale: float,
    causal: bool = True,
    window: int = 0,
    sinks: int = 0,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Softmax attention within each packed sequence.

    Args:
        query: ``[tokens, heads, head_dim]`` fp16/bf16, ``head_dim`` at most 256. Row and
            head strides are free (a slice of a fused projection is read in place).
        key, value: ``[key_tokens, kv_heads, head_dim]`` of the query's dtype; ``heads`` is a
            multiple of ``kv_heads``.
        cu_seqlens_q, cu_seqlens_k: int32 ``[sequences + 1]`` first rows, ascending from 0. A
            sequence's queries are the last positions of its keys, so a chunk of a prompt
            passes its new queries with all keys so far.
        softmax_scale: factor of the scores, ``head_dim ** -0.5`` as a rule.
        causal: a query sees no later position.
        window: positions a query sees, itself included (causal only); 0 for all.
        sinks: first positions that stay visible outside the window.
        out: optional contiguous ``[tokens, heads, head_dim]``.

    A query that sees nothing, and a row of no sequence, gives 0. Lengths are read on the
    device only: the operator can be captured in a graph and replayed with new contents.
    """
    _check(query, key, value, cu_seqlens_q, cu_seqlens_k)
    check_window(window, sinks)
    check_scale(softmax_scale)
    if window and not causal:
        raise ValueError("a window needs causal attention")
    if out is None:
        result = new_output(query)
    else:
        result = prepare_output(query, out, like_name="query")
        if not result.is_contiguous():
            raise ValueError("out must be contiguous")
    tokens, heads, dim = query.shape
    batch = cu_seqlens_q.shape[0] - 1
    if tokens == 0:
        return result
    if batch == 0:
        return result.zero_()
    query, key, value = rows_of_heads(query), rows_of_heads(key), rows_of_heads(value)
    # below 1024 keys a sequence on average no split is taken, and no workspace
    long = key.shape[0] >= 1024 * batch
    need = _lib.query("ayk_varlen_attention_split_workspace_bytes", batch, tokens, heads, dim) if long else 0
    workspace = torch.empty(need, dtype=torch.uint8, device=query.device) if need else None
    _lib.call("ayk_varlen_attention_split", query.data_ptr(), query.stride(0), query.stride(1), key.data_ptr(), key.stride(0),
              key.stride(1), value.data_ptr(), value.stride(0), value.stride(1), _lib.dtype_code(query.dtype),
              cu_seqlens_q.data_ptr(), cu_seqlens_k.data_ptr(), batch, tokens, key.shape[0], heads, key.shape[1], dim,
              softmax_scale, int(causal), window, sinks, result.data_ptr(), _lib.ptr(workspace), need,
              _lib.stream_of(query))
    return result
