"""A mixture-of-experts layer for the few tokens of a decode step, on the gfx950 kernels of
``csrc/moe_small.hip``.

The experts' weights and block scales are those of ``fp8_blockwise_scaled_grouped_mm``, which
larger batches take, with its tables, a quantizer, the activation and the weighted sum around
it. Here all of it is two launches and the activations stay 16-bit. The reference has no
counterpart. There is no CPU path.
"""

from __future__ import annotations

import torch

from ayaka.kernel.hip import _lib
from ayaka.kernel.hip._host import prepare_output, require_cuda, require_dtype, require_same_device, require_shape
from ayaka.kernel.hip.attention._checks import ATTENTION_DTYPES, on_device_of
from ayaka.kernel.ops import custom_op

__all__ = ["MAX_TOKENS", "fp8_block_moe_small"]

MAX_TOKENS = 64
MAX_EXPERTS = 1024
BLOCK = 128


def _fp8_block_moe_small_fake(x, gate_up, gate_up_scale, down, down_scale, topk_weights, topk_ids, out=None):
    return torch.empty(x.shape, dtype=x.dtype, device=x.device) if out is None else out


def _check_experts(codes, scale, name, shape) -> None:
    if codes.dtype != torch.float8_e4m3fn or scale.dtype != torch.float32:
        require_dtype(codes, name, (torch.float8_e4m3fn,))
        require_dtype(scale, f"{name}_scale", (torch.float32,))
    experts, rows, columns = shape
    if codes.shape != shape or scale.shape != (experts, rows // BLOCK, columns // BLOCK):
        require_shape(codes, name, shape)
        require_shape(scale, f"{name}_scale", (experts, rows // BLOCK, columns // BLOCK))
    if not codes.is_contiguous() or not scale.is_contiguous():
        raise ValueError(f"{name} and its scales must be contiguous")


def _check(x, gate_up, gate_up_scale, down, down_scale, topk_weights, topk_ids) -> None:
    if not on_device_of(x, gate_up, gate_up_scale, down, down_scale, topk_weights, topk_ids):
        require_cuda(x, "x")
        for name, t in (("gate_up", gate_up), ("gate_up_scale", gate_up_scale), ("down", down), ("down_scale", down_scale),
                        ("topk_weights", topk_weights), ("topk_ids", topk_ids)):
            require_cuda(t, name)
            require_same_device(t, name, x, "x")
    if x.dtype not in ATTENTION_DTYPES:
        require_dtype(x, "x", ATTENTION_DTYPES)
    if x.ndim != 2 or gate_up.ndim != 3 or down.ndim != 3:
        raise ValueError("x must be [tokens, hidden], gate_up [experts, 2 * inner, hidden] and down [experts, hidden, inner]")
    tokens, hidden = x.shape
    experts, inner = down.shape[0], down.shape[2]
    if tokens > MAX_TOKENS:
        raise ValueError(f"at most {MAX_TOKENS} tokens, got {tokens}: larger batches take fp8_blockwise_scaled_grouped_mm")
    if not 1 <= experts <= MAX_EXPERTS:
        raise ValueError(f"1 to {MAX_EXPERTS} experts, got {experts}")
    if hidden < BLOCK or inner < BLOCK or hidden % BLOCK or inner % BLOCK:
        raise ValueError(f"hidden and inner must be multiples of {BLOCK}, got {hidden} and {inner}")
    _check_experts(gate_up, gate_up_scale, "gate_up", (experts, 2 * inner, hidden))
    _check_experts(down, down_scale, "down", (experts, hidden, inner))
    if topk_weights.dtype != torch.float32 or topk_ids.dtype != torch.int32:
        require_dtype(topk_weights, "topk_weights", (torch.float32,))
        require_dtype(topk_ids, "topk_ids", (torch.int32,))
    if topk_ids.ndim != 2 or topk_ids.shape[0] != tokens or topk_ids.shape[1] < 1 or topk_weights.shape != topk_ids.shape:
        raise ValueError("topk_weights and topk_ids must be [tokens, topk]")


@custom_op(name="fp8_block_moe_small", fake_impl=_fp8_block_moe_small_fake, mutates_args=["out"])
def fp8_block_moe_small(
    x: torch.Tensor,
    gate_up: torch.Tensor,
    gate_up_scale: torch.Tensor,
    down: torch.Tensor,
    down_scale: torch.Tensor,
    topk_weights: torch.Tensor,
    topk_ids: torch.Tensor,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """``out[t] = sum_j topk_weights[t, j] * down[e] (silu(gate[e] x[t]) * (up[e] x[t]))``, ``e = topk_ids[t, j]``.

    Args:
        x: ``[tokens, hidden]`` fp16/bf16, at most 64 tokens; rows may be strided.
        gate_up: contiguous e4m3fn ``[experts, 2 * inner, hidden]``, an expert's gate rows and
            then its up rows; at most 1024 experts, ``hidden`` and ``inner`` multiples of 128.
        gate_up_scale: contiguous fp32 ``[experts, 2 * inner / 128, hidden / 128]``.
        down, down_scale: ``[experts, hidden, inner]`` and ``[experts, hidden / 128, inner / 128]``.
        topk_weights: fp32 ``[tokens, topk]``, used as they are.
        topk_ids: int32 ``[tokens, topk]``. An id outside the experts (-1: an expert that
            another rank holds) counts nothing; a token without experts gives zeros. An expert
            that a token names twice counts with both weights.
        out: optional ``[tokens, hidden]`` of x's dtype, rows may be strided; must not overlap x.

    Products are of the 16-bit activations and the exact weights, sums fp32; what lies between
    the projections keeps 16 significant bits. Ids are read on the device only: the operator
    can be captured in a graph and replayed with new contents.
    """
    _check(x, gate_up, gate_up_scale, down, down_scale, topk_weights, topk_ids)
    tokens, hidden = x.shape
    if out is None:
        result = torch.empty((tokens, hidden), dtype=x.dtype, device=x.device)
    else:
        result = prepare_output(x, out, like_name="x")
        if result.stride(1) != 1 or (tokens > 1 and result.stride(0) < hidden):
            raise ValueError("out must have stride(1) == 1 and rows that do not overlap")
    if tokens == 0:
        return result
    if x.stride(1) != 1 or x.data_ptr() % 16 or (tokens > 1 and (x.stride(0) < hidden or x.stride(0) % 8)):
        x = x.clone(memory_format=torch.contiguous_format)
    topk_weights, topk_ids = topk_weights.contiguous(), topk_ids.contiguous()
    experts, inner, topk = down.shape[0], down.shape[2], topk_ids.shape[1]
    need = _lib.query("ayk_fp8_block_moe_small_scratch_bytes", tokens, topk, experts, hidden, inner)
    with _lib.on_device(x):
        workspace = torch.empty(need, dtype=torch.uint8, device=x.device)
        _lib.call("ayk_fp8_block_moe_small", x.data_ptr(), _lib.dtype_code(x.dtype), x.stride(0) if tokens > 1 else hidden, tokens,
                  gate_up.data_ptr(), gate_up_scale.data_ptr(), down.data_ptr(), down_scale.data_ptr(), experts, hidden, inner,
                  topk_weights.data_ptr(), topk_ids.data_ptr(), topk, result.data_ptr(),
                  result.stride(0) if tokens > 1 else hidden, workspace.data_ptr(), need, _lib.stream_of(x))
    return result
