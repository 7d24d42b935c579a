"""Root-mean-square norm with the residual's addition and e4m3 output, on the gfx950 kernels
of ``csrc/norm_quant.hip``.

One pass instead of an addition, a norm and a quantizer: ``h = x + residual`` is stored as
the new residual, ``y = h * weight / sqrt(mean(h^2) + eps)`` is formed in fp32 from the
unrounded ``h`` and quantized by the rules of ``per_token_quant_fp8`` (``group_size=0``),
``per_token_group_quant_fp8`` or, with ``scale_dtype="e8m0"``, ``per_token_group_quant_mxfp8``.
What it returns feeds ``fp8_scaled_mm``, ``fp8_blockwise_mm`` and ``mxfp8_scaled_mm``. The
reference's FP8 path has no such operator.
"""

from __future__ import annotations

import math

import torch

from ayaka.kernel.hip import _lib
from ayaka.kernel.hip._host import require_cuda, require_dtype, require_same_device
from ayaka.kernel.hip.quant.fp8_quant import _check_group_size, _rows_2d, _validate_input
from ayaka.kernel.ops import custom_op

__all__ = ["add_rms_norm_quant_fp8", "rms_norm_quant_fp8"]

FP8 = torch.float8_e4m3fn
_FLOAT_DTYPES = (torch.float16, torch.bfloat16, torch.float32)
_SCALE_DTYPES = {"float32": torch.float32, "e8m0": torch.uint8}


def _outputs(x, group_size, scale_dtype, scale_col_major):
    *lead, k = x.shape
    rows = math.prod(lead)
    shape = (rows,) if group_size == 0 else (k // group_size, rows) if scale_col_major else (rows, k // group_size)
    q = (torch.empty_like(x, dtype=FP8, memory_format=torch.contiguous_format) if len(lead) == 1
         else x.new_empty((rows, k), dtype=FP8))
    return q, x.new_empty(shape, dtype=_SCALE_DTYPES[scale_dtype])


def _rms_norm_quant_fake(x, weight, eps, group_size=0, scale_dtype="float32", scale_col_major=False):
    return _outputs(x, group_size, scale_dtype, scale_col_major)


def _add_rms_norm_quant_fake(x, residual, weight, eps, group_size=0, scale_dtype="float32", scale_col_major=False):
    return (*_outputs(x, group_size, scale_dtype, scale_col_major), torch.empty(x.shape, dtype=x.dtype, device=x.device))


def _check(x, weight, eps, group_size, scale_dtype, scale_col_major) -> None:
    shape = x.shape
    if x.dtype not in _FLOAT_DTYPES or not x.is_cuda or not shape:
        _validate_input(x, "x")
    k = shape[-1]
    if k < 1:
        raise ValueError("x must have a positive last dimension")
    if weight.dtype not in _FLOAT_DTYPES or weight.get_device() != x.get_device():
        require_cuda(weight, "weight")
        require_dtype(weight, "weight", _FLOAT_DTYPES)
        require_same_device(weight, "weight", x, "x")
    if weight.shape != (k,) or not weight.is_contiguous():
        raise ValueError(f"weight must be a contiguous vector of shape [{k}]")
    if not (math.isfinite(eps) and eps >= 0):
        raise ValueError("eps must be finite and not negative")
    if scale_dtype not in _SCALE_DTYPES:
        raise ValueError("scale_dtype must be 'float32' or 'e8m0'")
    if group_size == 0 and not isinstance(group_size, bool):
        if scale_dtype == "e8m0" or scale_col_major:
            raise ValueError("e8m0 and column-major scales need a group_size")
        return
    _check_group_size(group_size, pow2=scale_dtype == "float32")
    if k % group_size:
        raise ValueError(f"K={k} must be divisible by group_size={group_size}")


def _rows(x, rows, k):
    """``x`` as ``[rows, k]`` with unit stride along ``k``, and the distance of its rows."""
    if not x.is_contiguous():
        x = _rows_2d(x)
        return x, x.stride(0) if rows > 1 else k
    return x, k


def _launch(x, residual, weight, eps, group_size, scale_dtype, scale_col_major):
    q, scale = _outputs(x, group_size, scale_dtype, scale_col_major)
    rows, k = q.shape
    residual_out = None if residual is None else torch.empty_like(x, memory_format=torch.contiguous_format)
    if rows:
        x2d, ldx = _rows(x, rows, k)
        r2d, ldr = (None, 0) if residual is None else _rows(residual, rows, k)
        scale_row, scale_group = (1, rows) if scale_col_major else (k // group_size if group_size else 1, 1)
        _lib.call("ayk_rms_norm_quant_fp8", x2d.data_ptr(), _lib.dtype_code(x.dtype), rows, k, ldx, _lib.ptr(r2d), ldr,
                  weight.data_ptr(), _lib.dtype_code(weight.dtype), eps, group_size, _lib.dtype_code(scale.dtype),
                  q.data_ptr(), scale.data_ptr(), scale_row, scale_group, _lib.ptr(residual_out), _lib.stream_of(x))
    return q, scale, residual_out


@custom_op(name="rms_norm_quant_fp8", fake_impl=_rms_norm_quant_fake)
def rms_norm_quant_fp8(
    x: torch.Tensor,
    weight: torch.Tensor,
    eps: float,
    group_size: int = 0,
    scale_dtype: str = "float32",
    scale_col_major: bool = False,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Norm and quantize ``x``, without a residual.

    Args:
        x: ``[..., K]`` fp16/bf16/fp32.
        weight: contiguous ``[K]`` fp16/bf16/fp32.
        eps: added to the mean square.
        group_size: K elements per scale (a power of two dividing ``K``; any divisor for
            e8m0); 0 for one scale per row.
        scale_dtype: ``"float32"``, or ``"e8m0"`` for MXFP8 exponent codes.
        scale_col_major: store group scales ``[K // group_size, M]``, the layout of
            ``fp8_blockwise_mm(..., a_scale_col_major=True)``.

    Returns:
        ``(q [M, K] e4m3, scale [M] or [M, K // group_size])``, ``M = numel // K``.
    """
    _check(x, weight, eps, group_size, scale_dtype, scale_col_major)
    return _launch(x, None, weight, eps, group_size, scale_dtype, scale_col_major)[:2]


@custom_op(name="add_rms_norm_quant_fp8", fake_impl=_add_rms_norm_quant_fake)
def add_rms_norm_quant_fp8(
    x: torch.Tensor,
    residual: torch.Tensor,
    weight: torch.Tensor,
    eps: float,
    group_size: int = 0,
    scale_dtype: str = "float32",
    scale_col_major: bool = False,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``rms_norm_quant_fp8`` of ``x + residual``; also returns that sum, of ``x``'s shape and
    dtype, as the next residual. ``residual`` has ``x``'s shape and dtype and is not changed.
    """
    _check(x, weight, eps, group_size, scale_dtype, scale_col_major)
    if residual.get_device() != x.get_device():
        require_cuda(residual, "residual")
        require_same_device(residual, "residual", x, "x")
    if residual.shape != x.shape or residual.dtype != x.dtype:
        raise ValueError("residual must have x's shape and dtype")
    return _launch(x, residual, weight, eps, group_size, scale_dtype, scale_col_major)
