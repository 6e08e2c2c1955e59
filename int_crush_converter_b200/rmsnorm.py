"""Residual addition, RMS norm, group Hadamard and quantization of activations in one pass."""

from __future__ import annotations

import torch

from . import _native as nat
from ._dev import back, call, device_of
from .fp4 import FORMATS, FP4Tensor, as_rows, empty_fp4, padded_columns, pitch
from .int8 import Int8Rows, empty_int8
from .rotation import _DT

_FORMATS = {"int8": nat.IC_INT8, **FORMATS}


def rmsnorm_quantize(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, eps: float = 1e-6,
                     fmt: str = "int8", rot_size: int = 0) -> tuple[Int8Rows | FP4Tensor, torch.Tensor | None]:
    """h = x + residual; y = h / sqrt(mean(h^2) + eps) * weight, rotated and quantized.

    x, residual: [..., K] of one type (fp32/fp16/bf16); weight [K].  ``fmt``: "int8"
    (:class:`Int8Rows`, the operand of ``matmul_int8``), "mxfp4" or "nvfp4"
    (:class:`FP4Tensor`, of ``matmul_fp4``).  ``rot_size``: 0 or a power of two in
    16..512, the group Hadamard that the layer's weights were rotated with.
    Returns (quantized rows, h in x's type), h None without a residual.  The sums
    and the norm are fp32 or wider, and the norm goes on from the fp32 sum
    x + residual, not from the rounded h that is returned: a layer that norms its
    rounded stream can get another code where a value lies next to a border.  A
    row with a value that is not finite has scale NaN (mxfp4: every block).
    """
    if fmt not in _FORMATS:
        raise ValueError(f"fmt must be one of {sorted(_FORMATS)}, got {fmt!r}")
    parts = nat.binding().rmsnorm_quantize(x, weight, residual, eps, _FORMATS[fmt], rot_size)
    if parts is not None:
        a, b, c, h = parts
        if fmt == "int8":
            return Int8Rows(a, b, c, x.shape[-1], rot_size, x.shape[:-1]), h
        return FP4Tensor(a, b, c, fmt, x.shape[-1], rot_size, x.shape[:-1]), h
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("rmsnorm_quantize needs at least one column")
    if x.dtype not in _DT or weight.dtype not in _DT:
        raise ValueError(f"x and weight must be float32, float16 or bfloat16, got {x.dtype} and {weight.dtype}")
    k = x.shape[-1]
    if weight.numel() != k:
        raise ValueError(f"weight must have {k} values, got {weight.numel()}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError("residual must have x's shape and type")
    if residual is not None and residual.device != x.device:
        raise ValueError("residual must be on x's device")
    if rot_size and (rot_size & (rot_size - 1) or not 16 <= rot_size <= 512):
        raise ValueError(f"rot_size must be 0 or a power of 2 in 16..512, got {rot_size}")
    if not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    dev = device_of(x)
    lead = x.shape[:-1]
    x2 = as_rows(x, dev)
    r2 = None if residual is None else as_rows(residual, dev)
    w = weight.to(dev).reshape(-1).contiguous()
    rows, kp = x2.shape[0], padded_columns(k, fmt, rot_size)
    h = None if residual is None else torch.empty(rows, k, dtype=x.dtype, device=dev)
    if fmt == "int8":
        q = empty_int8(rows, kp, dev, k, rot_size, lead)
        codes, ldq, scales, row, sums = q.codes, (kp + 15) & ~15, None, q.scales, q.sums
    else:
        q = empty_fp4(rows, kp, fmt, dev, k, rot_size, lead)
        codes, ldq, scales, row, sums = q.packed, kp // 2, q.scales, q.row_scale, None
    if rows:
        call("ic_rmsnorm_quantize", dev, x2.data_ptr(), nat.ptr(r2), _DT[x.dtype], rows, k, pitch(x2),
             0 if r2 is None else pitch(r2), w.data_ptr(), _DT[w.dtype], float(eps), _FORMATS[fmt], rot_size, kp, nat.ptr(h), k,
             codes.data_ptr(), ldq, nat.ptr(scales), nat.ptr(row), nat.ptr(sums))
    if not x.is_cuda:
        if fmt == "int8":
            q.codes, q.scales, q.sums = q.codes.to(x.device), q.scales.to(x.device), q.sums.to(x.device)
        else:
            q = q.to(x.device)
    return q, None if h is None else back(h if x.dim() == 2 else h.view(x.shape), x)
