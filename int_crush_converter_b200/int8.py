"""INT8 rows (one fp32 scale per row) and their product with INT8 weights on the GPU.

The weights are the codes, fp16 scales and zero-points that ``scales`` and
``gptq`` write (value = (code - zero_point) * scale); the rows come from
``rmsnorm_quantize``.  Nothing here has a gradient.
"""

from __future__ import annotations

import dataclasses

import torch

from . import _native as nat
from ._dev import back, call, device_of
from .fp4 import check_bias
from .rotation import _DT

MAX_K = 131071      # int32 sums of products
MAX_K_ASYM = 65535  # with zero-points


@dataclasses.dataclass
class Int8Rows:
    """``codes``: int8 [rows, columns] (columns contiguous; a row pitch of a multiple
    of 16 bytes is read in place); ``scales``: fp32 [rows, 1]; ``sums``: int32 [rows],
    the sum of each row's codes (asked for by asymmetric weights), or None."""

    codes: torch.Tensor
    scales: torch.Tensor
    sums: torch.Tensor | None = None
    in_features: int | None = None
    rot_size: int = 0
    lead: tuple | None = None

    @property
    def rows(self) -> int:
        return self.codes.shape[0]

    @property
    def columns(self) -> int:
        return self.codes.shape[1]

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def check(self, what: str) -> None:
        c, s, t = self.codes, self.scales, self.sums
        if c.dim() != 2 or c.dtype is not torch.int8:
            raise ValueError(f"{what}: codes must be int8 [rows, columns]")
        rows, device = c.shape[0], c.device
        if s.dtype is not torch.float32 or s.numel() != rows:
            raise ValueError(f"{what}: scales must be fp32 [rows, 1]")
        if t is not None and (t.dtype is not torch.int32 or t.numel() != rows):
            raise ValueError(f"{what}: sums must be int32 [rows]")
        if s.device != device or (t is not None and t.device != device):
            raise ValueError(f"{what}: codes, scales and sums must be on one device")


def empty_int8(rows: int, columns: int, dev: torch.device, in_features: int | None = None, rot_size: int = 0,
               lead: tuple | None = None) -> Int8Rows:
    """Int8Rows of uninitialised parts, rows at a pitch of a multiple of 16 bytes."""
    buf = torch.empty(rows, (columns + 15) & ~15, dtype=torch.int8, device=dev)
    return Int8Rows(buf[:, :columns] if columns & 15 else buf, torch.empty(rows, 1, dtype=torch.float32, device=dev),
                    torch.empty(rows, dtype=torch.int32, device=dev), in_features, rot_size, lead)


def flat(t: torch.Tensor, dev: torch.device) -> torch.Tensor:
    """One value per row, as the kernels read them."""
    if t.is_contiguous() and t.is_cuda:
        return t
    return t.to(dev).reshape(-1).contiguous()


def pitched(codes: torch.Tensor, dev: torch.device) -> tuple[torch.Tensor, int]:
    """(codes on ``dev`` as the product reads them, row pitch): 16-byte aligned rows,
    copied when they are not."""
    c = codes if codes.is_cuda else codes.to(dev)
    rows, k = c.shape
    if (k == 1 or c.stride(1) == 1) and c.data_ptr() % 16 == 0:
        if rows == 1:
            return c, (k + 15) & ~15
        if c.stride(0) % 16 == 0 and c.stride(0) >= k:
            return c, c.stride(0)
    buf = torch.zeros(rows, (k + 15) & ~15, dtype=torch.int8, device=dev)
    buf[:, :k] = c
    return buf, buf.shape[1]


def dequantize_int8(q: Int8Rows, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values of ``q``, [lead..., columns], in fp32/fp16/bf16."""
    out = nat.binding().int8_dequantize(q.codes, q.scales, dtype)
    if out is not None:
        return out if q.lead is None or len(q.lead) == 1 else out.reshape(*q.lead, out.shape[1])
    q.check("dequantize_int8")
    if dtype not in _DT:
        raise ValueError(f"dtype must be float32, float16 or bfloat16, got {dtype}")
    dev = device_of(q.codes)
    rows, columns = q.codes.shape
    out = torch.empty(rows, columns, dtype=dtype, device=dev)
    if rows and columns:
        codes = q.codes if q.codes.is_cuda else q.codes.to(dev)
        pitch, step = codes.stride()
        if step != 1 or pitch < columns:
            codes = codes.contiguous()
            pitch = columns
        call("ic_int8_dequantize", dev, codes.data_ptr(), pitch, flat(q.scales, dev).data_ptr(), rows, columns, _DT[dtype],
             out.data_ptr(), columns)
    if q.lead is not None and len(q.lead) != 1:
        out = out.reshape(*q.lead, columns)
    return back(out, q.codes)


def matmul_int8(a: Int8Rows, w_codes: torch.Tensor, w_scales: torch.Tensor,
                w_zero_points: torch.Tensor | None = None, bias: torch.Tensor | None = None,
                out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``a @ W.T + bias`` with W = (w_codes - w_zero_points) * w_scales.

    ``w_codes``: int8 [N, columns] as the quantizers return them (INT4 codes in
    int8 serve too); ``w_scales``: fp16 [N] or [N, 1]; ``w_zero_points``: int8 or
    None.  Sums are exact in int32 (columns up to 131071, with zero-points 65535),
    the scaling and the bias fp32, rounded once to ``out_dtype``; NaN where a wait
    on the device gave up, as in ``matmul_fp4``.  Weights whose
    rows are not 16-byte aligned are copied on every call: keep them at such a
    pitch.
    """
    y = nat.binding().int8_matmul(a.codes, a.scales, a.sums, w_codes, w_scales, w_zero_points, bias, out_dtype)
    if y is not None:
        return y if a.lead is None or len(a.lead) == 1 else y.reshape(*a.lead, y.shape[1])
    a.check("matmul_int8")
    if w_codes.dim() != 2 or w_codes.dtype != torch.int8:
        raise ValueError("matmul_int8: w_codes must be int8 [out, columns]")
    (m, ka), (n, k) = a.codes.shape, w_codes.shape
    if ka != k:
        raise ValueError(f"matmul_int8: rows have {ka} columns, the weights {k}")
    if k > (MAX_K if w_zero_points is None else MAX_K_ASYM):
        raise ValueError(f"matmul_int8: int32 sums hold {MAX_K} columns, {MAX_K_ASYM} with zero-points; got {k}")
    if w_scales.dtype != torch.float16 or w_scales.numel() != n:
        raise ValueError(f"matmul_int8: w_scales must be float16 with {n} values (one per row)")
    if w_zero_points is not None and (w_zero_points.dtype != torch.int8 or w_zero_points.numel() != n):
        raise ValueError(f"matmul_int8: w_zero_points must be int8 with {n} values (one per row)")
    if out_dtype not in _DT:
        raise ValueError(f"out_dtype must be float32, float16 or bfloat16, got {out_dtype}")
    device = a.codes.device
    if w_codes.device != device or w_scales.device != device or (w_zero_points is not None and w_zero_points.device != device):
        raise ValueError("matmul_int8: operands are on different devices")
    dev = device_of(a.codes)
    bias_d = check_bias(bias, n, dev)
    y = torch.empty(m, n, dtype=out_dtype, device=dev)
    if m and n:
        if k == 0:
            y.zero_() if bias_d is None else y.copy_(bias_d.float().expand(m, n))
        else:
            x, ldx = pitched(a.codes, dev)
            w, ldw = pitched(w_codes, dev)
            zp = sums = None
            if w_zero_points is not None:
                zp, sums = flat(w_zero_points, dev), a.sums
                if sums is None:
                    sums = torch.empty(m, dtype=torch.int32, device=dev)
                    call("ic_int8_row_sums", dev, x.data_ptr(), ldx, m, k, sums.data_ptr())
                else:
                    sums = flat(sums, dev)
            s, ws = flat(a.scales, dev), flat(w_scales, dev)
            call("ic_int8_matmul", dev, x.data_ptr(), ldx, s.data_ptr(), nat.ptr(sums), w.data_ptr(), ldw, ws.data_ptr(),
                 nat.ptr(zp), m, n, k, nat.ptr(bias_d), 0 if bias_d is None else _DT[bias_d.dtype], _DT[out_dtype],
                 y.data_ptr(), n)
    if a.lead is not None and len(a.lead) != 1:
        y = y.reshape(*a.lead, n)
    return back(y, a.codes)
