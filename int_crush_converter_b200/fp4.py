"""Microscaled 4-bit floating point on the GPU: quantization, values, product.

Two formats of E2M1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives):

* ``"mxfp4"``: one power-of-two scale per 32 columns;
* ``"nvfp4"``: one E4M3 scale per 16 columns and one fp32 scale per row.

Weights and activations are quantized the same way, after the same group
Hadamard rotation that the INT4 path uses (``rot_size``), and multiplied on the
block-scaled tensor cores.  Nothing here has a gradient.
"""

from __future__ import annotations

import dataclasses

import torch

from . import _native as nat
from ._dev import back, call, device_of
from .rotation import _DT, _is_power_of_two, _rotate_rows

FORMATS = {"mxfp4": nat.IC_MXFP4, "nvfp4": nat.IC_NVFP4}
BLOCK = {"mxfp4": 32, "nvfp4": 16}


def _ktiles(fmt: str, kp: int) -> int:
    return -(-kp // (4 * BLOCK[fmt]))


@dataclasses.dataclass
class FP4Tensor:
    """Rows in a 4-bit floating-point format.

    ``packed``: uint8 [rows, columns/2], low nibble = even column; columns are the
    input's, padded with zeros to a multiple of 32 (and of the rotation size).
    ``scales``: the block-scale bytes, uint8 [ceil(rows/128), ceil(blocks/4), 32, 4, 4]:
    row r, block b at [r//128, b//4, r%32, r%128//32, b%4] (the order in which the
    product reads them; :meth:`block_scales` gives them row by row).  The bytes of
    rows and blocks beyond the matrix are zero.
    ``row_scale``: fp32 [rows] (nvfp4), else None.
    ``lead``: the leading dimensions of the tensor that was quantized (default [rows]).
    """

    packed: torch.Tensor
    scales: torch.Tensor
    row_scale: torch.Tensor | None
    fmt: str = "mxfp4"
    in_features: int | None = None
    rot_size: int = 0
    lead: tuple | None = None

    @property
    def rows(self) -> int:
        return self.packed.shape[0]

    @property
    def columns(self) -> int:
        return self.packed.shape[1] * 2

    @property
    def device(self) -> torch.device:
        return self.packed.device

    def to(self, device) -> "FP4Tensor":
        move = lambda t: None if t is None else t.to(device)  # noqa: E731
        return dataclasses.replace(self, packed=move(self.packed), scales=move(self.scales), row_scale=move(self.row_scale))

    @classmethod
    def from_block_scales(cls, packed: torch.Tensor, block_scales: torch.Tensor, row_scale: torch.Tensor | None = None,
                          fmt: str = "mxfp4", **kw) -> "FP4Tensor":
        """From block-scale bytes kept row by row, uint8 [rows, blocks] (E8M0 or E4M3), as :meth:`block_scales` gives them."""
        if fmt not in FORMATS:
            raise ValueError(f"fmt must be one of {sorted(FORMATS)}, got {fmt!r}")
        rows, blocks = packed.shape[0], 2 * packed.shape[1] // BLOCK[fmt]
        if tuple(block_scales.shape) != (rows, blocks) or block_scales.element_size() != 1:
            raise ValueError(f"block_scales must be bytes [{rows}, {blocks}], got {block_scales.dtype} {tuple(block_scales.shape)}")
        a, b = -(-rows // 128), -(-blocks // 4)
        t = torch.zeros(a * 128, b * 4, dtype=torch.uint8, device=packed.device)
        t[:rows, :blocks] = block_scales.contiguous().view(torch.uint8)
        q = cls(packed.contiguous(), t.view(a, 4, 32, b, 4).permute(0, 3, 2, 1, 4).contiguous(), row_scale, fmt, **kw)
        q.check("from_block_scales")
        return q

    def block_scales(self) -> torch.Tensor:
        """The block-scale bytes as uint8 [rows, blocks]."""
        a, b = -(-self.rows // 128), _ktiles(self.fmt, self.columns)
        t = self.scales.reshape(a, b, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(a * 128, b * 4)
        return t[:self.rows, :self.columns // BLOCK[self.fmt]].contiguous()

    def check(self, what: str) -> None:
        """ValueError unless the parts have the types and sizes the kernels read."""
        p, s, g = self.packed, self.scales, self.row_scale
        block = BLOCK.get(self.fmt)
        if block is None:
            raise ValueError(f"{what}: fmt must be one of {sorted(FORMATS)}, got {self.fmt!r}")
        if p.dim() != 2 or p.dtype is not torch.uint8 or s.dtype is not torch.uint8:
            raise ValueError(f"{what}: packed must be uint8 [rows, columns/2] and scales uint8")
        rows, half = p.shape
        if half & 15:
            raise ValueError(f"{what}: the number of columns must be a multiple of 32, got {2 * half}")
        need = -(-rows // 128) * -(-half // (2 * block)) * 512
        if s.numel() != need:
            raise ValueError(f"{what}: {rows} rows of {2 * half} {self.fmt} columns have {need} scale bytes, got {s.numel()}")
        device = p.device
        if s.device != device:
            raise ValueError(f"{what}: packed and scales must be on one device")
        if (g is None) != (block == 32):
            raise ValueError(f"{what}: nvfp4 has row scales and mxfp4 none")
        if g is not None and (g.dtype is not torch.float32 or g.numel() != rows or g.device != device):
            raise ValueError(f"{what}: row_scale must be fp32 [rows] on the codes' device")
        if not p.is_contiguous() or not s.is_contiguous() or (g is not None and not g.is_contiguous()):
            raise ValueError(f"{what}: packed, scales and row_scale must be contiguous")
        if (p.data_ptr() | s.data_ptr()) & 15:
            raise ValueError(f"{what}: packed and scales must be 16-byte aligned")


def empty_fp4(rows: int, columns: int, fmt: str, dev: torch.device, in_features: int | None = None, rot_size: int = 0,
              lead: tuple | None = None) -> FP4Tensor:
    """An FP4Tensor of uninitialised parts."""
    return FP4Tensor(torch.empty(rows, columns // 2, dtype=torch.uint8, device=dev),
                     torch.empty(-(-rows // 128), _ktiles(fmt, columns), 32, 4, 4, dtype=torch.uint8, device=dev),
                     torch.empty(rows, dtype=torch.float32, device=dev) if fmt == "nvfp4" else None, fmt, in_features,
                     rot_size, lead)


def padded_columns(k: int, fmt: str, rot_size: int) -> int:
    """Columns held: ``k`` up to whole rotation groups and, for the 4-bit formats, whole runs of 32."""
    unit = max(rot_size, 1 if fmt == "int8" else 32)
    return -(-k // unit) * unit


def as_rows(x: torch.Tensor, dev: torch.device) -> torch.Tensor:
    """[..., K] -> 2-D rows on ``dev`` with unit column stride (a view where possible)."""
    if not x.is_cuda:
        x = x.to(dev)
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1])
    if not x.is_contiguous() and x.numel():
        pitch_, step = x.stride()
        if step != 1 or pitch_ < x.shape[1]:
            x = x.contiguous()
    return x


def pitch(x2: torch.Tensor) -> int:
    return max(x2.stride(0), x2.shape[1])


def quantize_fp4(x: torch.Tensor, fmt: str = "mxfp4", rot_size: int = 0,
                 row_scale: torch.Tensor | float | None = None) -> FP4Tensor:
    """Quantize [..., K] weights or activations (fp32/fp16/bf16) to ``fmt``.

    ``rot_size``: 0, or a power of two: the group Hadamard of ``rotate_weights``
    first, in fp32 (fused for 16..512).  ``row_scale`` (nvfp4): the second-level
    scale, one number for all rows or fp32 [rows]; by default each row's
    max|x|/2688, so that a row does not depend on its neighbours (a given one below
    2^-118 counts as 2^-118 where codes are formed).  A value that is
    not finite marks its mxfp4 block or its nvfp4 row as NaN.
    """
    if row_scale is None and fmt in FORMATS:
        parts = nat.binding().fp4_quantize(x, FORMATS[fmt], rot_size)
        if parts is not None:
            return FP4Tensor(*parts, fmt, x.shape[-1], rot_size, x.shape[:-1])
    if fmt not in FORMATS:
        raise ValueError(f"fmt must be one of {sorted(FORMATS)}, got {fmt!r}")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("quantize_fp4 needs at least one column")
    if rot_size and not _is_power_of_two(rot_size):
        raise ValueError(f"rot_size must be 0 or a power of 2, got {rot_size}")
    if x.dtype not in _DT:
        raise ValueError(f"x must be float32, float16 or bfloat16, got {x.dtype}")
    if row_scale is not None and fmt != "nvfp4":
        raise ValueError("row_scale is for nvfp4")
    dev = device_of(x)
    lead, k = x.shape[:-1], x.shape[-1]
    x2 = as_rows(x, dev)
    rows, rot = x2.shape[0], rot_size
    stride = 0
    if row_scale is not None:
        row_scale = torch.as_tensor(row_scale, dtype=torch.float32, device=dev).reshape(-1).contiguous()
        if row_scale.numel() not in (1, rows):
            raise ValueError(f"row_scale must have 1 or {rows} values, got {row_scale.numel()}")
        stride = int(row_scale.numel() == rows and rows > 1)
    if rot and not 16 <= rot <= 512:
        with torch.cuda.device(dev):
            x2 = _rotate_rows(x2, rot, dev) if rows else x2.new_empty(0, padded_columns(k, "int8", rot))
        rot = 0
    columns = padded_columns(x2.shape[1], fmt, rot)
    out = empty_fp4(rows, columns, fmt, dev, k, rot_size, lead)
    if rows:
        call("ic_fp4_quantize", dev, x2.data_ptr(), _DT[x2.dtype], rows, x2.shape[1], pitch(x2), FORMATS[fmt], rot, columns,
             nat.ptr(row_scale), stride, out.packed.data_ptr(), out.scales.data_ptr(), nat.ptr(out.row_scale))
    return out if x.is_cuda else out.to(x.device)


def dequantize_fp4(q: FP4Tensor, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values of ``q``, [lead..., columns] (padding included), in fp32/fp16/bf16."""
    out = nat.binding().fp4_dequantize(q.packed, q.scales, q.row_scale, FORMATS.get(q.fmt, 0), dtype)
    if out is not None:
        return out if q.lead is None or len(q.lead) == 1 else out.reshape(*q.lead, out.shape[1])
    q.check("dequantize_fp4")
    if dtype not in _DT:
        raise ValueError(f"dtype must be float32, float16 or bfloat16, got {dtype}")
    dev = device_of(q.packed)
    d = q if q.packed.is_cuda else q.to(dev)
    rows, columns = d.rows, d.columns
    out = torch.empty(rows, columns, dtype=dtype, device=dev)
    if rows and columns:
        call("ic_fp4_dequantize", dev, d.packed.data_ptr(), d.scales.data_ptr(), nat.ptr(d.row_scale), FORMATS[q.fmt], rows,
             columns, _DT[dtype], out.data_ptr(), columns)
    if q.lead is not None and len(q.lead) != 1:
        out = out.reshape(*q.lead, columns)
    return back(out, q.packed)


def check_bias(bias: torch.Tensor | None, n: int, dev: torch.device) -> torch.Tensor | None:
    if bias is None:
        return None
    if bias.numel() != n or bias.dtype not in _DT:
        raise ValueError(f"bias must have {n} values in float32, float16 or bfloat16")
    if bias.dim() == 1 and bias.device == dev and bias.is_contiguous():
        return bias
    return bias.to(dev).reshape(-1).contiguous()


def matmul_fp4(a: FP4Tensor, b: FP4Tensor, bias: torch.Tensor | None = None,
               out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``a @ b.T + bias``: activations [lead..., K] times weights [N, K], both in one format.

    Products of codes and scales are exact, their sums and the bias are held in
    fp32 and rounded once to ``out_dtype`` (fp32/fp16/bf16).  ``b``'s rows are the
    output's columns.  Elements that a wait on the device left without their sum
    (2 s without progress) are NaN.
    """
    if a.fmt == b.fmt and a.rot_size == b.rot_size and (a.in_features == b.in_features or a.in_features is None or b.in_features is None):
        y = nat.binding().fp4_matmul(a.packed, a.scales, a.row_scale, b.packed, b.scales, b.row_scale, FORMATS.get(a.fmt, 0), bias,
                                     out_dtype)
        if y is not None:
            return y if a.lead is None or len(a.lead) == 1 else y.reshape(*a.lead, y.shape[1])
    a.check("matmul_fp4")
    b.check("matmul_fp4")
    pa, pb = a.packed, b.packed
    m, half = pa.shape
    n, half_b = pb.shape
    if a.fmt != b.fmt or half != half_b:
        raise ValueError(f"matmul_fp4: operands differ: {a.fmt} with {2 * half} columns, {b.fmt} with {2 * half_b}")
    if a.rot_size != b.rot_size:
        raise ValueError(f"matmul_fp4: operands are rotated by {a.rot_size} and {b.rot_size}")
    if a.in_features != b.in_features and a.in_features is not None and b.in_features is not None:
        raise ValueError(f"matmul_fp4: operands have {a.in_features} and {b.in_features} input features")
    device = pa.device
    if device != pb.device:
        raise ValueError("matmul_fp4: operands are on different devices")
    if out_dtype not in _DT:
        raise ValueError(f"out_dtype must be float32, float16 or bfloat16, got {out_dtype}")
    dev = device_of(pa)
    bias_d = check_bias(bias, n, dev)
    da, db = (a, b) if pa.is_cuda else (a.to(dev), b.to(dev))
    y = torch.empty(m, n, dtype=out_dtype, device=dev)
    if m and n:
        if half == 0:
            y.zero_() if bias_d is None else y.copy_(bias_d.float().expand(m, n))
        else:
            call("ic_fp4_matmul", dev, da.packed.data_ptr(), da.scales.data_ptr(), nat.ptr(da.row_scale),
                 db.packed.data_ptr(), db.scales.data_ptr(), nat.ptr(db.row_scale), FORMATS[a.fmt], m, n, 2 * half,
                 nat.ptr(bias_d), 0 if bias_d is None else _DT[bias_d.dtype], _DT[out_dtype], y.data_ptr(), n)
    if a.lead is not None and len(a.lead) != 1:
        y = y.reshape(*a.lead, n)
    return back(y, pa)
