"""What the low-precision operators refuse, without a GPU: bad arguments raise before one is looked for."""

import pytest
import torch

import int_crush_converter_b200 as B
from int_crush_converter_b200 import _native as nat
from int_crush_converter_b200.fp4 import empty_fp4

CPU = torch.device("cpu")


def fp4(rows=4, columns=64, fmt="mxfp4", **kw):
    return empty_fp4(rows, columns, fmt, CPU, **kw)


def rows8(rows=4, columns=48):
    return B.Int8Rows(torch.zeros(rows, columns, dtype=torch.int8), torch.ones(rows, 1))


@pytest.mark.parametrize("kw, match", [
    (dict(fmt="int4"), "fmt"), (dict(rot_size=48), "power of 2"), (dict(row_scale=1.0), "row_scale"),
])
def test_quantize_fp4_arguments(kw, match):
    with pytest.raises(ValueError, match=match):
        B.quantize_fp4(torch.zeros(2, 64), **kw)


@pytest.mark.parametrize("x", [torch.zeros(3, 0), torch.zeros(3, 32, dtype=torch.float64), torch.zeros(3, 32, dtype=torch.int32)])
def test_quantize_fp4_inputs(x):
    with pytest.raises(ValueError):
        B.quantize_fp4(x)


@pytest.mark.parametrize("kw, match", [
    (dict(fmt="fp8"), "fmt"), (dict(rot_size=8), "rot_size"), (dict(rot_size=1024), "rot_size"), (dict(rot_size=96), "rot_size"),
    (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(residual=torch.zeros(2, 32)), "residual"),
    (dict(residual=torch.zeros(2, 64).half()), "residual"), (dict(weight=torch.ones(63)), "weight"),
    (dict(weight=torch.ones(64).double()), "weight"),
])
def test_rmsnorm_arguments(kw, match):
    args = dict(x=torch.zeros(2, 64), weight=torch.ones(64)) | kw
    with pytest.raises(ValueError, match=match):
        B.rmsnorm_quantize(**args)


@pytest.mark.parametrize("a, b, match", [
    (fp4(), fp4(fmt="nvfp4"), "differ"), (fp4(), fp4(columns=96), "differ"), (fp4(), fp4(rot_size=64), "rotated"),
    (fp4(in_features=60), fp4(in_features=62), "input features"),
    (B.FP4Tensor(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(256, dtype=torch.uint8), None), fp4(), "scale bytes"),
    (B.FP4Tensor(torch.zeros(4, 24, dtype=torch.uint8), torch.zeros(512, dtype=torch.uint8), None), fp4(), "multiple of 32"),
    (B.FP4Tensor(torch.zeros(4, 32, dtype=torch.int8), torch.zeros(512, dtype=torch.uint8), None), fp4(), "uint8"),
    (B.FP4Tensor(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(512, dtype=torch.uint8), torch.ones(4)), fp4(), "row scales"),
    (B.FP4Tensor(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(512, dtype=torch.uint8), torch.ones(3), "nvfp4"), fp4(fmt="nvfp4"), "row_scale"),
    (B.FP4Tensor(torch.zeros(8, 32, dtype=torch.uint8)[::2], torch.zeros(512, dtype=torch.uint8), None), fp4(), "contiguous"),
    (B.FP4Tensor(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(512, dtype=torch.uint8), None, "e2m1"), fp4(), "fmt"),
])
def test_matmul_fp4_operands(a, b, match):
    with pytest.raises(ValueError, match=match):
        B.matmul_fp4(a, b)


def test_matmul_fp4_alignment_and_types():
    base = torch.zeros(4 * 32 + 8, dtype=torch.uint8)
    off = B.FP4Tensor(base[8:].view(4, 32), torch.zeros(512, dtype=torch.uint8), None)
    if off.packed.data_ptr() % 16:
        with pytest.raises(ValueError, match="aligned"):
            B.matmul_fp4(off, fp4())
    with pytest.raises(ValueError, match="out_dtype"):
        B.matmul_fp4(fp4(), fp4(), out_dtype=torch.float64)
    with pytest.raises(ValueError, match="dtype"):
        B.dequantize_fp4(fp4(), torch.float64)


@pytest.mark.parametrize("kw, match", [
    (dict(w_codes=torch.zeros(3, 40, dtype=torch.int8)), "columns"), (dict(w_codes=torch.zeros(3, 48)), "int8"),
    (dict(w_scales=torch.ones(3, 1)), "float16"), (dict(w_scales=torch.ones(2, 1).half()), "w_scales"),
    (dict(w_zero_points=torch.zeros(3, 1)), "w_zero_points"), (dict(w_zero_points=torch.zeros(3, 2, dtype=torch.int8)), "w_zero_points"),
    (dict(out_dtype=torch.int32), "out_dtype"),
])
def test_matmul_int8_arguments(kw, match):
    args = dict(a=rows8(), w_codes=torch.zeros(3, 48, dtype=torch.int8), w_scales=torch.ones(3, 1).half()) | kw
    with pytest.raises(ValueError, match=match):
        B.matmul_int8(**args)


def test_matmul_int8_sums_must_fit():
    w = torch.zeros(1, 131072, dtype=torch.int8)
    with pytest.raises(ValueError, match="int32"):
        B.matmul_int8(rows8(1, 131072), w, torch.ones(1).half())
    w = w[:, :65536]
    with pytest.raises(ValueError, match="int32"):
        B.matmul_int8(rows8(1, 65536), w, torch.ones(1).half(), torch.zeros(1, dtype=torch.int8))


def test_int8_rows_types():
    for bad in (B.Int8Rows(torch.zeros(2, 4), torch.ones(2, 1)), B.Int8Rows(torch.zeros(2, 4, dtype=torch.int8), torch.ones(2, 1).half()),
                B.Int8Rows(torch.zeros(2, 4, dtype=torch.int8), torch.ones(2, 1), torch.zeros(2))):
        with pytest.raises(ValueError):
            B.dequantize_int8(bad)


def test_c_entry_points_refuse_before_any_launch():
    lib, p = nat.load(), 4096  # an aligned address that is never read
    inv = nat.IC_ERR_INVALID
    q = lambda **k: lib.ic_fp4_quantize(*(dict(x=p, dtype=0, M=2, K=64, ldx=64, fmt=1, rot=0, kp=64, rs=None, st=0, o=p,  # noqa: E731
                                               s=p, g=None, stream=None) | k).values())
    for bad in (dict(fmt=0), dict(fmt=3), dict(dtype=7), dict(M=-1), dict(K=0), dict(ldx=63), dict(rot=8), dict(rot=1024),
                dict(kp=96), dict(rs=p), dict(fmt=2, g=p, rs=p, st=2), dict(fmt=2), dict(x=None), dict(o=p + 8), dict(s=p + 4)):
        assert q(**bad) == inv, bad
    mm = lambda **k: lib.ic_fp4_matmul(*(dict(a=p, asc=p, ag=None, b=p, bsc=p, bg=None, fmt=1, m=2, n=2, k=64, bias=None, bt=0,  # noqa: E731
                                              ot=0, y=p, ldy=2, stream=None) | k).values())
    for bad in (dict(fmt=0), dict(k=0), dict(k=48), dict(m=-1), dict(ldy=1), dict(ot=3), dict(bias=p, bt=5), dict(a=None), dict(y=None),
                dict(fmt=2), dict(a=p + 8), dict(bsc=p + 1)):
        assert mm(**bad) == inv, bad
    assert mm(m=1 << 31) == nat.IC_ERR_UNSUPPORTED
    im = lambda **k: lib.ic_int8_matmul(*(dict(a=p, lda=64, s=p, sums=None, w=p, ldw=64, ws=p, zp=None, m=2, n=2, k=64, bias=None,  # noqa: E731
                                               bt=0, ot=0, y=p, ldy=2, stream=None) | k).values())
    for bad in (dict(lda=63), dict(lda=72), dict(ldw=8), dict(a=p + 4), dict(zp=p), dict(k=0), dict(s=None), dict(ldy=1)):
        assert im(**bad) == inv, bad
    assert im(k=131072, lda=131072, ldw=131072) == nat.IC_ERR_UNSUPPORTED
    assert im(k=65536, lda=65536, ldw=65536, zp=p, sums=p) == nat.IC_ERR_UNSUPPORTED
    rn = lambda **k: lib.ic_rmsnorm_quantize(*(dict(x=p, r=None, dtype=0, M=2, K=64, ldx=64, ldr=0, w=p, wt=0, eps=1e-6, fmt=0, rot=0,  # noqa: E731
                                                    kp=64, ro=None, ldo=64, q=p, ldq=64, s=None, g=p, sums=None, stream=None) | k).values())
    for bad in (dict(fmt=5), dict(wt=4), dict(eps=-1.0), dict(w=None), dict(r=p, ldr=64), dict(r=p, ldr=64, ro=p), dict(ldq=48),
                dict(ldq=72), dict(g=None), dict(rot=2), dict(kp=65), dict(fmt=1, ldq=32, s=None)):
        assert rn(**bad) == inv, bad


def test_block_scales_of_another_shape():
    p = torch.zeros(4, 32, dtype=torch.uint8)
    for bad, fmt in ((torch.zeros(4, 3, dtype=torch.uint8), "mxfp4"), (torch.zeros(4, 2, dtype=torch.int16), "mxfp4"),
                     (torch.zeros(4, 2, dtype=torch.uint8), "nvfp4"), (torch.zeros(4, 2, dtype=torch.uint8), "fp4")):
        with pytest.raises(ValueError):
            B.FP4Tensor.from_block_scales(p, bad, None, fmt)
    q = B.FP4Tensor.from_block_scales(p, torch.arange(8, dtype=torch.uint8).view(4, 2))
    assert torch.equal(q.block_scales(), torch.arange(8, dtype=torch.uint8).view(4, 2)) and int(q.scales.sum()) == 28
