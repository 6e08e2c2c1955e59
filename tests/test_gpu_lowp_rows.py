"""GPU tests of the row kernels where a CTA takes more than one group of rows, of what lies
beyond the matrix, and of roundings one by one."""

import numpy as np
import pytest
import torch

from tests import lowp_plain as P

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    import int_crush_converter_b200 as B


def rows(seed, m, k, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(m, k, device="cuda", generator=g) * torch.exp(torch.randn(k, device="cuda", generator=g))).to(dtype)


def parts(q):
    """Every tensor of quantized rows, one row of each per row."""
    if isinstance(q, B.Int8Rows):
        return [q.codes, q.scales, q.sums]
    return [q.packed, q.block_scales()] + ([] if q.row_scale is None else [q.row_scale])


def same_as_in_batches(f, m, step):
    """f(first, last) -> tensors of these rows: all rows at once give what `step` rows at a time give."""
    whole = f(0, m)
    for i in range(0, m, step):
        j = min(i + step, m)
        for a, b in zip(whole, f(i, j)):
            assert torch.equal(a[i:j], b), (i, j)


def beyond(q):
    """The scale bytes beyond the rows and blocks of the matrix."""
    t = q.scales.permute(0, 3, 2, 1, 4).reshape(q.scales.shape[0] * 128, -1).cpu().numpy().copy()
    t[:q.rows, :q.columns // P.BLOCK[q.fmt]] = 0
    return t


# More groups of rows than the device holds CTAs, the last one ragged: up to 8192 columns a pair of chunks
# per thread, up to 32768 two.  60 rows fill at most 128 groups, fewer than the 148 SMs.
LARGE = [(20001, 96, 32), (5001, 4096, 256), (3001, 5000, 0), (2001, 8192, 64), (1001, 9000, 128), (801, 16384, 256),
         (601, 32768, 256), (601, 32768, 0)]


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("m,k,rot", LARGE)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantize_many_groups(fmt, m, k, rot, dtype):
    x = rows(m, m, k, dtype)
    same_as_in_batches(lambda i, j: parts(B.quantize_fp4(x[i:j], fmt, rot_size=rot)), m, 60 if k > 512 else 1000)


@pytest.mark.parametrize("fmt", ["int8", "mxfp4", "nvfp4"])
@pytest.mark.parametrize("m,k,rot", LARGE)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rmsnorm_many_groups(fmt, m, k, rot, dtype):
    x, r = rows(m, m, k, dtype), rows(m + 1, m, k, dtype)
    w = 1 + 0.1 * rows(3, 1, k)[0].clamp(-3, 3)

    def f(i, j):
        q, h = B.rmsnorm_quantize(x[i:j], w, residual=r[i:j], fmt=fmt, rot_size=rot)
        return parts(q) + [h]
    same_as_in_batches(f, m, 60 if k > 512 else 1000)


@pytest.mark.parametrize("m,k,rot", [(5, 16384, 256), (3, 32768, 256), (4, 10000, 256)])
@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_wide_rotated_rows(fmt, m, k, rot):
    """Two pairs of chunks per thread under a rotation of 256: the rotation's own fp32 output, quantized."""
    x = rows(k, m, k)
    q, p = B.quantize_fp4(x, fmt, rot_size=rot), B.quantize_fp4(B.rotate_weights(x, rot), fmt)
    assert all(torch.equal(a, b) for a, b in zip(parts(q), parts(p)))


@pytest.mark.parametrize("rot", [0, 16, 32, 64, 128, 256, 512])
def test_rmsnorm_int8_rounds_each_step(rot):
    """The norm's products, the scaled value and the addition of 1/2 are rounded one by one.  Of 13 million
    codes a few dozen lie where a product merged with the addition would choose the other integer."""
    x, w = rows(rot + 1, 3000, 4480, torch.bfloat16), 1 + 0.3 * rows(2, 1, 4480)[0].clamp(-3, 3)
    q, _ = B.rmsnorm_quantize(x, w, eps=1e-5, rot_size=rot)
    h = x.float()
    rstd = (1.0 / torch.sqrt((h.double() ** 2).mean(1, keepdim=True) + float(np.float32(1e-5)))).float()
    z = h * rstd * w
    if rot:
        z = B.rotate_weights(z, rot)
    s = (z.abs().amax(1, keepdim=True) * float(np.float32(1 / 127))).clamp(min=1e-30)
    assert torch.equal(q.scales, s)
    y = z * (1.0 / s)
    want = torch.where(y >= 0, torch.floor(y + 0.5), torch.ceil(y - 0.5)).clamp(-128, 127).to(torch.int8)
    assert torch.equal(q.codes, want)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("k", [32, 160, 1000, 4096 + 32])
def test_scale_bytes_beyond_the_matrix(fmt, k):
    """They are zero, also next to a row that is not finite and with eps = 0."""
    x = rows(k, 130, k)
    w = torch.ones(k, device="cuda")
    x[3, 1], x[129, k - 1] = float("nan"), float("inf")
    for q in (B.quantize_fp4(x, fmt), B.rmsnorm_quantize(x, w, fmt=fmt)[0], B.rmsnorm_quantize(x, w, eps=0.0, fmt=fmt)[0],
              B.rmsnorm_quantize(x, w, residual=x, eps=0.0, fmt=fmt)[0]):
        assert not beyond(q).any()
        v = P.values(q)
        assert np.isfinite(np.delete(v, [3, 129], 0)).all() and np.isnan(v[[3, 129]]).any(1).all()


def test_given_row_scales_far_from_one():
    """Given scales of any size.  u = 2^-24; above 2^120 the reciprocal 1/(6g) is subnormal, at worst 2^-150 of
    1/(6 * 2^128) > 2^-131 off, i.e. 2^-19 relative; 1/(scale * g), of at least 1/2^128, at worst 2^-22."""
    for e in (-117, -100, 0, 100, 120, 123, 126, 127):
        g = float(np.ldexp(1.0, e))
        x = rows(e + 200, 50, 96) * (0.02 if e < 120 else 0.0002)
        x = x.clamp(-1, 1) * 300 * g if e < 120 else x.clamp(-1, 1) * 3e38  # within 448 * 6 g and fp32
        x[:, 32:48] = 0
        q = B.quantize_fp4(x, "nvfp4", row_scale=g)
        z = x.double().cpu().numpy()
        P.check_fp4(q, z, np.abs(z) * (2.0 ** -18 if e >= 120 else 0), given=True)
        assert not q.packed[:, 16:24].any() and not q.block_scales()[:, 2].any()
    for g in (2.0 ** -149, 1e-40, 1e-37, 2.0 ** -118):
        x = torch.zeros(2, 64, device="cuda")
        x[:, 3], x[:, 5] = 1.0, -1.0  # far above 448 * 6 g: they saturate; zeros stay zero
        q = B.quantize_fp4(x, "nvfp4", row_scale=g)
        v, s, h = P.decode(q)
        assert np.all(s[:, 0] == 448) and not s[:, 1:].any() and np.all(h == float(np.float32(g)))
        assert np.all(v[:, [3, 5]] == [6, -6]) and np.count_nonzero(v) == 4


def test_codes_and_outputs_beyond_32_bits():
    """Packed codes, int8 codes, values and products that really lie past 2^32 bytes: the last rows against the
    same rows alone."""
    last = rows(1, 5, 16384, torch.bfloat16)
    for make, m in ((lambda t: B.quantize_fp4(t, "nvfp4", rot_size=64), 530000),
                    (lambda t: B.rmsnorm_quantize(t, torch.ones(16384, device="cuda"))[0], 270000)):
        x = torch.zeros(m, 16384, dtype=torch.bfloat16, device="cuda")
        x[-5:] = last
        q, p = make(x), make(last)
        del x
        codes, few = (q.codes, p.codes) if isinstance(q, B.Int8Rows) else (q.packed, p.packed)
        assert codes.numel() > 2 ** 32 and torch.equal(codes[-5:], few) and not codes[:-5].any()
        if isinstance(q, B.Int8Rows):
            v = torch.randint(-5, 6, (40, 16384), device="cuda", dtype=torch.int8)
            one = torch.ones(40, device="cuda").half()
            y = B.matmul_int8(q, v, one, out_dtype=torch.float32)
            assert torch.equal(y[-5:], B.matmul_int8(p, v, one, out_dtype=torch.float32)) and not y[:-5].any()
            v = B.dequantize_int8(q, torch.float16)
            assert torch.equal(v[-5:], B.dequantize_int8(p, torch.float16))
        else:
            assert all(torch.equal(a[-5:], b) for a, b in zip(parts(q), parts(p)))
            v = B.dequantize_fp4(q, torch.float16)
            assert torch.equal(v[-5:], B.dequantize_fp4(p, torch.float16))
        assert not v[:-5].any()
        del q, codes, v
    # y of 5.6 GB; powers of two, so that the sums are exact whatever their order
    a = torch.exp2(torch.randint(-1, 3, (70000, 64), device="cuda").float())
    b = torch.exp2(torch.randint(-1, 3, (40000, 64), device="cuda").float())
    y = B.matmul_fp4(B.quantize_fp4(a), B.quantize_fp4(b))
    want = (a[-300:].double() @ b.double().T).to(torch.bfloat16)
    assert y.numel() * 2 > 2 ** 32 and torch.equal(y[-300:], want)
