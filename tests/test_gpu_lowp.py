"""GPU tests of the low-precision operators against plain 64-bit forms.

Tolerances count roundings: u = 2^-24 for an fp32 operation, half a step of the
type for the final rounding of an output (bf16 2^-9 of the power of two below,
i.e. at most 2^-8 relative; fp16 2^-11; fp32 2^-24).
"""

import numpy as np
import pytest
import torch

from tests import lowp_plain as P

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    import int_crush_converter_b200 as B
    from int_crush_converter_b200 import _native as nat

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}  # half the smallest step


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rows(seed, m, k, dtype=torch.float32, std=1.0):
    g = gen(seed)
    x = torch.randn(m, k, device="cuda", generator=g) * std
    x *= torch.exp(torch.randn(k, device="cuda", generator=g))
    return x.to(dtype)


def f64(t):
    return t.detach().double().cpu().numpy()


def rotated(x64, rot, kp):
    """64-bit rotated rows, and how far the fp32 butterflies may be from them: log2(rot)
    additions and one scaling, each off by u of at most sum|x|/sqrt(rot)."""
    z = P.rotate(x64, rot, kp)
    if not rot:
        return z, np.zeros_like(z)
    a = np.zeros_like(z)
    a[:, :x64.shape[1]] = np.abs(x64)
    s = np.repeat(a.reshape(-1, rot).sum(1) / np.sqrt(rot), rot).reshape(z.shape)
    return z, (np.log2(rot) + 2) * U * s


# ------------------------------------------------------------------ quantize_fp4
@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("m,k,rot,dtype", [
    (1, 1, 0, torch.float32), (1, 32, 0, torch.bfloat16), (3, 17, 0, torch.float16), (5, 100, 16, torch.float32),
    (129, 513, 32, torch.bfloat16), (128, 256, 256, torch.float16), (33, 640, 128, torch.float32),
    (300, 4096, 256, torch.bfloat16), (7, 1000, 512, torch.float16), (2, 16384, 64, torch.bfloat16),
    (2, 40000, 256, torch.float32), (1, 33333, 0, torch.float16),
])
def test_quantize_fp4(fmt, m, k, rot, dtype):
    x = rows(m * 31 + k, m, k, dtype, 0.02)
    q = B.quantize_fp4(x, fmt, rot_size=rot)
    kp = -(-k // max(32, rot)) * max(32, rot)
    assert (q.rows, q.columns, q.in_features, q.rot_size) == (m, kp, k, rot)
    z, slack = rotated(f64(x), rot, kp)
    P.check_fp4(q, z, slack)
    # bytes of rows and blocks beyond the matrix are zero
    t = q.scales.permute(0, 3, 2, 1, 4).reshape(q.scales.shape[0] * 128, -1).cpu().numpy()
    t[:m, :kp // P.BLOCK[fmt]] = 0
    assert not t.any()


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("rot", [2, 8, 16, 32, 64, 128, 256, 512, 1024])
def test_quantize_fp4_rotation_is_rotate_weights(fmt, rot):
    """Fused or not, the codes are those of the framework's own rotation's fp32 output."""
    x = rows(rot, 37, 1500, torch.float32)
    q, p = B.quantize_fp4(x, fmt, rot_size=rot), B.quantize_fp4(B.rotate_weights(x, rot), fmt)
    assert torch.equal(q.packed, p.packed) and torch.equal(q.scales, p.scales)
    assert q.row_scale is None or torch.equal(q.row_scale, p.row_scale)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_quantize_fp4_every_tie_and_border(fmt):
    """The grid, its midpoints (ties to the even code) and their neighbours, at scale 1."""
    grid = P.E2M1
    mids = (grid[1:] + grid[:-1]) / 2
    pts = np.concatenate([grid, mids, np.nextafter(mids.astype(np.float32), np.float32(0)), np.nextafter(mids.astype(np.float32), np.float32(9))])
    pts = np.concatenate([pts, -pts]).astype(np.float32)
    n = P.BLOCK[fmt]
    pts = np.concatenate([pts, np.zeros(-len(pts) % (n - 1), np.float32)]).reshape(-1, n - 1)
    x = torch.from_numpy(np.concatenate([np.full((len(pts), 1), 6, np.float32), pts], 1)).cuda()  # 6 makes the scale 1
    q = B.quantize_fp4(x, fmt, row_scale=1.0 if fmt == "nvfp4" else None)
    v, s, _ = P.decode(q)
    assert np.all(s[:, 0] == 1)
    even = grid[[0, 2, 2, 4, 4, 6, 6]]
    want = np.abs(pts.astype(np.float64))
    want = np.array([[even[np.flatnonzero(mids == a)[0]] if (mids == a).any() else grid[np.argmin(np.abs(grid - a))] for a in r] for r in want])
    assert np.array_equal(np.abs(v[:, 1:n]), want)
    assert np.array_equal(np.signbit(v[:, 1:n]) & (want > 0), np.signbit(pts) & (want > 0))


def test_quantize_fp4_range_of_scales():
    """Powers of two over the whole fp32 range, subnormals included, and all-zero blocks."""
    e = np.arange(-149, 128)
    x = np.zeros((len(e), 64), np.float32)
    x[:, 3] = np.ldexp(np.float32(1), e)
    x[:, 5] = -x[:, 3]
    q = B.quantize_fp4(torch.from_numpy(x).cuda(), "mxfp4")
    byte = P.block_scales(q)
    assert np.array_equal(byte[:, 0], np.maximum(e - 2, -127) + 127) and not byte[:, 1].any()
    P.check_fp4(q, x.astype(np.float64), np.zeros(x.shape))
    q = B.quantize_fp4(torch.from_numpy(x).cuda(), "nvfp4")
    big = e >= -88  # 2^-88 = 3.2e-27 > 2688e-30: above the row-scale floor the largest value comes back within the row scale's two roundings
    assert np.allclose(P.values(q)[big, 3], x[big, 3], rtol=4 * U, atol=0)
    assert np.all(np.isfinite(P.values(q)))
    assert np.all(np.abs(P.values(q)[~big]) <= 6 * 448 * 1e-30)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("rot", [0, 64])
def test_quantize_fp4_not_finite(bad, rot):
    x = rows(5, 3, 256)
    ref = {f: B.quantize_fp4(x, f, rot_size=rot) for f in ("mxfp4", "nvfp4")}
    x[1, 70] = bad
    v = P.values(B.quantize_fp4(x, "mxfp4", rot_size=rot))
    w = P.values(ref["mxfp4"])
    hit = slice(64, 96) if not rot else slice(64, 128)
    assert np.isnan(v[1, hit]).all()
    keep = np.ones(256, bool)
    keep[hit] = False
    assert np.array_equal(v[1, keep], w[1, keep]) and np.array_equal(v[[0, 2]], w[[0, 2]])
    q = B.quantize_fp4(x, "nvfp4", rot_size=rot)
    v, w = P.values(q), P.values(ref["nvfp4"])
    assert np.isnan(v[1]).all() and np.array_equal(v[[0, 2]], w[[0, 2]])
    assert not q.packed[1].any()
    q = B.quantize_fp4(x, "nvfp4", rot_size=rot, row_scale=1.0)  # given scales: only the blocks are marked
    v = P.values(q)
    assert np.isnan(v[1, 64:80]).all() and np.isfinite(v[1, :64]).all()


def test_quantize_fp4_given_row_scales():
    x = rows(9, 6, 96, torch.bfloat16)
    g = torch.tensor([0.5, 1e-3, 3.0, 0.0, float("nan"), -1.0], device="cuda")
    q = B.quantize_fp4(x, "nvfp4", row_scale=g)
    assert torch.equal(q.row_scale[:3], g[:3]) and torch.isnan(q.row_scale[3:]).all()
    assert np.isnan(P.values(q)[3:]).all()
    top = B.quantize_fp4(x[:3], "nvfp4", row_scale=g[:3])
    P.check_fp4(top, f64(x[:3]), np.zeros((3, 96)), given=True)
    for s in (0.25, torch.tensor(0.25), torch.tensor([0.25], device="cuda")):
        q = B.quantize_fp4(x, "nvfp4", row_scale=s)
        assert torch.equal(q.row_scale, torch.full((6,), 0.25, device="cuda"))
    with pytest.raises(ValueError, match="row_scale"):
        B.quantize_fp4(x, "nvfp4", row_scale=g[:4])


def same(q, p):
    return (torch.equal(q.packed, p.packed) and torch.equal(q.scales, p.scales)
            and (q.row_scale is None or torch.equal(q.row_scale, p.row_scale)))


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_quantize_fp4_layouts(fmt):
    """Strided, unaligned, transposed, leading dimensions, CPU tensors, no rows."""
    x = rows(3, 40, 201, torch.bfloat16)
    want = B.quantize_fp4(x[:, :160].contiguous(), fmt, rot_size=32)
    assert same(want, B.quantize_fp4(x[:, :160], fmt, rot_size=32))
    assert same(B.quantize_fp4(x[:, 1:161].contiguous(), fmt), B.quantize_fp4(x[:, 1:161], fmt))
    assert same(B.quantize_fp4(x.T.contiguous(), fmt), B.quantize_fp4(x.T, fmt))
    assert same(B.quantize_fp4(x[::2].contiguous(), fmt), B.quantize_fp4(x[::2], fmt))
    assert same(B.quantize_fp4(x[3:4].expand(5, -1).contiguous(), fmt), B.quantize_fp4(x[3:4].expand(5, -1), fmt))
    q = B.quantize_fp4(x[:, :160].reshape(5, 8, 160), fmt, rot_size=32)
    assert same(want, q) and tuple(B.dequantize_fp4(q).shape) == (5, 8, 160)
    assert tuple(B.dequantize_fp4(B.quantize_fp4(x[0], fmt)).shape) == (224,)
    c = B.quantize_fp4(x[:, :160].cpu(), fmt, rot_size=32)
    assert not c.packed.is_cuda and same(want, c.to("cuda"))
    assert torch.equal(B.dequantize_fp4(c), B.dequantize_fp4(want).cpu())
    e = B.quantize_fp4(x[:0], fmt, rot_size=1024)
    assert e.rows == 0 and tuple(B.dequantize_fp4(e).shape) == (0, 1024)
    assert torch.equal(want.block_scales().cpu(), torch.from_numpy(P.block_scales(want)))


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_dequantize_fp4(fmt, dtype):
    q = B.quantize_fp4(rows(8, 130, 700), fmt, rot_size=64)
    v, s, g = P.decode(q)
    want = torch.from_numpy((v * np.repeat(s, P.BLOCK[fmt], 1)).astype(np.float32))  # exact
    want = (want * torch.from_numpy(g.astype(np.float32))[:, None]).to(dtype)
    assert torch.equal(B.dequantize_fp4(q, dtype).cpu(), want)


# -------------------------------------------------------------- rmsnorm_quantize
def norm64(x, w, r, eps):
    h = f64(x) if r is None else f64(x) + f64(r)
    return h, h / np.sqrt((h ** 2).mean(1, keepdims=True) + eps) * f64(w)


@pytest.mark.parametrize("fmt", ["int8", "mxfp4", "nvfp4"])
@pytest.mark.parametrize("m,k,rot,dtype,wdtype,res", [
    (1, 1, 0, torch.float32, torch.float32, True), (1, 4096, 0, torch.bfloat16, torch.bfloat16, True),
    (3, 17, 0, torch.float16, torch.float32, False), (65, 100, 16, torch.float32, torch.float16, True),
    (130, 513, 32, torch.bfloat16, torch.bfloat16, True), (9, 5000, 64, torch.float16, torch.float16, False),
    (20, 4096, 256, torch.bfloat16, torch.float32, True), (4, 10000, 512, torch.float16, torch.float16, True),
    (2, 40000, 128, torch.bfloat16, torch.bfloat16, True),
])
def test_rmsnorm_quantize(fmt, m, k, rot, dtype, wdtype, res):
    x = rows(m + k, m, k, dtype)
    w = (1 + 0.3 * torch.randn(k, device="cuda", generator=gen(k))).to(wdtype)
    r = rows(m * k, m, k, dtype, 2.0) if res else None
    q, h = B.rmsnorm_quantize(x, w, residual=r, eps=1e-5, fmt=fmt, rot_size=rot)
    h64, y64 = norm64(x, w, r, float(np.float32(1e-5)))
    if res:
        want = (x.float() + r.float()).to(dtype)
        assert torch.equal(h, want)
    else:
        assert h is None
    unit = max(rot, 1 if fmt == "int8" else 32)
    kp = -(-k // unit) * unit
    z, slack = rotated(y64, rot, kp)
    # y carries five roundings: h, the mean over h's, the root, two products
    a = np.zeros_like(z)
    a[:, :k] = 5 * U * np.abs(y64)
    slack = slack * 1.01 + (a if not rot else np.repeat(a.reshape(-1, rot).sum(1) / np.sqrt(rot), rot).reshape(z.shape))
    if fmt != "int8":
        P.check_fp4(q, z, slack)
        return
    s, c = f64(q.scales), f64(q.codes)
    top = np.abs(z).max(1, keepdims=True)
    assert np.all(np.abs(s - np.maximum(top / 127, 1e-30)) <= 2 * U * top / 127 + slack.max(1, keepdims=True) / 127)
    # a code is the nearest integer to z/s up to the reciprocal, the product and the addition of 1/2
    y, off = z / s, np.abs(z / s - c)
    tol = 2 * U * np.abs(y) + U * (np.abs(y) + 1) + slack / s
    assert np.all(off <= 0.5 + tol) and np.abs(c).max() <= 128
    assert torch.equal(q.sums, q.codes.sum(1, dtype=torch.int32))
    want = (q.codes.float() * q.scales).to(torch.bfloat16)
    assert torch.equal(B.dequantize_int8(q, torch.bfloat16), want)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("rot", [0, 16, 32, 64, 128, 256, 512])
def test_rmsnorm_rounds_each_step(fmt, rot):
    """The norm's fp32 products, rounded one by one, are what is rotated and quantized: bit for bit the
    quantizer's own result on them (the norm itself in 64 bits, rounded to fp32)."""
    x, r = rows(rot + 1, 200, 1100, torch.bfloat16), rows(rot + 2, 200, 1100, torch.bfloat16)
    w = 1 + 0.3 * torch.randn(1100, device="cuda", generator=gen(4))
    q, _ = B.rmsnorm_quantize(x, w, residual=r, eps=1e-5, fmt=fmt, rot_size=rot)
    h = x.float() + r.float()
    rstd = (1.0 / torch.sqrt((h.double() ** 2).mean(1, keepdim=True) + float(np.float32(1e-5)))).float()
    assert same(q, B.quantize_fp4(h * rstd * w, fmt, rot_size=rot))


def test_rmsnorm_int8_rounds_half_away():
    """Ties go away from zero, as in the framework's other INT8 codes.  The squares sum to
    16 * 32^2 and the largest value is 127, so that norm and scale are exact."""
    x = [127, 2.5, -2.5, 0.5, -0.5, 1.5, -1.5, 3.5, -3.5, 14, 4, 1, 0, 0, 0, 0]
    q, _ = B.rmsnorm_quantize(torch.tensor([x], device="cuda"), torch.full((16,), 32.0, device="cuda"), eps=0.0)
    assert float(q.scales) == 1.0
    assert q.codes.tolist() == [[127, 3, -3, 1, -1, 2, -2, 4, -4, 14, 4, 1, 0, 0, 0, 0]]


@pytest.mark.parametrize("fmt", ["int8", "mxfp4", "nvfp4"])
def test_rmsnorm_special_rows(fmt):
    """A zero row, a tiny row, a large row and rows that are not finite, next to an ordinary one."""
    k = 96
    x = rows(1, 6, k)
    x[1] = 0
    x[2] *= 1e-20
    x[3] *= 1e18
    x[4, 7] = float("nan")
    x[5, 9] = float("inf")
    w = torch.ones(k, device="cuda")
    q, _ = B.rmsnorm_quantize(x, w, fmt=fmt)
    one, _ = B.rmsnorm_quantize(x[:1].contiguous(), w, fmt=fmt)
    v = f64(B.dequantize_int8(q)) if fmt == "int8" else P.values(q)
    o = f64(B.dequantize_int8(one)) if fmt == "int8" else P.values(one)
    assert np.array_equal(v[:1], o)
    assert not v[1].any() and np.isfinite(v[:4]).all() and np.isnan(v[4:]).all()
    y = norm64(x, w, None, 1e-6)[1]
    step = {"int8": np.abs(y).max(1, keepdims=True) / 127, "mxfp4": np.abs(y).max(1, keepdims=True) / 2, "nvfp4": np.abs(y).max(1, keepdims=True) / 3}[fmt]
    assert np.all(np.abs(v - y)[:4] <= step[:4] + 1e-30)


@pytest.mark.parametrize("fmt", ["int8", "mxfp4", "nvfp4"])
def test_rmsnorm_layouts(fmt):
    x, r = rows(3, 24, 130, torch.bfloat16), rows(4, 24, 130, torch.bfloat16)
    w = torch.ones(127, device="cuda")
    def parts(o):
        q, h = o
        return [h] + ([q.codes, q.scales, q.sums] if fmt == "int8" else [t for t in (q.packed, q.scales, q.row_scale) if t is not None])
    want = parts(B.rmsnorm_quantize(x[:, 3:].contiguous(), w, r[:, 3:].contiguous(), fmt=fmt, rot_size=32))
    got = parts(B.rmsnorm_quantize(x[:, 3:], w, r[:, 3:], fmt=fmt, rot_size=32))
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    q, h = B.rmsnorm_quantize(x[:, 3:].reshape(2, 12, 127), w, r[:, 3:].reshape(2, 12, 127), fmt=fmt, rot_size=32)
    assert tuple(h.shape) == (2, 12, 127) and torch.equal(h.reshape(24, 127), want[0]) and q.lead == (2, 12)
    q, h = B.rmsnorm_quantize(x[:, 3:].cpu(), w.cpu(), r[:, 3:].cpu(), fmt=fmt, rot_size=32)
    assert not h.is_cuda and torch.equal(h.cuda(), want[0])
    assert all(torch.equal(a.cpu(), b) for a, b in zip(want, parts((q, h))))
    q, h = B.rmsnorm_quantize(x[:0], torch.ones(130, device="cuda"), r[:0], fmt=fmt)
    assert q.rows == 0 and tuple(h.shape) == (0, 130)


# ---------------------------------------------------------------------- products
def steps_tol(k, out):
    """Sums of exact products in fp32: the k/64 tensor-core steps may each truncate (2^-23) when
    their 64 products are aligned and again when they are added to the running sum; then at
    most eight partial sums are added and two row factors and the bias applied (u each)."""
    return (-(-k // 64) * 2 * 2.0 ** -23) + 11 * U


def check_product(y, a64, b64, bias, k, out):
    ref = a64 @ b64.T
    mag = np.abs(a64) @ np.abs(b64).T
    if bias is not None:
        ref, mag = ref + f64(bias), mag + np.abs(f64(bias))
    tol = steps_tol(k, out) * mag + HALF[out] * np.abs(ref) * (1 + 1e-3) + TINY[out]
    got = f64(y)
    assert got.shape == ref.shape
    bad = ~(np.abs(got - ref) <= tol)
    assert not bad.any(), (bad.sum(), np.argwhere(bad)[:5], got[bad][:5], ref[bad][:5])


PRODUCTS = [
    (1, 1, 32, torch.float32, False), (1, 128, 64, torch.bfloat16, True), (2, 130, 96, torch.float16, False),
    (16, 256, 256, torch.float32, True), (17, 100, 288, torch.bfloat16, False), (33, 1000, 1433, torch.float16, True),
    (64, 64, 4096, torch.float32, False), (65, 200, 512, torch.bfloat16, True), (128, 384, 1024, torch.float32, True),
    (129, 128, 320, torch.bfloat16, False), (300, 520, 2080, torch.float32, True), (257, 1024, 4096, torch.bfloat16, True),
    (1, 4096, 16384, torch.bfloat16, False), (1000, 77, 640, torch.float16, False), (5, 3000, 32, torch.float32, False),
    (2304, 2200, 800, torch.bfloat16, True), (2400, 2177, 1433, torch.float16, True), (4700, 1300, 320, torch.float32, False),
    (2305, 2304, 4096, torch.float32, True), (300, 4096, 4096, torch.bfloat16, True), (700, 600, 2048, torch.float16, True),
    (180, 5000, 1024, torch.float32, False), (1024, 1024, 512, torch.bfloat16, True), (90, 12288, 256, torch.float16, True),
    (520, 333, 8192, torch.bfloat16, True),
]


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("m,n,k,out,bias", PRODUCTS)
def test_matmul_fp4(fmt, m, n, k, out, bias):
    a = B.quantize_fp4(rows(m + k, m, k), fmt)
    b = B.quantize_fp4(rows(n + 7 * k, n, k, std=0.05), fmt)
    bv = torch.randn(n, device="cuda", generator=gen(n)).to(torch.float32 if n % 2 else out) if bias else None
    y = B.matmul_fp4(a, b, bias=bv, out_dtype=out)
    assert y.dtype == out
    check_product(y, P.values(a), P.values(b), bv, a.columns, out)


@pytest.mark.parametrize("m,n,k,out,bias", PRODUCTS + [(3, 40, 1, torch.float32, True), (200, 150, 15, torch.bfloat16, True)])
@pytest.mark.parametrize("asym", [False, True])
def test_matmul_int8(m, n, k, out, bias, asym):
    """The integer sums are exact: only the scaling, the bias and the last rounding are left."""
    g = gen(m + n + k)
    ld = (k + 15) & ~15
    c = torch.randint(-128, 128, (m, ld), device="cuda", generator=g).to(torch.int8)[:, :k]
    w = torch.randint(-128, 128, (n, ld), device="cuda", generator=g).to(torch.int8)[:, :k]
    s = torch.rand(m, 1, device="cuda", generator=g) + 0.1
    ws = (torch.rand(n, 1, device="cuda", generator=g) * 1e-3 + 1e-4).half()
    zp = torch.randint(-128, 128, (n, 1), device="cuda", generator=g).to(torch.int8) if asym else None
    bv = torch.randn(n, device="cuda", generator=g) if bias else None
    y = B.matmul_int8(B.Int8Rows(c, s), w, ws, zp, bias=bv, out_dtype=out)
    acc = f64(c) @ (f64(w) - (f64(zp) if asym else 0)).T
    ref = acc * f64(s) * f64(ws).T
    tol = 3 * U * np.abs(ref) * (1 + 1e-3)
    if bias:
        ref = ref + f64(bv)
        tol = tol + U * np.abs(ref) * (1 + 1e-3)
    tol = tol + HALF[out] * np.abs(ref) * (1 + 1e-3) + TINY[out]
    bad = ~(np.abs(f64(y) - ref) <= tol)
    assert not bad.any(), (bad.sum(), np.argwhere(bad)[:5])
    sums = c.sum(1, dtype=torch.int32)
    assert torch.equal(y, B.matmul_int8(B.Int8Rows(c, s, sums), w, ws, zp, bias=bv, out_dtype=out))
    # contiguous codes of any width and unaligned ones give the same
    assert torch.equal(y, B.matmul_int8(B.Int8Rows(c.contiguous(), s), w.contiguous(), ws.reshape(-1), zp, bias=bv, out_dtype=out))
    wide = torch.zeros(n, k + 5, dtype=torch.int8, device="cuda")
    wide[:, 5:] = w
    assert torch.equal(y, B.matmul_int8(B.Int8Rows(c, s), wide[:, 5:], ws, zp, bias=bv, out_dtype=out))


def test_matmul_int8_extreme_sums():
    """The largest sums that int32 holds, with and without zero-points."""
    for k, zp in ((131071, None), (65535, 127)):
        c = torch.full((2, k), -128, dtype=torch.int8, device="cuda")
        w = torch.full((3, k), -128, dtype=torch.int8, device="cuda")
        c[1] = 127
        z = None if zp is None else torch.full((3, 1), zp, dtype=torch.int8, device="cuda")
        y = B.matmul_int8(B.Int8Rows(c, torch.ones(2, 1, device="cuda")), w, torch.ones(3, 1, device="cuda").half(), z, out_dtype=torch.float32)
        want = f64(c).sum(1)[:, None] * (-128 - (zp or 0))
        assert np.all(np.abs(f64(y) - want) <= U * np.abs(want))


def test_products_with_no_rows_and_leading_dimensions():
    for m, n in ((0, 5), (4, 0), (0, 0)):
        a, b = B.quantize_fp4(rows(1, 6, 64)[:m], "nvfp4"), B.quantize_fp4(rows(2, 6, 64)[:n], "nvfp4")
        assert tuple(B.matmul_fp4(a, b).shape) == (m, n)
        c = B.Int8Rows(torch.zeros(m, 64, dtype=torch.int8, device="cuda"), torch.ones(m, 1, device="cuda"))
        y = B.matmul_int8(c, torch.zeros(n, 64, dtype=torch.int8, device="cuda"), torch.ones(n, 1, device="cuda").half())
        assert tuple(y.shape) == (m, n)
    x = rows(3, 12, 96)
    b = B.quantize_fp4(rows(4, 20, 96), "mxfp4")
    flat = B.matmul_fp4(B.quantize_fp4(x, "mxfp4"), b)
    lead = B.matmul_fp4(B.quantize_fp4(x.reshape(3, 4, 96), "mxfp4"), b)
    assert tuple(lead.shape) == (3, 4, 20) and torch.equal(lead.reshape(12, 20), flat)
    cpu = B.matmul_fp4(B.quantize_fp4(x, "mxfp4").to("cpu"), b.to("cpu"))
    assert not cpu.is_cuda and torch.equal(cpu, flat.cpu())
    none = B.FP4Tensor(torch.empty(3, 0, dtype=torch.uint8, device="cuda"), torch.empty(0, dtype=torch.uint8, device="cuda"), None)
    bias = torch.arange(3.0, device="cuda")
    assert torch.equal(B.matmul_fp4(none, none, bias=bias, out_dtype=torch.float32), bias.expand(3, 3))


@pytest.mark.parametrize("m", [1, 20, 40, 100, 200])
def test_products_do_not_depend_on_other_rows(m):
    """A token's outputs are the same whatever else is in a batch of the same tile shape, and run to run."""
    x, w = rows(5, m, 2000), rows(6, 300, 2000)
    for fmt in ("mxfp4", "nvfp4"):
        b = B.quantize_fp4(w, fmt)
        y = B.matmul_fp4(B.quantize_fp4(x, fmt), b, out_dtype=torch.float32)
        assert torch.equal(y, B.matmul_fp4(B.quantize_fp4(x, fmt), b, out_dtype=torch.float32))
        x2 = x.clone()
        x2[1:] = 3.0
        assert torch.equal(y[0], B.matmul_fp4(B.quantize_fp4(x2, fmt), b, out_dtype=torch.float32)[0])


@pytest.mark.parametrize("m", [3, 50, 200])
@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_nan_stays_in_its_row_and_column(fmt, m):
    x, w = rows(7, m, 300), rows(8, 140, 300)
    clean = B.matmul_fp4(B.quantize_fp4(x, fmt), B.quantize_fp4(w, fmt), out_dtype=torch.float32)
    x[1, 250], w[9, 3] = float("nan"), float("inf")
    y = B.matmul_fp4(B.quantize_fp4(x, fmt), B.quantize_fp4(w, fmt), out_dtype=torch.float32)
    hit = torch.zeros_like(y, dtype=torch.bool)
    hit[1], hit[:, 9] = True, True
    assert torch.isnan(y[hit]).all() and torch.equal(y[~hit], clean[~hit])


def test_products_write_only_their_output():
    """A wider output buffer keeps what lies beyond the columns and rows."""
    a, b = B.quantize_fp4(rows(1, 50, 128), "mxfp4"), B.quantize_fp4(rows(2, 70, 128), "mxfp4")
    big = B.quantize_fp4(rows(1, 150, 128), "mxfp4")
    for q in (a, big):
        want = B.matmul_fp4(q, b, out_dtype=torch.float32)
        buf = torch.full((q.rows + 2, 80), 7.0, device="cuda")
        nat.check(nat.load().ic_fp4_matmul(q.packed.data_ptr(), q.scales.data_ptr(), None, b.packed.data_ptr(), b.scales.data_ptr(),
                                           None, nat.IC_MXFP4, q.rows, 70, 128, None, 0, nat.IC_F32, buf[1].data_ptr(), 80,
                                           nat.stream_ptr(buf.device)))
        assert torch.equal(buf[1:-1, :70], want)
        buf[1:-1, :70] = 7.0
        assert (buf == 7.0).all()


# ------------------------------------------------------------- used together
def layer64(x, r, w, lin, rot):
    h, y = norm64(x, w, r, float(np.float32(1e-6)))
    return h, y @ f64(lin).T


@pytest.mark.parametrize("fmt", ["int8", "mxfp4", "nvfp4"])
@pytest.mark.parametrize("m", [1, 24, 150])
def test_quantized_layer(fmt, m):
    """norm -> rotation -> quantized product with weights of the framework's own converters,
    against the unquantized layer: the error is that of the codes, far below the signal."""
    k, n, rot = 1024, 768, 256
    x, r = rows(1, m, k, torch.bfloat16), rows(2, m, k, torch.bfloat16)
    w = torch.ones(k, device="cuda")
    lin = torch.randn(n, k, device="cuda", generator=gen(3)) * 0.02
    q, h = B.rmsnorm_quantize(x, w, residual=r, fmt=fmt, rot_size=rot)
    if fmt == "int8":
        d = B.rtn_quantize_fused(lin, rot, int_bits=8, asymmetric=True)
        y = B.matmul_int8(q, d["codes"], d["scales"], d["zero_points"], out_dtype=torch.float32)
    else:
        y = B.matmul_fp4(q, B.quantize_fp4(lin, fmt, rot_size=rot), out_dtype=torch.float32)
    want = layer64(x, r, w, lin, rot)[1]
    rel = np.linalg.norm(f64(y) - want) / np.linalg.norm(want)
    # uniform 8-bit codes of a rotated (near-normal) row are off by about (4 sigma/127)/sqrt(12) of its
    # rms, twice over; E2M1 codes by about a tenth, twice over: factors of two to three of margin
    assert rel < (0.04 if fmt == "int8" else 0.3)
    assert torch.equal(h, (x.float() + r.float()).to(torch.bfloat16))


@pytest.mark.parametrize("fmt", ["int8", "nvfp4"])
def test_quantized_layer_on_a_stream_and_in_a_graph(fmt):
    k, n, rot = 512, 256, 64
    lin = torch.randn(n, k, device="cuda", generator=gen(3)) * 0.02
    d = B.rtn_quantize_fused(lin, rot, int_bits=8, asymmetric=True)
    wq = B.quantize_fp4(lin, "nvfp4", rot_size=rot)
    w = torch.ones(k, device="cuda")

    def layer(x, r):
        q, h = B.rmsnorm_quantize(x, w, residual=r, fmt=fmt, rot_size=rot)
        return (B.matmul_int8(q, d["codes"], d["scales"], d["zero_points"]) if fmt == "int8" else B.matmul_fp4(q, wq)), h

    x, r = rows(1, 9, k, torch.bfloat16), rows(2, 9, k, torch.bfloat16)
    want = layer(x, r)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = layer(x, r)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graphs = []
    for _ in range(2):  # two graphs over the same operands, replayed in turn
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = layer(x, r)
        graphs.append((g, out))
    x2, r2 = rows(3, 9, k, torch.bfloat16), rows(4, 9, k, torch.bfloat16)
    want2 = layer(x2, r2)
    x.copy_(x2), r.copy_(r2)
    for g, out in graphs + graphs[::-1]:
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want2[0]) and torch.equal(out[1], want2[1])


def test_offsets_beyond_32_bits():
    """Rows whose elements, codes and outputs lie past 2^32 bytes."""
    m, k = 70000, 36000  # 2.5e9 elements
    x = torch.zeros(m, k, device="cuda", dtype=torch.bfloat16)
    last = rows(1, 3, k, torch.bfloat16)
    x[-3:] = last
    w = torch.ones(k, device="cuda")
    for fmt in ("mxfp4", "nvfp4"):
        q, p = B.quantize_fp4(x, fmt), B.quantize_fp4(last, fmt)
        assert torch.equal(q.packed[-3:], p.packed) and np.array_equal(P.values(tail(q, 3)), P.values(p))
        del q
    q, _ = B.rmsnorm_quantize(x, w)
    p, _ = B.rmsnorm_quantize(last, w)
    assert torch.equal(q.codes[-3:], p.codes) and torch.equal(q.scales[-3:], p.scales)
    v = torch.randint(-5, 6, (64, k), device="cuda", generator=gen(2)).to(torch.int8)
    y = B.matmul_int8(q, v, torch.ones(64, device="cuda").half())
    assert torch.equal(y[-3:].float(), B.matmul_int8(p, v, torch.ones(64, device="cuda").half()).float())
    assert not y[:-3].any()


def tail(q, n):
    """The last n rows of q as a tensor of their own."""
    return B.FP4Tensor.from_block_scales(q.packed[-n:], q.block_scales()[-n:],
                                         None if q.row_scale is None else q.row_scale[-n:].contiguous(), q.fmt)


FIRST_IN_CAPTURE = """
import torch
import int_crush_converter_b200 as B
x = torch.randn(5, 256, device="cuda")
w = torch.randn(256, device="cuda")
codes = torch.randint(-9, 10, (48, 256), device="cuda").to(torch.int8)
scales = torch.ones(48, 1, device="cuda").half()
torch.cuda.synchronize()
def f():
    q, _ = B.rmsnorm_quantize(x, w)
    p = B.quantize_fp4(x, "nvfp4", rot_size=64)
    return B.matmul_int8(q, codes, scales), B.matmul_fp4(p, p), B.dequantize_fp4(p), B.dequantize_int8(q)
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    out = f()
g.replay()
torch.cuda.synchronize()
for a, b in zip(out, f()):
    assert torch.equal(a, b)
print("captured")
"""


def test_first_calls_may_be_captured():
    """A process whose first calls of the library are part of a stream capture."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST_IN_CAPTURE], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("m,k", [(1, 32), (128, 128), (129, 512), (300, 1000)])
def test_block_scales_round_trip(fmt, m, k):
    q = B.quantize_fp4(rows(m, m, k), fmt)
    p = B.FP4Tensor.from_block_scales(q.packed, q.block_scales(), q.row_scale, fmt)
    assert torch.equal(p.scales, q.scales) and torch.equal(B.dequantize_fp4(p), B.dequantize_fp4(q))


@pytest.mark.parametrize("kind", ["mxfp4", "nvfp4", "int8"])
def test_products_on_two_streams_at_once(kind):
    """Large and small products overlapping on two streams give what they give alone."""
    big, small, w = rows(1, 2600, 1024), rows(2, 3, 1024), rows(3, 2400, 1024)
    if kind == "int8":
        c = torch.randint(-99, 100, (2400, 1024), device="cuda", generator=gen(5)).to(torch.int8)
        s = torch.ones(2400, 1, device="cuda").half()
        one = torch.ones(1024, device="cuda")
        qb, qs = B.rmsnorm_quantize(big, one)[0], B.rmsnorm_quantize(small, one)[0]
        f = lambda q: B.matmul_int8(q, c, s)  # noqa: E731
    else:
        qw, qb, qs = (B.quantize_fp4(t, kind) for t in (w, big, small))
        f = lambda q: B.matmul_fp4(q, qw)  # noqa: E731
    want = f(qb), f(qs)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for i in range(12):
        with torch.cuda.stream(streams[i % 2]):
            got.append((i % 3 == 0, f(qb) if i % 3 == 0 else f(qs)))
    torch.cuda.synchronize()
    for large, y in got:
        assert torch.equal(y, want[0] if large else want[1])


class NoBinding:
    """Every function of the native binding declines, as for arguments out of the ordinary."""

    def __getattr__(self, name):
        return lambda *a: None


@pytest.mark.parametrize("fmt", ["int8", "mxfp4", "nvfp4"])
def test_long_way_gives_the_same(fmt, monkeypatch):
    """With and without the native binding: the same tensors, shapes and types."""
    x, r = rows(1, 12, 300, torch.bfloat16).reshape(3, 4, 300), rows(2, 12, 300, torch.bfloat16).reshape(3, 4, 300)
    w, bias = torch.rand(300, device="cuda", generator=gen(3)), torch.rand(70, device="cuda", generator=gen(4))
    lin = rows(5, 70, 300)

    def layer():
        q, h = B.rmsnorm_quantize(x, w, residual=r, fmt=fmt, rot_size=32)
        if fmt == "int8":
            d = B.rtn_quantize_fused(lin, 32, int_bits=8, asymmetric=True)
            return [q.codes, q.scales, q.sums, h, B.dequantize_int8(q, torch.float16),
                    B.matmul_int8(q, d["codes"], d["scales"], d["zero_points"], bias=bias, out_dtype=torch.float32)]
        p = B.quantize_fp4(lin, fmt, rot_size=32)
        return [q.packed, q.scales, p.packed, p.scales, h, B.dequantize_fp4(q, torch.float16),
                B.matmul_fp4(q, p, bias=bias, out_dtype=torch.float32)] + ([] if fmt == "mxfp4" else [q.row_scale, p.row_scale])

    short = layer()
    monkeypatch.setattr(nat, "_fast", NoBinding())
    long = layer()
    assert [(t.shape, t.dtype, t.stride()) for t in short] == [(t.shape, t.dtype, t.stride()) for t in long]
    assert all(torch.equal(a, b) for a, b in zip(short, long))


def test_no_timeouts_were_recorded():
    import ctypes
    f = ctypes.c_uint()
    nat.check(nat.load().ic_device_status(ctypes.byref(f), nat.stream_ptr(torch.device("cuda", 0))))
    assert not f.value & nat.DEV_TIMEOUT
