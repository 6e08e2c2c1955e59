"""GPU tests of every way a low-precision product is cut: tile width, orientation and K split.  Operands
are small whole numbers (and powers of two as scales), so that the sums are exact in fp32 whatever their
order and every plan has to give the one right result, bit for bit."""

import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    import int_crush_converter_b200 as B
    from int_crush_converter_b200 import _native as nat

PLANS = [(w, s, k) for w in (16, 32, 64, 128, 192, 256) for s in (0, 1) for k in (1, 2, 4, 8)] + [(0, 0, 1)]


def operands(kind, m, n, k):
    """(a call of the product, its exact result): |sums| < 2^24 times a power of two; the row factors are powers of two."""
    g = torch.Generator(device="cuda").manual_seed(m * 7 + n * 3 + k)

    def whole(r, lim):
        return torch.randint(-lim, lim + 1, (r, k), device="cuda", generator=g)

    def twos(r):
        return torch.exp2(torch.randint(-3, 4, (r,), device="cuda", generator=g).float())
    bias = torch.randint(-9, 10, (n,), device="cuda", generator=g).float()
    if kind == "int8":
        ld = (k + 15) & ~15
        a, w = (torch.zeros(r, ld, dtype=torch.int8, device="cuda")[:, :k].copy_(whole(r, 30)) for r in (m, n))
        z = torch.randint(-20, 21, (n, 1), device="cuda", generator=g).to(torch.int8)
        s, ws = twos(m), twos(n)
        q = B.Int8Rows(a, s[:, None], a.sum(1, dtype=torch.int32))
        want = (a.double() @ (w.double() - z.double()).T) * s.double()[:, None] * ws.double() + bias.double()
        return lambda out, b: B.matmul_int8(q, w, ws.half()[:, None], z, bias=bias if b else None, out_dtype=out), want, bias.double()
    x, y = whole(m, 4), whole(n, 4)  # all of them E2M1 values
    rows = []
    for t in (x, y):
        scales = twos(t.shape[0])
        t[:, ::16] = 4  # the largest of every block: mxfp4's scale is the row's power of two
        rows.append((t.float() * scales[:, None], scales))
    if kind == "mxfp4":
        a, b = (B.quantize_fp4(t, kind) for t, _ in rows)
    else:  # amax / (6 * 2s) = 1/3: every block's scale is the nearest E4M3 number, 11/32, and sums are multiples of (11/64)^2
        a, b = (B.quantize_fp4(t, kind, row_scale=s * 2) for t, s in rows)
    want = B.dequantize_fp4(a).double() @ B.dequantize_fp4(b).double().T + bias.double()
    return lambda out, c: B.matmul_fp4(a, b, bias=bias if c else None, out_dtype=out), want, bias.double()


def check(f, want, bias, plan, out, with_bias):
    nat.check(nat.load().ic_selftest_matmul_plan(*plan))
    got = f(out, with_bias)
    exact = want if with_bias else want - bias
    assert torch.equal(got, exact.float().to(out)), plan


# rows of activations x rows of weights x K: ragged against every width, K tails, aligned rows of y and others,
# tiles that begin inside a 128-row scale tile
SHAPES = [(1, 333, 4100), (16, 520, 1088), (13, 17, 1500), (31, 1000, 2080), (130, 300, 1433), (300, 200, 1100), (385, 449, 1024),
          (700, 513, 1120)]


@pytest.mark.parametrize("kind", ["int8", "mxfp4", "nvfp4"])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_every_plan(kind, m, n, k):
    f, want, bias = operands(kind, m, n, k)
    stages = -(-(k if kind == "int8" else -(-k // 32) * 16) // 128)
    ran = 0
    for i, (width, swap, splits) in enumerate(PLANS):
        qn = m if swap else n
        if (width in (16, 32) and qn > width) or splits > stages:
            nat.check(nat.load().ic_selftest_matmul_plan(width, swap, splits))
            with pytest.raises(ValueError, match="plan"):
                one_call(kind, f)
            continue
        for j, out in enumerate((torch.float32, torch.float16, torch.bfloat16)):
            check(f, want, bias, (width, swap, splits), out, (i + j) % 2 == 0)
            ran += 1
    assert ran >= 3 * 9


def one_call(kind, f):
    """The native binding declines where the entry point refuses, and the long way calls it again: the refusal
    is seen with the binding out of the way."""
    fast, nat._fast = nat._fast, type("None_", (), {"__getattr__": lambda self, name: lambda *a: None})()
    try:
        f(torch.float32, False)
    finally:
        nat._fast = fast


def test_plan_arguments():
    for bad in ((8, 0, 1), (48, 0, 1), (512, 0, 1), (-16, 0, 1), (64, 2, 1), (64, 0, 3), (64, 0, 16), (64, 0, 0)):
        with pytest.raises(ValueError):
            nat.check(nat.load().ic_selftest_matmul_plan(*bad))
