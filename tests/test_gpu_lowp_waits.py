"""GPU test of products whose waits give up: the loads of some stages are left out, so that a barrier
never completes; after a short limit the kernels return, with NaN for every element that lacks its sum."""

import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    import int_crush_converter_b200 as B
    from int_crush_converter_b200 import _native as nat


def timed_out():
    f = ctypes.c_uint()
    nat.check(nat.load().ic_device_status(ctypes.byref(f), nat.stream_ptr(torch.device("cuda", 0))))
    return bool(f.value & nat.DEV_TIMEOUT)


def product(kind, m, n, k, out):
    g = torch.Generator(device="cuda").manual_seed(m + n + k)
    x, w = torch.randn(m, k, device="cuda", generator=g), torch.randn(n, k, device="cuda", generator=g)
    if kind == "int8":
        q, _ = B.rmsnorm_quantize(x, torch.ones(k, device="cuda"))
        c = torch.randint(-99, 100, (n, k), device="cuda", generator=g).to(torch.int8)
        s, z = torch.ones(n, 1, device="cuda").half(), torch.ones(n, 1, dtype=torch.int8, device="cuda")
        return lambda: B.matmul_int8(q, c, s, z, out_dtype=out)
    a, b = B.quantize_fp4(x, kind), B.quantize_fp4(w, kind)
    return lambda: B.matmul_fp4(a, b, out_dtype=out)


# one token (weights in P, split K), a few hundred rows, one narrow tile without a split, CTA pairs with
# one tile and with several tiles each, rows of y that are not 16-byte aligned
SHAPES = [(1, 700, 4096), (300, 520, 4096), (40, 64, 128), (2600, 2400, 512), (5000, 4100, 256), (130, 77, 256)]


@pytest.mark.parametrize("kind", ["int8", "mxfp4", "nvfp4"])
@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("out", [torch.float32, torch.float16, torch.bfloat16])
def test_waits_that_give_up_leave_nan(kind, m, n, k, out):
    f = product(kind, m, n, k, out)
    want = f()
    assert not want.isnan().any()
    timed_out()
    nat.check(nat.load().ic_selftest_matmul_stall(0, 1_000_000))  # nothing is loaded
    got = f()
    assert timed_out() and got.isnan().all()
    assert torch.equal(f(), want) and not timed_out()  # the next product is an ordinary one


@pytest.mark.parametrize("kind", ["int8", "mxfp4", "nvfp4"])
@pytest.mark.parametrize("m,n,k,stages", [
    (1, 700, 4608, 4), (1, 700, 2100, 2), (300, 520, 2100, 3), (2600, 2400, 512, 2), (5000, 4100, 256, 1), (5000, 4100, 256, 2),
    (5000, 4100, 512, 7),
])
def test_some_stages_missing(kind, m, n, k, stages):
    """What has its sum keeps it; all else is NaN: some CTAs of a split, or a pair's later tiles."""
    f = product(kind, m, n, k, torch.float32)
    want = f()
    timed_out()
    nat.check(nat.load().ic_selftest_matmul_stall(stages, 1_000_000))
    got = f()
    nan = got.isnan()
    assert torch.equal(got[~nan], want[~nan])
    assert timed_out() == bool(nan.any())
    assert torch.equal(f(), want) and not timed_out()


def test_stall_arguments():
    lib = nat.load()
    for stages, limit in ((-1, 1_000_000), (0, 99_999), (0, 2_000_000_001)):
        with pytest.raises(ValueError):
            nat.check(lib.ic_selftest_matmul_stall(stages, limit))
