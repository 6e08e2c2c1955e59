"""GPU test of the low-precision operators beside other Python threads."""

import threading
import time

import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    import int_crush_converter_b200 as B


def operators():
    x, w = torch.randn(4, 64, device="cuda"), torch.ones(64, device="cuda")
    q, p = B.rmsnorm_quantize(x, w)[0], B.quantize_fp4(x, "nvfp4")
    c, s = torch.ones(32, 64, dtype=torch.int8, device="cuda"), torch.ones(32, 1, device="cuda").half()
    return {"quantize_fp4": lambda: B.quantize_fp4(x), "dequantize_fp4": lambda: B.dequantize_fp4(p),
            "matmul_fp4": lambda: B.matmul_fp4(p, p), "rmsnorm_int8": lambda: B.rmsnorm_quantize(x, w),
            "rmsnorm_fp4": lambda: B.rmsnorm_quantize(x, w, fmt="mxfp4"), "dequantize_int8": lambda: B.dequantize_int8(q),
            "matmul_int8": lambda: B.matmul_int8(q, c, s)}


@pytest.mark.parametrize("name", ["quantize_fp4", "dequantize_fp4", "matmul_fp4", "rmsnorm_int8", "rmsnorm_fp4", "dequantize_int8",
                                  "matmul_int8"])
def test_other_threads_run_while_a_launch_waits(name):
    """The stream is busy for about a second, so that some launch waits for room in its queue; this thread
    goes on meanwhile."""
    f = operators()[name]
    f()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    stop = threading.Event()

    def calls():
        with torch.cuda.stream(side):
            torch.cuda._sleep(1_500_000_000)
            for _ in range(4000):
                f()
        stop.set()

    t = threading.Thread(target=calls)
    start = last = time.perf_counter()
    t.start()
    gap = 0.0
    while not stop.is_set():
        time.sleep(0.001)
        now = time.perf_counter()
        gap, last = max(gap, now - last), now
    t.join()
    torch.cuda.synchronize()
    assert last - start > 0.4, "no launch waited"
    assert gap < 0.3
