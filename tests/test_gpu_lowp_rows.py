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


def beyond(q):
    """The scale bytes beyond the rows and blocks of the matrix."""
    t = q.scales.permute(0, 3, 2, 1, 4).reshape(q.scales.shape[0] * 128, -1).cpu().numpy().copy()
    t[:q.rows, :q.columns // P.BLOCK[q.fmt]] = 0
    return t


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
