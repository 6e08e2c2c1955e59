"""Plain 64-bit forms of the low-precision operators (numpy), shared by their tests."""

import numpy as np

E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
BLOCK = {"mxfp4": 32, "nvfp4": 16}


def e4m3(byte):
    """Values of E4M3 bytes (all here are non-negative)."""
    b = byte.astype(np.int64)
    e, m = b >> 3, b & 7
    v = np.where(e > 0, (1 + m / 8.0) * 2.0 ** (e - 7.0), m * 2.0 ** -9)
    return np.where(b == 0x7F, np.nan, v)


E4M3_GRID = e4m3(np.arange(0x7F))


def block_scales(q):
    """Scale bytes row by row from the tiled layout, indexed as documented."""
    t = q.scales.cpu().numpy()
    r = np.arange(q.rows)[:, None]
    b = np.arange(q.columns // BLOCK[q.fmt])[None, :]
    return t[r // 128, b // 4, r % 32, r % 128 // 32, b % 4]


def decode(q):
    """(codes as values, block scales, row scales) of an FP4Tensor in 64 bits."""
    p = q.packed.cpu().numpy().astype(np.int64)
    code = np.empty((q.rows, q.columns), np.int64)
    code[:, 0::2], code[:, 1::2] = p & 15, p >> 4
    v = np.where(code & 8, -1.0, 1.0) * E2M1[code & 7]
    byte = block_scales(q)
    s = np.where(byte == 255, np.nan, 2.0 ** (byte.astype(np.float64) - 127)) if q.fmt == "mxfp4" else e4m3(byte)
    g = np.ones(q.rows) if q.row_scale is None else q.row_scale.cpu().numpy().astype(np.float64)
    return v, s, g


def values(q):
    v, s, g = decode(q)
    return v * np.repeat(s, BLOCK[q.fmt], 1) * g[:, None]


def hadamard(rot):
    if rot & 0x55555555 == rot:
        base = np.array([[1, 1, 1, -1], [1, 1, -1, 1], [1, -1, 1, 1], [-1, 1, 1, 1]], np.float64)
    else:
        base = np.array([[1, 1], [1, -1]], np.float64)
    h = np.ones((1, 1))
    while h.shape[0] < rot:
        h = np.kron(h, base)
    return h / np.sqrt(rot)


def rotate(x, rot, kp):
    z = np.zeros((x.shape[0], kp))
    z[:, :x.shape[1]] = x
    return z if not rot else (z.reshape(-1, rot) @ hadamard(rot).T).reshape(z.shape)


def off_nearest(y, chosen, grid):
    """How much further `chosen` is from y than the nearest value of `grid` (ascending)."""
    i = np.clip(np.searchsorted(grid, y), 1, len(grid) - 1)
    best = np.minimum(np.abs(y - grid[i - 1]), np.abs(y - grid[i]))
    return np.abs(y - chosen) - best


def check_fp4(q, z, slack, given=None):
    """`q` against the 64-bit rows z it quantizes; `slack`: how far an fp32 input of the
    quantizer may be from z (absolute, same shape).  Every chosen scale and code is the
    nearest one up to the fp32 roundings made before choosing: u = 2^-24 each, at most
    three for a scale (6g, its reciprocal, the product) and three for a code (s*g, its
    reciprocal, the product); a choice made at y(1+d) is at most 2|y||d| further off."""
    u = 2.0 ** -24
    v, s, g = decode(q)
    rows, kp = z.shape
    blk = BLOCK[q.fmt]
    zb, sb = np.abs(z).reshape(rows, -1, blk), slack.reshape(rows, -1, blk)
    top, tops = zb.max(2), sb.max(2)
    if q.fmt == "mxfp4":
        def exponent(a):
            with np.errstate(divide="ignore"):
                return 2.0 ** np.clip(np.floor(np.log2(a)) - 2, -127, 127)
        assert np.all((exponent(np.maximum(top - tops, 0)) <= s) & (s <= exponent(top + tops)))
        step = s
    else:
        if given is None:
            want = np.maximum(np.abs(z).max(1) / 2688, 1e-30)
            assert np.all(np.abs(g - want) <= 2 * u * want + slack.max(1) / 2688 + 2.0 ** -150)
        t = np.minimum(top / (6 * g[:, None]), 448.0)
        ts = tops / (6 * g[:, None])
        assert np.all(off_nearest(t, s, E4M3_GRID) <= 2 * (3 * u * t * (1 + 1e-6) + ts))
        step = s * g[:, None]
    step = np.repeat(step, blk, 1)
    live = step > 0
    y = np.where(live, np.abs(z) / np.where(live, step, 1), 0.0)
    ys = np.where(live, slack / np.where(live, step, 1), 0.0)
    off = off_nearest(np.minimum(y, 6.0), np.where(live, np.abs(v), 0.0), E2M1)
    assert np.all(off <= 2 * (3 * u * y * (1 + 1e-6) + ys))
    assert np.all((v == 0) | (np.sign(v) == np.sign(z)) | (np.abs(z) <= slack))
    assert np.all(v[~live] == 0)
