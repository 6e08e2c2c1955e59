"""Measured cases of the low-precision linear-layer operators.

Four operators, used one after another in a quantized linear layer:

* ``quantize_fp4``: rows to microscaled 4-bit floating point ("mxfp4": E2M1 codes, one power-of-two
  scale per 32; "nvfp4": E2M1 codes, one E4M3 scale per 16 and one fp32 scale per row), after the group
  Hadamard rotation when asked;
* ``rmsnorm_quantize``: residual addition, root-mean-square norm, rotation, and rows in 8 bits ("int8",
  one fp32 scale per row) or in either 4-bit format;
* ``matmul_fp4``: the product of two 4-bit operands;
* ``matmul_int8``: the product of 8-bit rows with INT8 weights (fp16 scale, optional zero-point per row).

``run`` computes them from elementary torch operations, or with ``own`` calls the package.  What is held
in 4 or 8 bits comes back as the values it stands for.
"""

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"fp32": 4, "fp16": 2, "bf16": 2}
FLOOR = 1e-30  # smallest per-row scale
ROTS = (0, 16, 32, 64, 128, 256, 512)
LARGEST = 4608 * 16384 * 4096  # multiply-adds of the largest product


# ------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # a projection's weight converted once, with the rotation the INT4 path uses
        dict(name="quantize_proj_mxfp4_rot256", op="quantize", rows=4096, k=4096, fmt="mxfp4", rot=256, dtype="fp16"),
        # the widest weight of the model
        dict(name="quantize_mlp_up_nvfp4_rot256", op="quantize", rows=16384, k=4096, fmt="nvfp4", rot=256, dtype="bf16"),
        # an odd layer: ragged rows and columns, no rotation, full-precision input
        dict(name="quantize_odd_nvfp4", op="quantize", rows=1001, k=1433, fmt="nvfp4", rot=0, dtype="fp32"),
        # one token between two layers: launch latency
        dict(name="norm_1_token_int8", op="norm", rows=1, k=4096, fmt="int8", rot=0, dtype="bf16", residual=True),
        # a whole image's tokens into a rotated 4-bit layer
        dict(name="norm_tokens_nvfp4_rot256", op="norm", rows=4608, k=4096, fmt="nvfp4", rot=256, dtype="bf16", residual=True),
        # a ragged batch into a rotated INT8 layer, no residual
        dict(name="norm_ragged_int8_rot64", op="norm", rows=777, k=5000, fmt="int8", rot=64, dtype="fp16", residual=False),
        # one token through the qkv projection: the weight's bytes
        dict(name="fp4_1_token_qkv", op="fp4", m=1, n=12288, k=4096, fmt="mxfp4", out="bf16", bias=True),
        # a few tokens and odd sizes
        dict(name="fp4_few_odd", op="fp4", m=19, n=1000, k=1433, fmt="nvfp4", out="fp16", bias=False),
        # a whole image's tokens through the widest layer: the largest
        dict(name="fp4_tokens_mlp_up", op="fp4", m=4608, n=16384, k=4096, fmt="nvfp4", out="bf16", bias=True),
        # a batch of a few hundred rows through the down projection
        dict(name="fp4_batch_mlp_down", op="fp4", m=300, n=4096, k=16384, fmt="mxfp4", out="bf16", bias=False),
        # one token through the INT8 down projection, asymmetric weights
        dict(name="int8_1_token_mlp_down", op="int8", m=1, n=4096, k=16384, asym=True, out="bf16", bias=True),
        # a whole image's tokens through the INT8 qkv projection
        dict(name="int8_tokens_qkv", op="int8", m=4608, n=12288, k=4096, asym=False, out="bf16", bias=False),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("quantize", "norm", "fp4", "int8"))
    if op in ("quantize", "norm"):
        k = _log(rng, 64, 16384)
        most = (16384 * 4096 if op == "quantize" else 4608 * 4096) // k
        case = dict(op=op, rows=_log(rng, 1, min(16384 if op == "quantize" else 8192, most)), k=k,
                    fmt=rng.choice(("mxfp4", "nvfp4") if op == "quantize" else ("int8", "mxfp4", "nvfp4")),
                    rot=rng.choice(ROTS), dtype=rng.choice(("fp32", "fp16", "bf16") if op == "quantize" else ("fp16", "bf16")))
        if op == "norm":
            case["residual"] = rng.random() < 0.5
        return case
    k, n = _log(rng, 64, 16384), _log(rng, 16, 16384)
    m = _log(rng, 1, max(1, min(8192, LARGEST // (k * n))))
    case = dict(op=op, m=m, n=n, k=k, out=rng.choice(("fp32", "fp16", "bf16")), bias=rng.random() < 0.5)
    if op == "fp4":
        case["fmt"] = rng.choice(("mxfp4", "nvfp4"))
    else:
        case["asym"] = rng.random() < 0.5
    return case


def _up(n, m):
    return -(-n // m) * m


def _kpad(case):
    """Columns held: whole rotation groups, and for the 4-bit formats whole runs of 32."""
    k = _up(case["k"], max(case.get("rot", 0), 1))
    return k if case.get("fmt") == "int8" or case["op"] == "int8" else _up(k, 32)


def _held(fmt, rows, kp):
    """Bytes of `rows` quantized rows."""
    if fmt == "int8":
        return rows * (kp + 4)
    return rows * kp // 2 + (rows * kp // 32 if fmt == "mxfp4" else rows * (kp // 16 + 4))


def work(case):
    kp = _kpad(case)
    if case["op"] in ("quantize", "norm"):
        rows, k, e = case["rows"], case["k"], SIZE[case["dtype"]]
        moved = rows * k * e + _held(case["fmt"], rows, kp) + rows * kp * 2  # input, quantized rows, their values in bf16
        flops = 6 * rows * kp + (rows * kp * int(math.log2(case["rot"])) if case["rot"] else 0)
        if case["op"] == "norm":
            moved += k * e + (2 * rows * k * e if case["residual"] else 0)
            flops += 5 * rows * k
        return {"bytes": moved, "flops": flops}
    m, n, k = case["m"], case["n"], case["k"]
    out = m * n * SIZE[case["out"]] + (n * 4 if case["bias"] else 0)
    if case["op"] == "fp4":
        return {"bytes": _held(case["fmt"], m, kp) + _held(case["fmt"], n, kp) + out, "flops": 2 * m * n * k}
    return {"bytes": m * (k + 4) + n * (k + 2 + case["asym"]) + out, "flops": 2 * m * n * k}


# ----------------------------------------------------------------------------------------- inputs
def _rows(g, rows, k, std, dtype):
    """Normal rows whose channels differ in scale, with a few outlier columns."""
    x = torch.randn(rows, k, device=DEV, generator=g) * std
    x *= torch.exp(0.5 * torch.randn(k, device=DEV, generator=g))
    n = max(1, k // 1000)
    x[:, torch.randint(0, k, (n,), device=DEV, generator=g)] *= 20.0
    return x.to(DTYPES[dtype])


def _padded(codes):
    """Codes in rows whose pitch is a multiple of 16 bytes, as the quantizers return them."""
    rows, k = codes.shape
    buf = torch.zeros(rows, _up(k, 16), dtype=codes.dtype, device=DEV)
    buf[:, :k] = codes
    return buf[:, :k]


def _fp4_operand(x, fmt):
    """A 4-bit operand as the quantizer holds it: packed codes, tiled scale bytes, row scales."""
    value, scale, row = _fp4(torch.nn.functional.pad(x, (0, _up(x.shape[1], 32) - x.shape[1])), fmt)
    code = (value.abs() * 2).to(torch.int64)  # 0, 1, 2, 3, 4, 6, 8, 12
    code = torch.tensor([0, 1, 2, 3, 4, 0, 5, 0, 6, 0, 0, 0, 7], device=DEV)[code] + 8 * (value < 0)
    code = code.to(torch.uint8)
    packed = code[:, 0::2] | (code[:, 1::2] << 4)
    if fmt == "mxfp4":
        byte = (torch.log2(scale) + 127).round().to(torch.uint8)
    else:
        byte = scale.to(torch.float8_e4m3fn).view(torch.uint8)
    return dict(packed=packed.contiguous(), scales=_tile(byte), row_scale=row)


def _tile(byte):
    """Row-major scale bytes [rows, blocks] -> [rows/128, blocks/4, 32, 4, 4]: 512-byte tiles of 128 rows x 4 blocks."""
    r, b = byte.shape
    t = torch.zeros(_up(r, 128), _up(b, 4), dtype=torch.uint8, device=DEV)
    t[:r, :b] = byte
    return t.view(t.shape[0] // 128, 4, 32, t.shape[1] // 4, 4).permute(0, 3, 2, 1, 4).contiguous()


def _untile(tiled, rows, blocks):
    a, b = tiled.shape[:2]
    return tiled.permute(0, 3, 2, 1, 4).reshape(a * 128, b * 4)[:rows, :blocks]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    s = dict(case=case)
    if case["op"] == "quantize":
        s["x"] = _rows(g, case["rows"], case["k"], 0.02, case["dtype"])
        return s
    if case["op"] == "norm":
        s["x"] = _rows(g, case["rows"], case["k"], 1.0, case["dtype"])
        s["weight"] = (1 + 0.1 * torch.randn(case["k"], device=DEV, generator=g)).to(DTYPES[case["dtype"]])
        s["residual"] = _rows(g, case["rows"], case["k"], 2.0, case["dtype"]) if case["residual"] else None
        return s
    m, n, k = case["m"], case["n"], case["k"]
    s["bias"] = torch.randn(n, device=DEV, generator=g) if case["bias"] else None
    if case["op"] == "fp4":
        s["a"] = _fp4_operand(_rows(g, m, k, 1.0, "fp32"), case["fmt"])
        s["b"] = _fp4_operand(_rows(g, n, k, 0.02, "fp32"), case["fmt"])
        return s
    codes = _padded((torch.randn(m, k, device=DEV, generator=g) * 30).round().clamp(-127, 127).to(torch.int8))
    s["codes"], s["sums"] = codes, codes.sum(1, dtype=torch.int32)
    s["scales"] = torch.rand(m, 1, device=DEV, generator=g) * 0.05 + 0.01
    s["w_codes"] = _padded((torch.randn(n, k, device=DEV, generator=g) * 35).round().clamp(-128, 127).to(torch.int8))
    s["w_scales"] = (torch.rand(n, 1, device=DEV, generator=g) * 5e-4 + 1e-4).to(torch.float16)
    s["w_zero_points"] = torch.randint(-20, 21, (n, 1), device=DEV, generator=g).to(torch.int8) if case["asym"] else None
    return s


# ------------------------------------------------------------------------------------ plain forms
def _rotate(x, rot):
    """Group Hadamard of the last dimension in fp32 butterflies, lowest digit first: H4 factors when
    `rot` is a power of four, H2 factors otherwise, and the normalisation once at the end."""
    rows, k = x.shape
    four = rot & 0x55555555 == rot
    st = 1
    while st < rot:
        r = 4 if four else 2
        x = x.view(rows, k // (r * st), r, st)
        if four:
            a, b, c, d = x.unbind(2)
            p, m, q, w = a + b, a - b, c + d, c - d
            x = torch.stack((p + w, p - w, m + q, q - m), 2)
        else:
            a, b = x.unbind(2)
            x = torch.stack((a + b, a - b), 2)
        x = x.view(rows, k)
        st *= r
    return x * float(1 / math.sqrt(rot))


def _e2m1(y):
    """Nearest E2M1 value, ties to the even code, saturating at 6."""
    a = y.abs()
    r = torch.where(a < 2, torch.round(a * 2) / 2, torch.where(a < 4, torch.round(a), torch.round(a / 2) * 2))
    return torch.copysign(r.clamp(max=6.0), y)


def _fp4(x, fmt):
    """fp32 rows -> (E2M1 values, block scales, row scales or None); their product is what the codes stand for."""
    rows, k = x.shape
    if fmt == "mxfp4":
        b = x.view(rows, k // 32, 32)
        e = (torch.frexp(b.abs().amax(2)).exponent - 3).clamp(-127, 127)
        e = torch.where(b.abs().amax(2) > 0, e, -127)
        scale = torch.exp2(e.float())
        return _e2m1(b * torch.exp2(-e.float()).unsqueeze(2)).view(rows, k), scale, None
    b = x.view(rows, k // 16, 16)
    amax = b.abs().amax(2)
    g = (amax.amax(1, keepdim=True) * (1.0 / 2688.0)).clamp(min=FLOOR)
    scale = (amax * (1.0 / (6.0 * g))).clamp(max=448.0).to(torch.float8_e4m3fn).float()
    inv = torch.where(scale > 0, 1.0 / (scale * g), 0.0)
    return _e2m1(b * inv.unsqueeze(2)).view(rows, k), scale, g.squeeze(1)


def _values(value, scale, row):
    rows, k = value.shape
    v = (value.view(rows, scale.shape[1], -1) * scale.unsqueeze(2)).view(rows, k)
    return v if row is None else v * row.unsqueeze(1)


def _quantized(y, case):
    """The outputs of quantizing fp32 rows."""
    kp = _kpad(case)
    y = torch.nn.functional.pad(y, (0, kp - y.shape[1]))
    if case["rot"]:
        y = _rotate(y, case["rot"])
    if case["fmt"] != "int8":
        value, scale, row = _fp4(y, case["fmt"])
        out = {"values": _values(value, scale, row).to(torch.bfloat16)}
        return out if row is None else out | {"row_scale": row}
    s = (y.abs().amax(1, keepdim=True) * (1.0 / 127.0)).clamp(min=FLOOR)
    q = y * (1.0 / s)
    q = torch.where(q >= 0, torch.floor(q + 0.5), torch.ceil(q - 0.5)).clamp(-128, 127)
    return {"values": (q * s).to(torch.bfloat16), "scales": s}


def _plain_fp4_values(p, fmt):
    packed = p["packed"]
    rows, k = packed.shape[0], packed.shape[1] * 2
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], device=DEV)
    code = torch.stack((packed & 15, packed >> 4), 2).view(rows, k)
    byte = _untile(p["scales"], rows, k // (32 if fmt == "mxfp4" else 16))
    scale = torch.exp2(byte.float() - 127) if fmt == "mxfp4" else byte.contiguous().view(torch.float8_e4m3fn).float()
    return _values(table[code.int()], scale, p["row_scale"])


def _plain(s):
    case = s["case"]
    if case["op"] == "quantize":
        return _quantized(s["x"].float(), case)
    if case["op"] == "norm":
        h = s["x"].float()
        out = {}
        if s["residual"] is not None:
            h = h + s["residual"].float()
            out["residual"] = h.to(s["x"].dtype)
        # the sum in 64 bits: a code next to a rounding border goes by the norm's last bit
        rstd = (1.0 / torch.sqrt((h.double() ** 2).mean(1, keepdim=True) + 1e-6)).float()
        return out | _quantized(h * rstd * s["weight"].float(), case)
    if case["op"] == "fp4":
        y = _plain_fp4_values(s["a"], case["fmt"]) @ _plain_fp4_values(s["b"], case["fmt"]).T
    else:
        w = s["w_codes"].float()
        if s["w_zero_points"] is not None:
            w = w - s["w_zero_points"].float()
        y = (s["codes"].float() @ w.T) * s["scales"] * s["w_scales"].float().T
    if s["bias"] is not None:
        y = y + s["bias"]
    return {"y": y.to(DTYPES[case["out"]])}


# -------------------------------------------------------------------------------------- own calls
def _own(s):
    import int_crush_converter_b200 as B
    case = s["case"]
    if case["op"] == "quantize":
        q = B.quantize_fp4(s["x"], case["fmt"], rot_size=case["rot"])
        out = {"values": B.dequantize_fp4(q, torch.bfloat16)}
        return out if q.row_scale is None else out | {"row_scale": q.row_scale}
    if case["op"] == "norm":
        q, residual = B.rmsnorm_quantize(s["x"], s["weight"], residual=s["residual"], eps=1e-6, fmt=case["fmt"],
                                         rot_size=case["rot"])
        out = {} if residual is None else {"residual": residual}
        if case["fmt"] == "int8":
            return out | {"values": B.dequantize_int8(q, torch.bfloat16), "scales": q.scales}
        out["values"] = B.dequantize_fp4(q, torch.bfloat16)
        return out if q.row_scale is None else out | {"row_scale": q.row_scale}
    if case["op"] == "fp4":
        a, b = (B.FP4Tensor(p["packed"], p["scales"], p["row_scale"], case["fmt"]) for p in (s["a"], s["b"]))
        return {"y": B.matmul_fp4(a, b, bias=s["bias"], out_dtype=DTYPES[case["out"]])}
    a = B.Int8Rows(s["codes"], s["scales"], s["sums"])
    return {"y": B.matmul_int8(a, s["w_codes"], s["w_scales"], s["w_zero_points"], bias=s["bias"],
                               out_dtype=DTYPES[case["out"]])}


def run(state):
    if own:
        return _own(state)
    return _plain(state)


# -------------------------------------------------------------------------- definitions in 64 bits
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _exact_hadamard(rot):
    four = rot in (4, 16, 64, 256, 1024)
    base = torch.tensor([[1, 1, 1, -1], [1, 1, -1, 1], [1, -1, 1, 1], [-1, 1, 1, 1]] if four else [[1, 1], [1, -1]],
                        dtype=torch.float64, device=DEV)
    h = torch.ones(1, 1, dtype=torch.float64, device=DEV)
    while h.shape[0] < rot:
        h = torch.kron(h, base)
    return h / math.sqrt(rot)


def _exact_nearest(y):
    """Nearest entry of E2M1 by its borders; a border itself goes to the even entry."""
    grid = torch.tensor(E2M1, dtype=torch.float64, device=DEV)
    mid = (grid[1:] + grid[:-1]) / 2
    a = y.abs().contiguous()
    low, high = torch.searchsorted(mid, a), torch.searchsorted(mid, a, right=True)
    return torch.sign(y) * grid[torch.where(low % 2 == 0, low, high)]


def _exact_fp4(y, fmt):
    rows, k = y.shape
    size = 32 if fmt == "mxfp4" else 16
    b = y.reshape(rows, -1, size)
    top = b.abs().amax(2, keepdim=True)
    if fmt == "mxfp4":
        step = torch.exp2((torch.floor(torch.log2(top)) - 2).clamp(-127, 127))
        return (_exact_nearest(b / step) * step).reshape(rows, k), None
    row = (y.abs().amax(1) / (6 * 448)).clamp(min=FLOOR)
    g = row.view(rows, 1, 1)
    t = (top / (6 * g)).clamp(max=448)
    ulp = torch.exp2((torch.floor(torch.log2(t)) - 3).clamp(min=-9))  # E4M3: 4 significant bits, smallest step 2^-9
    step = torch.round(t / ulp) * ulp * g
    v = torch.where(step > 0, _exact_nearest(b / torch.where(step > 0, step, 1.0)) * step, 0.0)
    return v.reshape(rows, k), row


def _exact_quantized(y, case):
    kp = _kpad(case)
    z = torch.zeros(y.shape[0], kp, dtype=torch.float64, device=DEV)
    z[:, :y.shape[1]] = y
    if case["rot"]:
        z = (z.reshape(-1, case["rot"]) @ _exact_hadamard(case["rot"]).T).reshape(y.shape[0], kp)
    if case["fmt"] != "int8":
        v, row = _exact_fp4(z, case["fmt"])
        return {"values": v} if row is None else {"values": v, "row_scale": row}
    s = (z.abs().amax(1, keepdim=True) / 127).clamp(min=FLOOR)
    q = torch.sign(z) * torch.floor((z / s).abs() + 0.5)
    return {"values": q * s, "scales": s}


def _exact_operand(p, fmt):
    packed = p["packed"].long()
    rows, k = packed.shape[0], packed.shape[1] * 2
    code = torch.empty(rows, k, dtype=torch.int64, device=DEV)
    code[:, 0::2], code[:, 1::2] = packed % 16, packed // 16
    v = torch.tensor(E2M1 + [-x for x in E2M1], dtype=torch.float64, device=DEV)[code]
    size = 32 if fmt == "mxfp4" else 16
    r = torch.arange(rows, device=DEV).unsqueeze(1)
    c = torch.arange(k // size, device=DEV).unsqueeze(0)
    byte = p["scales"][r // 128, c // 4, r % 32, r % 128 // 32, c % 4].long()
    if fmt == "mxfp4":
        scale = torch.exp2(byte.double() - 127)
    else:
        e, m = byte // 8, (byte % 8).double()
        scale = torch.where(e > 0, (1 + m / 8) * torch.exp2(e.double() - 7), m * 2.0 ** -9)
    v = v * scale.repeat_interleave(size, 1)
    return v if p["row_scale"] is None else v * p["row_scale"].double().unsqueeze(1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quantize":
        return _exact_quantized(s["x"].double(), case)
    if case["op"] == "norm":
        h, out = s["x"].double(), {}
        if s["residual"] is not None:
            h = h + s["residual"].double()
            out["residual"] = h
        y = h / torch.sqrt(h.square().sum(1, keepdim=True) / h.shape[1] + 1e-6) * s["weight"].double()
        return out | _exact_quantized(y, case)
    if case["op"] == "fp4":
        y = _exact_operand(s["a"], case["fmt"]) @ _exact_operand(s["b"], case["fmt"]).T
    else:
        w = s["w_codes"].double() * s["w_scales"].double()
        if s["w_zero_points"] is not None:
            w = w - s["w_zero_points"].double() * s["w_scales"].double()
        y = (s["codes"].double() * s["scales"].double()) @ w.T
    return {"y": y if s["bias"] is None else y + s["bias"].double()}
