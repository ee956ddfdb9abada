"""Cases of the 4-bit microscaled operators: quantisation, expansion, product, gated product and MLP.

A matrix of 4-bit values [rows, k] is held as

* codes: row r at r * 16 * ceil(k / 32) bytes, value i in the low (even i) or high (odd i) half of byte i / 2,
  each the sign and index of one of 0, 0.5, 1, 1.5, 2, 3, 4, 6; values behind k are zero;
* scales: one byte for each block of 32 values ("mx": a power of two, 2^(byte - 127)) or 16 values ("nv": an 8-bit
  float with 4 exponent and 3 mantissa bits, times the tensor's own scale, a power of two), in tiles of 128 rows by
  4 blocks: the byte of row r and block b is at (r % 32) * 16 + (r % 128 / 32) * 4 + b % 4 of tile (r / 128, b / 4),
  and the tiles of one 128 rows follow each other.
"""
import math

import torch

own = False

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
BLOCK = {"mx": 32, "nv": 16}
VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
# the tensors' own scales of the "nv" format: activations up to 42, weights up to 0.65
X_SCALE = {"mx": 1.0, "nv": 2.0 ** -6}
W_SCALE = {"mx": 1.0, "nv": 2.0 ** -12}


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one token's activations to 4 bits and back: the smallest call
        dict(name="quant_nv_token", op="roundtrip", fmt="nv", m=1, k=1024, x="f32", y="f32", pad=0),
        # the activations of a full batch of patches (65,536 tokens of the 1024-wide model)
        dict(name="quant_mx_batch", op="roundtrip", fmt="mx", m=65536, k=1024, x="bf16", y="bf16", pad=0),
        # rows of an odd width that sit in a wider buffer
        dict(name="quant_nv_odd", op="roundtrip", fmt="nv", m=4099, k=1001, x="f16", y="f16", pad=7),
        # a stored layer back to 16 bits (the 1024-wide model's gate and up rows)
        dict(name="expand_mx_layer", op="expand", fmt="mx", m=8192, k=1024, x="f32", y="bf16", pad=0),
        # one token through a square layer
        dict(name="linear_mx_token", op="linear", fmt="mx", m=1, n=4096, k=4096, x="bf16", y="bf16", bias=False, pad=0),
        # q, k and v of a single forecast (context 512, horizon 96) of the 512-wide model
        dict(name="linear_nv_forecast", op="linear", fmt="nv", m=19, n=1536, k=512, x="f32", y="f32", bias=True, pad=0),
        # sizes that end inside every tile
        dict(name="linear_nv_odd", op="linear", fmt="nv", m=333, n=1001, k=1000, x="f16", y="f16", bias=True, pad=8),
        # attention's output projection over a batch of series of the 1024-wide model
        dict(name="linear_mx_batch", op="linear", fmt="mx", m=65536, n=1024, k=1024, x="bf16", y="f32", bias=True, pad=0),
        # the largest product
        dict(name="linear_nv_large", op="linear", fmt="nv", m=8192, n=8192, k=8192, x="bf16", y="bf16", bias=False, pad=0),
        # the gated half of the 512-wide model's MLP, its result used in 16 bits
        dict(name="glu_mx_series", op="glu", fmt="mx", m=1072, n=2048, k=512, x="f32", y="bf16", bias=True, pad=0),
        # the whole MLP of a single forecast, 1024-wide model
        dict(name="mlp_nv_forecast", op="mlp", fmt="nv", m=19, n=4096, k=1024, x="f32", y="bf16", bias=True, pad=0),
        # and of a batch of series
        dict(name="mlp_mx_batch", op="mlp", fmt="mx", m=32768, n=4096, k=1024, x="bf16", y="bf16", bias=True, pad=0),
    ]


def draw(rng):
    def size(lo, hi):
        v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
        if rng.random() < 0.5:  # half of the sizes are the round ones of real layers
            unit = 256 if v >= 512 else 32 if v >= 64 else 1
            v = max(lo, v // unit * unit)
        return min(hi, v)

    op = rng.choice(("roundtrip", "expand", "linear", "linear", "glu", "mlp"))
    c = dict(op=op, fmt=rng.choice(("mx", "nv")), m=size(1, 65536), k=size(16, 8192), x=rng.choice(("f32", "f16", "bf16")),
             pad=rng.choice((0, 0, 1, 8)))
    if op in ("roundtrip", "expand"):
        c["m"] = max(1, min(c["m"], (1 << 26) // c["k"]))
        c["y"] = rng.choice(("f32", "f16", "bf16"))
        return c
    c["n"] = size(16, 8192)
    c["bias"] = rng.random() < 0.5
    c["m"] = max(1, min(c["m"], (1 << 37) // (c["n"] * c["k"]), (1 << 27) // max(c["n"], c["k"])))
    # results in 32 bits follow short sums (the models' own layers); long ones and those through 4-bit
    # hidden values are used in 16 bits
    c["y"] = rng.choice(("f32", "f16", "bf16") if c["k"] <= 1024 and op != "mlp" else ("f16", "bf16"))
    return c


def work(case):
    m, k, fmt = case["m"], case["k"], case["fmt"]
    held = lambda rows, cols: rows * (-(-cols // 2) + -(-cols // BLOCK[fmt]))  # noqa: E731
    x = m * k * SIZE[case["x"]]
    if case["op"] == "roundtrip":  # x, its 4-bit form, and what that stands for
        return {"bytes": x + held(m, k) + m * k * SIZE[case["y"]], "flops": 0}
    if case["op"] == "expand":
        return {"bytes": held(m, k) + m * k * SIZE[case["y"]], "flops": 0}
    n = case["n"]
    if case["op"] == "linear":
        return {"bytes": x + held(n, k) + 4 * n * case["bias"] + m * n * SIZE[case["y"]], "flops": 2 * m * n * k}
    if case["op"] == "glu":
        return {"bytes": x + held(2 * n, k) + 8 * n * case["bias"] + m * n * SIZE[case["y"]], "flops": 4 * m * n * k}
    return {"bytes": x + held(2 * n, k) + held(k, n) + (8 * n + 4 * k) * case["bias"] + m * k * SIZE[case["y"]],
            "flops": 6 * m * n * k}


# ------------------------------------------------------------------ the inputs
def _inputs(case, seed):
    """The floating-point inputs: activations as they leave a norm (a few wide channels, some empty rows of padding
    tokens), weights and biases of small deviation."""
    g = torch.Generator(device=DEV).manual_seed(seed * 1000003 + case["m"] * 131 + case["k"])
    rnd = lambda *s: torch.randn(s, device=DEV, generator=g)  # noqa: E731
    m, k = case["m"], case["k"]
    if case["op"] == "expand":
        return {"w": [rnd(m, k) * 0.02]}
    x = rnd(m, k + case["pad"])
    x *= 1 + 3 * (torch.rand(k + case["pad"], device=DEV, generator=g) < 0.02)
    if m >= 16:
        x *= (torch.rand((m, 1), device=DEV, generator=g) >= 0.02)
    x = x.to(TYPES[case["x"]])[:, :k]
    if case["op"] == "roundtrip":
        return {"x": x}
    n = case["n"]
    shapes = {"linear": [(n, k)], "glu": [(2 * n, k)], "mlp": [(2 * n, k), (k, n)]}[case["op"]]
    return {"x": x, "w": [rnd(*s) * 0.02 for s in shapes], "b": [rnd(s[0]) * 0.02 if case["bias"] else None for s in shapes]}


def _widths(case):
    """Rows and values of the result."""
    return case["m"], case["n"] if case["op"] in ("linear", "glu") else case["k"]


def prepare(case, seed):
    inp, fmt, m, k = _inputs(case, seed), case["fmt"], case["m"], case["k"]
    s = dict(case, input=inp.get("x"), bias=inp.get("b", []), weights=[_pack(w, fmt, W_SCALE[fmt]) for w in inp.get("w", [])])
    # the result's buffer, and those of the 4-bit activations and hidden values, kept from call to call
    s["out"] = torch.empty(_widths(case), dtype=TYPES[case["y"]], device=DEV)
    if own:
        from t0_web_b200 import fp4
        s["engine"] = _engine()
        s["w"] = [fp4.Fp4Matrix(fmt, w["rows"], w["k"], w["codes"], w["scales"], W_SCALE[fmt]) for w in s["weights"]]
        s["xq"] = fp4.Fp4Matrix.empty(fmt, m, k, DEV, X_SCALE[fmt])
        s["zq"] = fp4.Fp4Matrix.empty(fmt, m, case["n"], DEV, X_SCALE[fmt]) if case["op"] == "mlp" else None
    return s


_engines = []


def _engine():
    if not _engines:
        from t0_web_b200 import t0_fast
        _engines.append(t0_fast.Engine(0))
    return _engines[0]


# ------------------------------------------------------------------ the plain forms
def _blocks(x, fmt):
    """x [rows, k] in 32 bits as [rows, blocks, block], zeros behind k."""
    rows, k = x.shape
    b = BLOCK[fmt]
    nb = -(-k // b)
    return torch.nn.functional.pad(x.float(), (0, nb * b - k)).view(rows, nb, b)


def _round(x, fmt, tensor_scale):
    """x -> the blocks' scale bytes [rows, blocks], their values and the rounded quotients [rows, blocks, block].
    Each product and quotient that decides a rounding is exact or correctly rounded in 32 bits: the divisors have
    at most four significant bits."""
    u = _blocks(x, fmt)
    amax = u.abs().amax(2)
    if fmt == "mx":  # the largest power of two that leaves the block's largest value at 4 or above
        e = torch.where(amax > 0, torch.frexp(amax).exponent + (127 - 3), torch.zeros_like(amax, dtype=torch.int32)).clamp(0, 254)
        byte = e.to(torch.uint8)
        scale = torch.ldexp(torch.ones_like(amax), e - 127)
    else:
        s8 = (amax / (6 * tensor_scale)).clamp(max=448.0).to(torch.float8_e4m3fn)
        byte = s8.view(torch.uint8)
        scale = s8.float() * tensor_scale
    q = u / torch.where(scale > 0, scale, torch.ones_like(scale))[:, :, None]
    q = torch.where(scale[:, :, None] > 0, q, torch.zeros_like(q))
    a = q.abs().clamp(max=6.0)
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return byte, scale, torch.copysign(torch.round(a / step) * step, q)


def _quantized(x, fmt, tensor_scale):
    """What x's 4-bit form stands for, in 32 bits."""
    _, scale, q = _round(x, fmt, tensor_scale)
    return (q * scale[:, :, None]).flatten(1)[:, :x.shape[1]]


def _pack(x, fmt, tensor_scale):
    """x's 4-bit form as it is held."""
    byte, _, q = _round(x, fmt, tensor_scale)
    rows, nb = byte.shape
    idx = torch.bucketize(q.abs(), torch.tensor(VALUES, device=x.device)).to(torch.uint8) | (q.signbit().to(torch.uint8) << 3)
    idx = torch.nn.functional.pad(idx.flatten(1), (0, -(nb * BLOCK[fmt]) % 32))
    codes = idx[:, 0::2] | (idx[:, 1::2] << 4)
    rt, kt = -(-rows // 128), -(-nb // 4)
    t = torch.nn.functional.pad(byte, (0, kt * 4 - nb, 0, rt * 128 - rows)).view(rt, 4, 32, kt, 4)
    return {"rows": rows, "k": x.shape[1], "codes": codes.contiguous(), "scales": t.permute(0, 3, 2, 1, 4).contiguous().flatten()}


def _unpack(w, fmt, tensor_scale):
    """The values of a held matrix, in 32 bits."""
    rows, k, b = w["rows"], w["k"], BLOCK[fmt]
    nb = -(-k // b)
    rt, kt = -(-rows // 128), -(-nb // 4)
    byte = w["scales"].view(rt, kt, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(rt * 128, kt * 4)[:rows, :nb]
    if fmt == "mx":
        scale = torch.ldexp(torch.ones(byte.shape, device=byte.device), byte.int() - 127)
    else:
        scale = byte.contiguous().view(torch.float8_e4m3fn).float() * tensor_scale
    lut = torch.tensor(VALUES + tuple(-v for v in VALUES), device=byte.device)
    v = torch.stack((lut[(w["codes"] & 15).int()], lut[(w["codes"] >> 4).int()]), 2).flatten(1)[:, :nb * b]
    return (v.view(rows, nb, b) * scale[:, :, None]).flatten(1)[:, :k]


def _plus(y, b):
    return y if b is None else y + b


def _gated(x, w, b):
    """silu(x . gate^T + bg) * (x . up^T + bu); the gate rows come first."""
    h = _plus(x @ w.T, b)
    gate, up = h.chunk(2, 1)
    return gate / (1 + torch.exp(-gate)) * up


def run(state):
    s = state
    op, fmt, x, y = s["op"], s["fmt"], s["input"], s["out"]
    if own:
        from t0_web_b200 import fp4
        e = s["engine"]
        if op == "roundtrip":
            fp4.quantize(e, x, s["xq"])
            fp4.dequantize(e, s["xq"], y)
        elif op == "expand":
            fp4.dequantize(e, s["w"][0], y)
        elif op == "linear":
            fp4.linear(e, s["w"][0], x, s["xq"], y, s["bias"][0])
        elif op == "glu":
            fp4.quantize(e, x, s["xq"])
            fp4.glu(e, s["w"][0], s["xq"], y, s["bias"][0])
        else:
            fp4.mlp(e, s["w"][0], s["w"][1], x, s["xq"], s["zq"], y, s["bias"][0], s["bias"][1])
        return y
    if op == "roundtrip":
        return _quantized(x, fmt, X_SCALE[fmt]).to(y.dtype)
    w = [_unpack(v, fmt, W_SCALE[fmt]) for v in s["weights"]]
    if op == "expand":
        return w[0].to(y.dtype)
    xq = _quantized(x, fmt, X_SCALE[fmt])
    if op == "linear":
        return _plus(xq @ w[0].T, s["bias"][0]).to(y.dtype)
    z = _gated(xq, w[0], s["bias"][0])
    if op == "glu":
        return z.to(y.dtype)
    return _plus(_quantized(z, fmt, X_SCALE[fmt]) @ w[1].T, s["bias"][1]).to(y.dtype)


# ------------------------------------------------------------------ from the definition, in 64 bits
def _nearest(a, grid):
    """For each of a >= 0 the nearest entry of the ascending grid, at equal distance the one of even index."""
    grid = torch.tensor(grid, dtype=torch.float64, device=a.device)
    mid = (grid[1:] + grid[:-1]) / 2
    below, upto = torch.searchsorted(mid, a, right=False), torch.searchsorted(mid, a, right=True)
    return grid[torch.where(below % 2 == 0, below, upto)]


def _exact4(x, fmt, tensor_scale):
    x = x.double()
    out = torch.zeros_like(x)
    b = BLOCK[fmt]
    whole = x.shape[1] // b * b
    for part, width in ((slice(0, whole), b), (slice(whole, None), x.shape[1] - whole)):
        v = x[:, part]
        if not v.numel():
            continue
        v = v.reshape(x.shape[0], -1, width)
        top = v.abs().amax(2, keepdim=True)
        if fmt == "mx":
            s = torch.exp2(torch.floor(torch.log2(torch.where(top > 0, top, 1.0))) - 2)
            s = torch.where(top < s * 4, s / 2, torch.where(top >= s * 8, s * 2, s)).clamp(min=2.0 ** -127)
        else:
            eights = [i / 8 * 2.0 ** -6 for i in range(8)] + [(1 + i / 8) * 2.0 ** e for e in range(-6, 9) for i in range(8)][:-1]
            s = _nearest(top / (6 * tensor_scale), eights) * tensor_scale
        q = torch.where(s > 0, v.abs() / torch.where(s > 0, s, 1.0), 0.0)
        out[:, part] = (_nearest(q, VALUES) * s * v.sign()).reshape(x.shape[0], -1)
    return out


def exact(case, seed):
    inp, fmt = _inputs(case, seed), case["fmt"]
    if case["op"] == "roundtrip":
        return _exact4(inp["x"], fmt, X_SCALE[fmt])
    w = [_exact4(v, fmt, W_SCALE[fmt]) for v in inp["w"]]
    if case["op"] == "expand":
        return w[0]
    y = _exact4(inp["x"], fmt, X_SCALE[fmt])
    for i, (v, b) in enumerate(zip(w, inp["b"])):
        y = y @ v.T + (0 if b is None else b.double())
        if case["op"] != "linear" and i == 0:
            n = case["n"]
            y = y[:, :n] * torch.sigmoid(y[:, :n]) * y[:, n:]
            if case["op"] == "mlp":
                y = _exact4(y, fmt, X_SCALE[fmt])
    return y
