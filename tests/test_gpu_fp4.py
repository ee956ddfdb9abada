"""4-bit microscaled operators on the GPU against 64-bit restatements.

Quantisation and expansion are compared bit for bit: every rounding is decided
exactly.  A product y = sum_k x_k w_k of 4-bit values accumulates in f32; each
of its ceil(K / 64) accumulation steps may lose up to four units of 2^-23 of
the largest partial sum, which sum_k |x_k w_k| bounds, and each join of partial
sums one more (at most 16 of them): |y - ref| <= (4 ceil(K / 64) + 16) 2^-23
sum|xw|, plus half a step of the output type (2^-24, 2^-11, 2^-8 relative, and
half the smallest float16 subnormal, 2^-25).  A gated product adds d(silu) <=
1.1 dg, |silu(g)| <= |g| and 8 units of 2^-24 for exp, quotient and products.
"""
import os
import subprocess
import sys
import threading

import numpy as np
import pytest
import torch

import fp4_oracle as O
from t0_web_b200 import fp4
from t0_web_b200._lib import T0bError

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
FMT = ["mx", "nv"]
TS = {"mx": 1.0, "nv": 2.0 ** -6}


def mat_from(x, fmt, ts=None):
    """A device matrix of the oracle's quantisation of x, and its values."""
    ts = TS[fmt] if ts is None else ts
    byte, code = O.quantize(x, fmt, ts)
    c, s = O.pack(byte, code, fmt)
    m = fp4.Fp4Matrix(fmt, *x.shape, torch.from_numpy(c).to(DEV), torch.from_numpy(s).to(DEV), ts)
    return m, O.values(byte, code, fmt, ts)


def empty(fmt, rows, k, ts=None):
    """Memory filled with 0xFF (NaN scales), so that an unwritten byte shows."""
    m = fp4.Fp4Matrix.empty(fmt, rows, k, DEV, TS[fmt] if ts is None else ts)
    m.codes.fill_(255)
    m.scales.fill_(255)
    return m


def rnd(seed, *shape, dev=1.0):
    return np.random.default_rng(seed).standard_normal(shape) * dev


def sum_bound(x, w, ts=1.0):
    k = x.shape[1]
    return (4 * -(-k // 64) + 16) * 2.0 ** -23 * (np.abs(x) @ np.abs(w).T)


def out_bound(ref, y):
    return HALF_STEP[y] * np.abs(ref) + (2.0 ** -25 if y == "f16" else 0)


def check_close(got, ref, bound):
    got = got.double().cpu().numpy()
    worst = np.max(np.abs(got - ref) - bound)
    assert worst <= 0, f"off by {worst:.3e} more than the bound, at {np.unravel_index(np.argmax(np.abs(got - ref) - bound), ref.shape)}"


def check_matrix(m, x):
    byte, code = O.quantize(x, m.format, m.tensor_scale)
    c, s = O.pack(byte, code, m.format)
    gs, gc = m.scales.cpu().numpy(), m.codes.cpu().numpy()
    nan = O.unpack(c, s, m.rows, m.k, m.format)[0] == (255 if m.format == "mx" else 127)
    assert np.array_equal(gs, s)
    if nan.any():  # codes of a NaN block say nothing
        live = ~np.repeat(nan, O.BLOCK[m.format], 1)[:, :m.k]
        assert np.array_equal(O.unpack(gc, gs, m.rows, m.k, m.format)[1][live], code[live])
    else:
        assert np.array_equal(gc, c)


# ------------------------------------------------------------ quantisation
@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("ty", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,k,pad,shift", [(1, 1, 0, 0), (1, 1024, 0, 0), (3, 15, 0, 0), (5, 17, 3, 1), (128, 64, 0, 0),
                                              (129, 65, 0, 0), (33, 1001, 7, 0), (300, 512, 8, 8), (257, 256, 1, 0), (2, 8192, 0, 0),
                                              (140, 100, 0, 0), (33, 128, 4, 0)])
def test_quantize(engine, fmt, ty, rows, k, pad, shift):
    buf = torch.from_numpy(rnd(rows * 7 + k, rows * (k + pad) + shift, dev=3.0)).to(DT[ty]).to(DEV)
    x = buf[shift:].view(rows, k + pad)[:, :k]
    m = fp4.quantize(engine, x, empty(fmt, rows, k))
    fp4.sync(engine)
    check_matrix(m, x.double().cpu().numpy())


def edge_blocks(fmt, ts):
    """Rows of one block each: ties, borders one step off them, empty, tiny, huge and non-finite values."""
    b = O.BLOCK[fmt]
    mids = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    rows = []
    for s in (1.0, 1.125, 1.5, 1.875, 2.0 ** -9, 3 * 2.0 ** -9, 448.0):
        if fmt == "mx":
            s = 2.0 ** round(np.log2(s))
        d = np.float32(s * ts)
        for f in (lambda v: v, lambda v: np.nextafter(v, np.float32(0)), lambda v: np.nextafter(v, np.float32(1e38))):
            r = np.zeros(b, np.float32)
            r[:7] = f((mids * d).astype(np.float32))
            r[7:14] = -r[:7]
            r[14] = 6 * d if fmt == "nv" else 4 * d
            rows.append(r)
    if fmt == "nv":  # borders of the scale itself
        for i in range(0, 126):
            mid = np.float32((O.E4M3[i] + O.E4M3[i + 1]) / 2 * 6 * ts)
            for a in (mid, np.nextafter(mid, np.float32(0)), np.nextafter(mid, np.float32(1e38))):
                r = np.zeros(b, np.float32)
                r[3], r[5] = -a, a / 3
                rows.append(r)
    else:
        for e in range(-126, 128):
            for a in (np.float32(2.0 ** e), np.nextafter(np.float32(2.0 ** e), np.float32(0))):
                r = np.zeros(b, np.float32)
                r[b - 1], r[0] = a, -a / 5
                rows.append(r)
    for a in (0.0, -0.0, 1e-45, 1e-40, 1.1754944e-38, 2.0 ** -126, 1e-30, 3e38, 3.4028235e38, -3.4028235e38, np.inf, -np.inf, np.nan):
        r = np.zeros(b, np.float32)
        r[b // 2], r[1] = a, a / 2
        rows.append(r)
    r = np.full(b, 1.0, np.float32)
    r[-1] = np.nan
    rows += [r, np.full(b, -6.0, np.float32)]
    return np.stack(rows)


@pytest.mark.parametrize("fmt,ts", [("mx", 1.0), ("nv", 1.0), ("nv", 2.0 ** -64), ("nv", 2.0 ** -6), ("nv", 2.0 ** 64)])
def test_quantize_edges(engine, fmt, ts):
    x = edge_blocks(fmt, ts)
    m = fp4.quantize(engine, torch.from_numpy(x).to(DEV), empty(fmt, *x.shape, ts=ts))
    check_matrix(m, x)
    wide = x[:-(len(x) % 4) or None].reshape(-1, 4 * x.shape[1])  # several blocks a row
    m = fp4.quantize(engine, torch.from_numpy(wide).to(DEV), empty(fmt, *wide.shape, ts=ts))
    check_matrix(m, wide)


@pytest.mark.parametrize("ty", ["f16", "bf16"])
@pytest.mark.parametrize("fmt", FMT)
def test_quantize_every_16_bit_value(engine, ty, fmt):
    v = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(DT[ty]).view(1024, 64).to(DEV)
    perm = torch.from_numpy(np.random.default_rng(3).permutation(65536)).to(DEV)
    for x in (v, v.flatten()[perm].view(1024, 64)):
        m = fp4.quantize(engine, x, empty(fmt, 1024, 64))
        check_matrix(m, x.double().cpu().numpy())


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("ty", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,k,pad", [(1, 1, 0), (1, 1024, 0), (7, 33, 2), (130, 1001, 1), (129, 256, 8), (64, 48, 0), (140, 100, 3),
                                        (33, 128, 0)])
def test_dequantize(engine, fmt, ty, rows, k, pad):
    m, v = mat_from(rnd(rows + k, rows, k), fmt)
    y = torch.full((rows, k + pad), 77.0, dtype=DT[ty], device=DEV)
    fp4.dequantize(engine, m, y[:, :k])
    got = y.cpu()
    assert torch.equal(got[:, :k], torch.from_numpy(v).to(DT[ty]))
    assert bool((got[:, k:] == 77).all())


@pytest.mark.parametrize("fmt", FMT)
def test_dequantize_every_byte(engine, fmt):
    b = O.BLOCK[fmt]
    byte = np.arange(256, dtype=np.uint8)[:, None] if fmt == "mx" else np.arange(128, dtype=np.uint8)[:, None]
    code = np.tile(np.arange(16, dtype=np.uint8), (len(byte), b // 16))
    c, s = O.pack(byte, code, fmt)
    m = fp4.Fp4Matrix(fmt, len(byte), b, torch.from_numpy(c).to(DEV), torch.from_numpy(s).to(DEV))
    y = torch.empty((len(byte), b), device=DEV)
    fp4.dequantize(engine, m, y)
    with np.errstate(over="ignore"):
        ref = O.values(byte, code, fmt).astype(np.float32)
    assert np.array_equal(y.cpu().numpy(), ref, equal_nan=True)


@pytest.mark.parametrize("m", [7, 700])
def test_any_tensor_scale_in_expansion_and_product(engine, m):
    """Scales of matrices made elsewhere need not be powers of two: one f32 rounding in expansion, a factor in products."""
    n, k, ts = 70, 96, (np.float32(0.3), np.float32(1.7e-5))
    mats = []
    for rows, t in zip((m, n), ts):
        byte, code = O.quantize(rnd(rows, rows, k), "nv", 2.0 ** -6)
        c, s = O.pack(byte, code, "nv")
        mats.append((fp4.Fp4Matrix("nv", rows, k, torch.from_numpy(c).to(DEV), torch.from_numpy(s).to(DEV), float(t)),
                     O.values(byte, code, "nv", np.float64(t))))
    (xq, x), (wq, w) = mats
    y = fp4.dequantize(engine, xq, torch.empty((m, k), device=DEV))
    assert np.array_equal(y.cpu().numpy(), x.astype(np.float32))
    p = fp4.gemm(engine, wq, xq, torch.empty((m, n), device=DEV))
    # the factors' f32 product and the multiplication by it: two half steps
    check_close(p, x @ w.T, sum_bound(x, w) + 2 * 2.0 ** -24 * np.abs(x @ w.T))
    again = fp4.gemm(engine, xq, xq, torch.empty((m, m), device=DEV))  # one matrix on both sides
    check_close(again, x @ x.T, sum_bound(x, x) + 2 * 2.0 ** -24 * np.abs(x @ x.T))
    assert torch.equal(again, again.T)


# ----------------------------------------------------------------- product
SHAPES = [(1, 1, 1), (1, 128, 256), (1, 4096, 4096), (2, 16, 31), (3, 100, 1000), (8, 512, 512), (16, 129, 257), (17, 1536, 512),
          (19, 512, 2048), (31, 257, 96), (33, 1000, 1001), (64, 640, 1024), (65, 64, 64), (100, 1024, 512), (127, 128, 128),
          (128, 256, 256), (129, 257, 320), (200, 8, 5000), (256, 192, 63), (300, 1001, 1000), (333, 384, 4096), (513, 2048, 512),
          (1000, 300, 128), (2100, 130, 96), (4, 128, 70000), (300, 260, 20000), (700, 64, 64), (1025, 33, 257)]


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_gemm(engine, fmt, m, n, k):
    xq, x = mat_from(rnd(m + k, m, k), fmt)
    wq, w = mat_from(rnd(n + 2 * k, n, k, dev=0.05), fmt)
    bias = rnd(n, n).astype(np.float32)
    ref, bound = x @ w.T, sum_bound(x, w)
    for y_ty, b, pad in (("f32", None, 0), ("bf16", bias, 3), ("f16", bias, 8)):
        buf = torch.full((m + 2, n + pad), 77.0, dtype=DT[y_ty], device=DEV)
        fp4.gemm(engine, wq, xq, buf[:m, :n], None if b is None else torch.from_numpy(b).to(DEV))
        fp4.sync(engine)
        r = ref if b is None else ref + b
        # the f32 addition of the bias is one more rounding
        check_close(buf[:m, :n], r, bound + out_bound(r, y_ty) * (1 + 2.0 ** -10) + (0 if b is None else 2.0 ** -24 * np.abs(r)))
        assert bool((buf[m:] == 77).all()) and bool((buf[:, n:] == 77).all())


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("m", [1, 7, 40, 130, 600])
def test_gemm_exact_sums(engine, fmt, m):
    """Scales of one: every product is a multiple of 1/4 and every sum is below 2^17, so the result is exact."""
    n, k = 300, 2000
    rng = np.random.default_rng(m)
    mats = []
    for rows in (m, n):
        code = rng.integers(0, 16, (rows, k)).astype(np.uint8)
        byte = np.full((rows, -(-k // O.BLOCK[fmt])), 127 if fmt == "mx" else 56, np.uint8)
        c, s = O.pack(byte, code, fmt)
        mats.append((fp4.Fp4Matrix(fmt, rows, k, torch.from_numpy(c).to(DEV), torch.from_numpy(s).to(DEV)), O.values(byte, code, fmt)))
    y = torch.empty((m, n), device=DEV)
    fp4.gemm(engine, mats[1][0], mats[0][0], y)
    assert np.array_equal(y.double().cpu().numpy(), mats[0][1] @ mats[1][1].T)


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("m", [3, 200, 900])
def test_gemm_non_finite_blocks_stay_in_their_rows(engine, fmt, m):
    n, k = 150, 200
    xv, wv = rnd(1, m, k), rnd(2, n, k)
    xv[1, 40], wv[100, 199] = np.nan, np.inf
    xq, x = mat_from(xv, fmt)
    wq, w = mat_from(wv, fmt)
    y = torch.empty((m, n), device=DEV)
    fp4.gemm(engine, wq, xq, y)
    got = y.cpu().numpy()
    bad = np.zeros((m, n), bool)
    bad[1], bad[:, 100] = True, True
    assert np.isnan(got[bad]).all() and np.isfinite(got[~bad]).all()


@pytest.mark.parametrize("m", [5, 600])
@pytest.mark.parametrize("fmt", FMT)
def test_gemm_every_scale_byte(engine, fmt, m):
    """Random codes under every finite scale byte (mx: those whose products stay normal), subnormal scales among them."""
    n, k = 140, 256
    rng = np.random.default_rng(m)
    mats = []
    for rows in (m, n):
        code = rng.integers(0, 16, (rows, k)).astype(np.uint8)
        byte = rng.integers(*((70, 185) if fmt == "mx" else (0, 127)), (rows, k // O.BLOCK[fmt])).astype(np.uint8)
        c, s = O.pack(byte, code, fmt)
        mats.append((fp4.Fp4Matrix(fmt, rows, k, torch.from_numpy(c).to(DEV), torch.from_numpy(s).to(DEV)), O.values(byte, code, fmt)))
    y = torch.empty((m, n), device=DEV)
    fp4.gemm(engine, mats[1][0], mats[0][0], y)
    (_, x), (_, w) = mats
    check_close(y, x @ w.T, sum_bound(x, w) + 2.0 ** -24 * np.abs(x @ w.T))


def test_gemm_wide_range_of_scales(engine):
    """Blocks of very different scale, in rows of their own: the result follows the largest."""
    m, n, k = 40, 130, 512
    xv, wv = rnd(1, m, k), rnd(2, n, k)
    xv *= 2.0 ** np.linspace(-60, 60, m)[:, None].round()
    wv *= 2.0 ** np.linspace(-50, 50, n)[:, None].round()
    xv[:, 32:64] *= 2.0 ** -20
    for mm in (m, 200):
        xx = np.resize(xv, (mm, k))
        xq, x = mat_from(xx, "mx")
        wq, w = mat_from(wv, "mx")
        y = torch.empty((mm, n), device=DEV)
        fp4.gemm(engine, wq, xq, y)
        check_close(y, x @ w.T, sum_bound(x, w) + 2.0 ** -24 * np.abs(x @ w.T))


GLU_SHAPES = [(1, 1, 1), (1, 4096, 1024), (2, 33, 100), (16, 16, 64), (19, 2048, 512), (33, 130, 257), (40, 1000, 1000),
              (64, 96, 320), (100, 512, 512), (129, 260, 96), (300, 2048, 512), (520, 1001, 70), (1072, 128, 512)]


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("m,f,k", GLU_SHAPES)
def test_glu(engine, fmt, m, f, k):
    xq, x = mat_from(rnd(m + k, m, k), fmt)
    wq, w = mat_from(rnd(f + 2 * k, 2 * f, k, dev=1.5 / np.sqrt(k)), fmt)
    bias = (rnd(f, 2 * f) * 0.1).astype(np.float32)
    bd = torch.from_numpy(bias).to(DEV)
    db = sum_bound(x, w)
    z32 = None
    for y_ty, b in (("f32", bias), ("bf16", None), ("f16", bias), ("f32", None)):
        z = torch.full((m, f + 5), 77.0, dtype=DT[y_ty], device=DEV)
        fp4.glu(engine, wq, xq, z[:, :f], None if b is None else bd)
        fp4.sync(engine)
        h = x @ w.T + (0 if b is None else b)
        e = db + 2.0 ** -24 * np.abs(h)
        ref = O.glu(h, f)
        bound = 1.1 * e[:, :f] * (np.abs(h[:, f:]) + e[:, f:]) + np.abs(h[:, :f]) * e[:, f:] + 8 * 2.0 ** -24 * np.abs(ref)
        check_close(z[:, :f], ref, bound + out_bound(ref, y_ty) * (1 + 2.0 ** -10))
        assert bool((z[:, f:] == 77).all())
        z32 = z[:, :f]
    # quantised in the product: bit for bit what quantising its f32 result gives
    zq = empty(fmt, m, f)
    fp4.glu(engine, wq, xq, zq)
    want = fp4.quantize(engine, z32, empty(fmt, m, f))
    fp4.sync(engine)
    assert torch.equal(zq.scales, want.scales) and torch.equal(zq.codes, want.codes)


def test_glu_extreme_gates(engine):
    """Gates where exp overflows or vanishes: silu(-big) = 0, silu(big) = big, NaN rows stay NaN."""
    k = 64
    x = np.zeros((4, k))
    x[0, 0], x[1, 0], x[2, 0], x[3, 1] = 4, -4, 6, np.nan
    w = np.zeros((2 * 40, k))
    w[:40, 0], w[40:, 0] = 2.0 ** 10, 1.0
    xq, xv = mat_from(x, "mx")
    wq, wv = mat_from(w, "mx")
    z = torch.empty((4, 40), device=DEV)
    fp4.glu(engine, wq, xq, z)
    got = z.cpu().numpy()
    assert (got[0] == 4096 * 4).all() and (got[1] == 0).all() and (got[2] == 6144 * 6).all() and np.isnan(got[3]).all()
    zq = fp4.glu(engine, wq, xq, empty("mx", 4, 40))
    y = fp4.dequantize(engine, zq, torch.empty((4, 40), device=DEV)).cpu().numpy()
    assert (y[0] == 4096 * 4).all() and (y[1] == 0).all() and np.isnan(y[3]).all()


# ---------------------------------------------------- the operators together
@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("ty", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m,n,k,pad", [(1, 512, 512, 0), (5, 100, 1001, 3), (19, 1536, 512, 0), (32, 1000, 64, 1), (150, 257, 200, 8),
                                       (64, 300, 256, 1), (63, 40, 2048, 0), (2, 64, 8192, 5), (700, 300, 130, 1)])
def test_linear_is_quantize_and_gemm(engine, fmt, ty, m, n, k, pad):
    x = torch.from_numpy(rnd(m, m, k + pad)).to(DT[ty]).to(DEV)[:, :k]
    wq, w = mat_from(rnd(n, n, k, dev=0.05), fmt)
    b = torch.from_numpy(rnd(k, n).astype(np.float32)).to(DEV)
    y, y2 = (torch.full((m, n), float("nan"), device=DEV) for _ in range(2))
    fp4.linear(engine, wq, x, empty(fmt, m, k), y, b)
    fp4.gemm(engine, wq, fp4.quantize(engine, x, empty(fmt, m, k)), y2, b)
    fp4.sync(engine)
    assert torch.equal(y, y2)
    byte, code = O.quantize(x.double().cpu().numpy(), fmt, TS[fmt])
    xv = O.values(byte, code, fmt, TS[fmt])
    r = xv @ w.T + b.cpu().numpy()
    check_close(y, r, sum_bound(xv, w) + 2 * 2.0 ** -24 * np.abs(r))


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("m,f,k,n2", [(1, 2048, 512, 512), (19, 4096, 1024, 1024), (3, 33, 50, 70), (70, 500, 130, 90), (300, 2048, 512, 512)])
def test_mlp_is_its_parts(engine, fmt, m, f, k, n2):
    x = torch.from_numpy(rnd(m, m, k)).to(torch.bfloat16).to(DEV)
    w0, w0v = mat_from(rnd(f, 2 * f, k, dev=1.5 / np.sqrt(k)), fmt)
    w2, w2v = mat_from(rnd(f + 1, n2, f, dev=0.05), fmt)
    b0, b2 = (torch.from_numpy(rnd(i, n).astype(np.float32) * np.float32(0.1)).to(DEV) for i, n in ((1, 2 * f), (2, n2)))
    y, y2 = (torch.full((m, n2), float("nan"), device=DEV) for _ in range(2))
    fp4.mlp(engine, w0, w2, x, empty(fmt, m, k), empty(fmt, m, f), y, b0, b2)
    xq = fp4.quantize(engine, x, empty(fmt, m, k))
    zq = fp4.glu(engine, w0, xq, empty(fmt, m, f), b0)
    fp4.gemm(engine, w2, zq, y2, b2)
    fp4.sync(engine)
    assert torch.equal(y, y2)
    # against 64 bits from the hidden values that were used
    byte, code = O.unpack(zq.codes.cpu().numpy(), zq.scales.cpu().numpy(), m, f, fmt)
    zv = O.values(byte, code, fmt, TS[fmt])
    r = zv @ w2v.T + b2.cpu().numpy()
    check_close(y, r, sum_bound(zv, w2v) + 2 * 2.0 ** -24 * np.abs(r))
    # and those hidden values: a step away from the 64-bit ones at most
    byte, code = O.quantize(x.double().cpu().numpy(), fmt, TS[fmt])
    zr = O.glu(O.values(byte, code, fmt, TS[fmt]) @ w0v.T + b0.cpu().numpy(), f)
    rb, rc = O.quantize(zr, fmt, TS[fmt])
    step = np.repeat(O.scale_values(fmt, rb, TS[fmt]), O.BLOCK[fmt], 1)[:, :f]
    diff = np.abs(zv - O.values(rb, rc, fmt, TS[fmt]))
    assert (diff <= 4 * step).all() and np.mean(diff > 0) < 1e-2


@pytest.mark.parametrize("m", [1, 19, 256])
def test_graph_replay_and_streams(engine, m):
    """Captured on one stream and replayed with new inputs, while the same operators run on another stream."""
    f, k = 512, 256
    w0, _ = mat_from(rnd(1, 2 * f, k, dev=0.1), "nv")
    w2, _ = mat_from(rnd(2, k, f, dev=0.1), "nv")
    xs = [torch.from_numpy(rnd(10 + i, m, k).astype(np.float32)).to(DEV) for i in range(4)]

    def bufs():
        return empty("nv", m, k), empty("nv", m, f), torch.full((m, k), float("nan"), device=DEV)

    want = []
    for x in xs:
        xq, zq, y = bufs()
        want.append(fp4.mlp(engine, w0, w2, x, xq, zq, y).clone())
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):  # two graphs of the same weights, memory of their own
        s, x, (xq, zq, y) = torch.cuda.Stream(), xs[0].clone(), bufs()
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=s):
            fp4.mlp(engine, w0, w2, x, xq, zq, y)
        graphs.append((g, s, x, y, xq, zq))  # a graph's buffers live as long as it does
    torch.cuda.synchronize()
    other, (oxq, ozq, oy) = torch.cuda.Stream(), bufs()
    for i in range(4):
        for j, (g, s, x, y, *_) in enumerate(graphs):
            with torch.cuda.stream(s):
                x.copy_(xs[(i + j) % 4])
                g.replay()
        with torch.cuda.stream(other):
            fp4.mlp(engine, w0, w2, xs[3 - i], oxq, ozq, oy)
        torch.cuda.synchronize()
        for j, (g, s, x, y, *_) in enumerate(graphs):
            assert torch.equal(y, want[(i + j) % 4])
        assert torch.equal(oy, want[3 - i])
    fp4.sync(engine)


def test_two_threads(engine):
    k, n = 512, 700
    wq, _ = mat_from(rnd(1, n, k), "mx")
    xs = [torch.from_numpy(rnd(i, 5 + 60 * i, k).astype(np.float32)).to(DEV) for i in range(4)]
    want = [fp4.linear(engine, wq, x, empty("mx", len(x), k), torch.empty((len(x), n), device=DEV)).clone() for x in xs]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(20):
                y = torch.empty((len(xs[i]), n), device=DEV)
                fp4.linear(engine, wq, xs[i], empty("mx", len(xs[i]), k), y)
                s.synchronize()
                if not torch.equal(y, want[i]):
                    bad.append(i)

    ts = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert not bad


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("m", [6, 40, 300])
def test_linear_and_mlp_of_empty_and_non_finite_rows(engine, fmt, m):
    """Rows of zeros, of one value, with a NaN or an infinity, very large and very small ones: as by the parts."""
    k, f = 300, 200
    xv = rnd(m, m, k).astype(np.float32)
    xv[0], xv[1], xv[2, 7], xv[3, 299], xv[4] = 0, -0.0, np.nan, -np.inf, 1e-38
    xv[5] *= 2.0 ** 60
    x = torch.from_numpy(xv).to(DEV)
    w0, _ = mat_from(rnd(1, 2 * f, k, dev=0.1), fmt)
    w2, _ = mat_from(rnd(2, k, f, dev=0.1), fmt)
    y, h, y2 = torch.empty((m, k), device=DEV), torch.empty((m, 2 * f), device=DEV), torch.empty((m, k), device=DEV)
    fp4.mlp(engine, w0, w2, x, empty(fmt, m, k), empty(fmt, m, f), y)
    fp4.linear(engine, w0, x, empty(fmt, m, k), h)
    xq = fp4.quantize(engine, x, empty(fmt, m, k))
    check_matrix(xq, xv.astype(np.float64))
    fp4.gemm(engine, w2, fp4.glu(engine, w0, xq, empty(fmt, m, f)), y2)
    h2 = fp4.gemm(engine, w0, xq, torch.empty_like(h))
    fp4.sync(engine)
    for a, b in ((y, y2), (h, h2)):
        assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num())
    assert bool((h[:2] == 0).all()) and bool((y[:2] == 0).all())
    assert bool(h[2:4].isnan().all()) and bool(y[2:4].isnan().all()) and bool(h[4:].isfinite().all())


def test_kernels_of_every_kind_at_once(engine):
    """Products in clusters of several sizes, on CTA pairs and fused, from four streams at the same time."""
    jobs = []
    for i, (m, n, k, fmt) in enumerate([(1, 512, 4096, "nv"), (40, 1024, 2048, "mx"), (700, 2048, 512, "nv"), (19, 4096, 1024, "mx"),
                                        (100, 130, 8192, "nv"), (2000, 512, 256, "mx"), (64, 512, 512, "nv"), (300, 4000, 300, "mx")]):
        w, _ = mat_from(rnd(i, 2 * n, k, dev=0.1), fmt)
        x = torch.from_numpy(rnd(50 + i, m, k).astype(np.float32)).to(DEV)
        jobs.append((w, x, fmt, m, n, k))

    def run(job, y, z):
        w, x, fmt, m, n, k = job
        fp4.linear(engine, w, x, empty(fmt, m, k), y)
        fp4.glu(engine, w, fp4.quantize(engine, x, empty(fmt, m, k)), z)

    outs = [[(torch.empty((j[3], 2 * j[4]), device=DEV), torch.empty((j[3], j[4]), device=DEV)) for j in jobs] for _ in range(5)]
    for j, o in zip(jobs, outs[4]):
        run(j, *o)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    for rep in range(10):
        for i in range(len(jobs)):
            for s in range(4):
                with torch.cuda.stream(streams[s]):
                    a = (i + 2 * s) % len(jobs)
                    run(jobs[a], *outs[s][a])
    torch.cuda.synchronize()
    fp4.sync(engine)
    for s in range(4):
        for (y, z), (y0, z0) in zip(outs[s], outs[4]):
            assert torch.equal(y, y0) and torch.equal(z, z0)


def test_capture_across_streams(engine):
    """A captured fork and join: operators that follow another stream's work by events."""
    m, f, k = 33, 256, 128
    w0, _ = mat_from(rnd(1, 2 * f, k, dev=0.1), "mx")
    x = torch.from_numpy(rnd(2, m, k).astype(np.float32)).to(DEV)
    xq, xq2 = empty("mx", m, k), empty("mx", m, k)
    z, y, total = torch.empty((m, f), device=DEV), torch.empty((m, 2 * f), device=DEV), torch.empty((m, f), device=DEV)

    def run(s1, s2):
        with torch.cuda.stream(s1):
            x.mul_(2.0)
            fp4.quantize(engine, x, xq)
        s2.wait_stream(s1)
        with torch.cuda.stream(s2):
            fp4.gemm(engine, w0, xq, y)
        with torch.cuda.stream(s1):
            fp4.glu(engine, w0, xq, z)
        s1.wait_stream(s2)
        with torch.cuda.stream(s1):
            fp4.quantize(engine, x, xq2)
            torch.add(z, y[:, :f], out=total)

    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    run(s1, s2)
    torch.cuda.synchronize()
    want, x0 = total.clone(), x.clone()
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s1):
        run(s1, s2)
    for _ in range(3):
        x.copy_(x0 / 2)
        total.fill_(float("nan"))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(total, want) and torch.equal(xq.codes, xq2.codes)
    fp4.sync(engine)


@pytest.mark.parametrize("fmt", FMT)
def test_many_rows_and_many_columns(engine, fmt):
    k, n = 48, 20
    base = torch.from_numpy(rnd(1, 1000, k).astype(np.float32)).to(DEV)
    x = base.repeat(2101, 1)  # 2,101,000 tokens
    w, _ = mat_from(rnd(2, n, k), fmt)
    xq = fp4.quantize(engine, x, empty(fmt, len(x), k))
    y = fp4.gemm(engine, w, xq, torch.empty((len(x), n), dtype=torch.bfloat16, device=DEV))
    small = fp4.gemm(engine, w, fp4.quantize(engine, base, empty(fmt, 1000, k)), torch.empty((1000, n), dtype=torch.bfloat16, device=DEV))
    assert torch.equal(y.view(2101, 1000, n), small.expand(2101, 1000, n))
    back = fp4.dequantize(engine, xq, torch.empty_like(x))
    assert torch.equal(back.view(2101, 1000, k), back[:1000].expand(2101, 1000, k))
    # the same matrices the other way round: 2,101,000 weight rows, a few tokens and a few hundred
    for m in (3, 300):
        t = fp4.quantize(engine, base[:m].contiguous(), empty(fmt, m, k))
        wide = fp4.gemm(engine, xq, t, torch.empty((m, len(x)), dtype=torch.bfloat16, device=DEV))
        assert torch.equal(wide.view(m, 2101, 1000), wide[:, None, :1000].expand(m, 2101, 1000))


def test_offsets_past_32_bits(engine):
    """Rows of x and y that lie more than 2^32 bytes into their buffers."""
    rows, k, ld = 2200, 96, 1 << 20
    x = torch.zeros((rows, ld), dtype=torch.bfloat16, device=DEV)[:, :k]
    v = torch.from_numpy(rnd(5, rows, k)).to(torch.bfloat16).to(DEV)
    x.copy_(v)
    for fmt in FMT:
        m, m2 = fp4.quantize(engine, x, empty(fmt, rows, k)), fp4.quantize(engine, v, empty(fmt, rows, k))
        assert torch.equal(m.codes, m2.codes) and torch.equal(m.scales, m2.scales)
        y, y2 = x, torch.empty_like(v)
        fp4.dequantize(engine, m, y)
        fp4.dequantize(engine, m, y2)
        assert torch.equal(y, y2)
        wq, _ = mat_from(rnd(6, 80, k), fmt)
        fp4.gemm(engine, wq, m, x[:, :80])
        g2 = torch.empty((rows, 80), dtype=torch.bfloat16, device=DEV)
        fp4.gemm(engine, wq, m, g2)
        assert torch.equal(x[:, :80], g2)
        x.copy_(v)


def _process(*args):
    r = subprocess.run([sys.executable, os.path.join(os.path.dirname(__file__), "fp4_cases.py"), *args], capture_output=True,
                       text=True, timeout=300)
    assert r.returncode == 0, f"{args}: {r.stdout[-2000:]}\n{r.stderr[-4000:]}"


def test_checked_build_matches_product_bit_for_bit(tmp_path):
    """No index check of the checked build fails, and it computes the same bits."""
    _process("product", str(tmp_path / "p.npz"))
    _process("checked", str(tmp_path / "c.npz"))
    a, b = np.load(tmp_path / "p.npz"), np.load(tmp_path / "c.npz")
    assert sorted(a.files) == sorted(b.files) and len(a.files) == 96
    for k in a.files:
        assert np.isfinite(b[k]).all(), k
        assert np.array_equal(a[k], b[k]), k


def test_first_calls_of_a_process_can_be_captured():
    _process("capture")


# ---------------------------------------------------------------- refusals
def test_refusals(engine):
    e = engine
    m = empty("mx", 4, 64)
    x = torch.zeros((4, 64), device=DEV)
    y = torch.zeros((4, 4), device=DEV)
    w = empty("mx", 4, 64)
    nv = empty("nv", 4, 64)

    def refused(f, *a, **k):
        with pytest.raises(T0bError):
            f(e, *a, **k)

    refused(fp4.quantize, x.double(), m)
    refused(fp4.quantize, x[:, :63], m)
    refused(fp4.quantize, x.cpu(), m)
    refused(fp4.quantize, x.t().contiguous().t(), m)
    refused(fp4.quantize, x[:1].expand(4, 64), m)  # rows that overlap
    refused(fp4.quantize, x, empty("mx", 4, 64, ts=0.5))
    for ts in (0.3, 0.0, -1.0, float("nan"), float("inf"), 2.0 ** 65, 2.0 ** -65):
        refused(fp4.quantize, x, empty("nv", 4, 64, ts=ts))
    refused(fp4.gemm, w, nv, y)
    refused(fp4.gemm, w, empty("mx", 4, 32), y)
    refused(fp4.gemm, w, m, y[:, :3])
    refused(fp4.gemm, w, m, y, torch.zeros(3, device=DEV))
    refused(fp4.gemm, w, m, y, torch.zeros(4, device=DEV, dtype=torch.bfloat16))
    refused(fp4.gemm, empty("nv", 4, 64, ts=1e38), empty("nv", 4, 64, ts=1e38), y)
    refused(fp4.glu, empty("mx", 5, 64), m, torch.zeros((4, 2), device=DEV))
    refused(fp4.glu, w, m, empty("mx", 4, 3))
    refused(fp4.glu, w, m, empty("nv", 4, 2))
    refused(fp4.glu, w, m, empty("mx", 3, 2))
    refused(fp4.linear, w, x, nv, y)
    refused(fp4.mlp, w, empty("mx", 4, 3), x, m, empty("mx", 4, 2), y)
    refused(fp4.mlp, w, empty("mx", 4, 2), x, m, empty("mx", 4, 3), y)
    # a tensor scale that is no power of two: products and expansion take it, quantisation does not
    odd = fp4.Fp4Matrix("nv", 4, 64, nv.codes.zero_(), nv.scales.zero_(), 0.3)
    fp4.gemm(e, odd, odd, y)
    assert bool((y == 0).all())
    refused(fp4.quantize, x, odd)
    from t0_web_b200._lib import T0B_ERR_INVALID, T0B_ERR_UNSUPPORTED, lib
    import ctypes as C
    L, h = lib(), e.handle
    bad = type(m._c)(m._c.format, 4, 64, 1.0, m._c.codes + 1, m._c.scales)
    assert L.t0b_fp4_quantize(h, 0, x.data_ptr(), 64, C.byref(bad), None) == T0B_ERR_INVALID
    assert L.t0b_fp4_quantize(h, 0, x.data_ptr() + 2, 64, m._ref, None) == T0B_ERR_INVALID
    assert L.t0b_fp4_quantize(h, 0, x.data_ptr(), 63, m._ref, None) == T0B_ERR_INVALID
    assert L.t0b_fp4_quantize(h, 0, None, 64, m._ref, None) == T0B_ERR_INVALID
    assert L.t0b_fp4_quantize(h, 8, x.data_ptr(), 64, m._ref, None) == T0B_ERR_UNSUPPORTED
    assert L.t0b_fp4_glu(h, w._ref, m._ref, None, 0, y.data_ptr(), 4, m._ref, None) == T0B_ERR_INVALID
    assert L.t0b_fp4_glu(h, w._ref, m._ref, None, 0, None, 4, None, None) == T0B_ERR_INVALID
    assert b"either z_dev or zq" in L.t0b_last_error()
    fp4.sync(e)
