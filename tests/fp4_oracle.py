"""Plain 64-bit restatement of the 4-bit microscaled format, for the tests."""
import numpy as np

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
BLOCK = {"mx": 32, "nv": 16}
# value of every scale byte of the "nv" format (4 exponent bits of bias 7, 3 mantissa bits; 127 is NaN)
E4M3 = np.array([(b & 7) / 8 * 2.0 ** -6 if b < 8 else (1 + (b & 7) / 8) * 2.0 ** ((b >> 3) - 7) for b in range(127)] + [np.nan])


def nearest_even(a, grid):
    """Index of the nearest grid entry, ties to the even index, clamped at the last."""
    mid = (grid[1:] + grid[:-1]) / 2
    lo, hi = np.searchsorted(mid, a, "left"), np.searchsorted(mid, a, "right")
    return np.where(lo % 2 == 0, lo, hi)


def scale_values(fmt, byte, ts):
    byte = np.asarray(byte)
    if fmt == "mx":
        return np.where(byte == 255, np.nan, 2.0 ** (np.minimum(byte, 254).astype(np.float64) - 127))
    return E4M3[np.minimum(byte, 127)] * ts


def quantize(x, fmt, ts=1.0):
    """x [rows, k] -> (scale bytes [rows, blocks], codes [rows, k] with sign bit 3)."""
    x = np.asarray(x, np.float64)
    rows, k = x.shape
    b = BLOCK[fmt]
    nb = -(-k // b)
    u = np.pad(x, ((0, 0), (0, nb * b - k))).reshape(rows, nb, b)
    top = np.abs(u).max(2)  # NaN propagates
    bad = ~np.isfinite(top)
    t = np.where(bad, 0, top)
    if fmt == "mx":
        _, ex = np.frexp(t)
        byte = np.where(t > 0, np.clip(ex - 1 - 2 + 127, 0, 254), 0)
        byte = np.where(bad, 255, byte)
    else:
        byte = np.where(bad, 127, nearest_even(t / (6 * ts), E4M3[:127]))
    s = scale_values(fmt, byte, ts)[:, :, None]
    with np.errstate(invalid="ignore", divide="ignore"):
        q = np.where(s > 0, np.abs(np.where(np.isfinite(u), u, 0)) / np.where(s > 0, s, 1), 0)
    # a block whose scale rounded to zero is zero as a whole, without signs
    code = np.where(s == 0, 0, nearest_even(q, GRID) | (np.signbit(u).astype(int) << 3))
    return byte.astype(np.uint8), code.reshape(rows, -1)[:, :k].astype(np.uint8)


def values(byte, code, fmt, ts=1.0):
    k = code.shape[1]
    v = np.where(code & 8, -1.0, 1.0) * GRID[code & 7]
    return v * np.repeat(scale_values(fmt, byte, ts), BLOCK[fmt], 1)[:, :k]


def pack(byte, code, fmt):
    """The two arrays as they are held: codes, tiled scales (uint8, flat)."""
    rows, k = code.shape
    c = np.pad(code, ((0, 0), (0, -k % 32)))
    codes = (c[:, 0::2] | (c[:, 1::2] << 4)).astype(np.uint8)
    nb = byte.shape[1]
    rt, kt = -(-rows // 128), -(-nb // 4)
    t = np.zeros((rt, kt, 512), np.uint8)
    r, b = np.meshgrid(np.arange(rows), np.arange(nb), indexing="ij")
    t[r // 128, b // 4, (r % 32) * 16 + (r % 128 // 32) * 4 + b % 4] = byte
    return codes.reshape(-1), t.reshape(-1)


def unpack(codes, scales, rows, k, fmt):
    c = codes.reshape(rows, -1)
    code = np.stack([c & 15, c >> 4], 2).reshape(rows, -1)[:, :k]
    nb = -(-k // BLOCK[fmt])
    r, b = np.meshgrid(np.arange(rows), np.arange(nb), indexing="ij")
    t = scales.reshape(-(-rows // 128), -(-nb // 4), 512)
    return t[r // 128, b // 4, (r % 32) * 16 + (r % 128 // 32) * 4 + b % 4], code


def glu(h, f):
    g, u = h[:, :f], h[:, f:]
    with np.errstate(over="ignore"):
        return g / (1 + np.exp(-g)) * u
