"""4-bit operators: corners of the results, of the matrix layout, of error reporting and of the sigmoid.

Bounds of products and gated products: see test_gpu_fp4.py, whose helpers are used.
"""
import numpy as np
import pytest
import torch

import fp4_oracle as O
from t0_web_b200 import fp4
from test_gpu_fp4 import DEV, DT, FMT, check_close, empty, mat_from, out_bound, rnd, sum_bound

pytestmark = pytest.mark.gpu


# ---------------------------------------------------- zeros behind the matrix
def check_padding(m):
    """Codes behind k and scales of blocks and rows behind the matrix are zero."""
    kp = -(-m.k // 32) * 32
    code = O.unpack(m.codes.cpu().numpy(), m.scales.cpu().numpy(), m.rows, kp, m.format)[1]
    assert not code[:, m.k:].any()
    nb = -(-m.k // O.BLOCK[m.format])
    s = m.scales.cpu().numpy().reshape(-(-m.rows // 128), -(-nb // 4), 32, 4, 4)
    s = s.transpose(0, 3, 2, 1, 4).reshape(-(-m.rows // 128) * 128, -(-nb // 4) * 4)
    assert not s[m.rows:].any() and not s[:, nb:].any()


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("ty", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,k,pad", [(3, 15, 1), (5, 17, 3), (200, 33, 0), (129, 100, 4), (33, 1001, 0), (140, 1001, 7), (2, 200, 8)])
def test_codes_behind_k_of_blocks_with_nan(engine, fmt, ty, rows, k, pad):
    x = torch.from_numpy(rnd(k, rows, k + pad)).to(DT[ty])[:, :k].to(DEV)
    buf = torch.zeros((rows, k + pad), dtype=DT[ty], device=DEV)
    x = buf[:, :k].copy_(x)
    x[0, k - 1], x[rows - 1, k - 1] = float("nan"), float("-inf")
    x[rows // 2, k - 1] = float("inf")
    m = fp4.quantize(engine, x, empty(fmt, rows, k))
    check_padding(m)
    byte = O.unpack(m.codes.cpu().numpy(), m.scales.cpu().numpy(), rows, k, fmt)[0]
    assert (byte[[0, rows // 2, rows - 1], -1] == (255 if fmt == "mx" else 127)).all()


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("m", [1, 5, 40, 130, 700])  # few tokens, clusters, CTA pairs
@pytest.mark.parametrize("f", [70, 257, 1001])
def test_hidden_codes_behind_f_of_blocks_with_nan(engine, fmt, m, f):
    k = 96
    wv = rnd(f, 2 * f, k, dev=0.1)
    wv[f - 1, 3] = np.nan  # the last gate row: the last hidden value of every token
    w, _ = mat_from(wv, fmt)
    x, _ = mat_from(rnd(m, m, k), fmt)
    z = fp4.glu(engine, w, x, empty(fmt, m, f))
    check_padding(z)
    byte = O.unpack(z.codes.cpu().numpy(), z.scales.cpu().numpy(), m, f, fmt)[0]
    assert (byte[:, -1] == (255 if fmt == "mx" else 127)).all() and (byte[:, :-1] < 127 + 128 * (fmt == "mx")).all()


# ----------------------------------------------------------- aligned results
@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("m,f,k", [(300, 2048, 512), (700, 1000, 96), (1072, 2048, 512), (520, 1001, 70), (513, 384, 1024), (300, 260, 256),
                                   (19, 1000, 200)])
def test_glu_into_aligned_rows(engine, fmt, m, f, k):
    """Results whose rows start on 16-byte boundaries (written by TMA on CTA pairs), every type."""
    xq, x = mat_from(rnd(m + k, m, k), fmt)
    wq, w = mat_from(rnd(f + 2 * k, 2 * f, k, dev=1.5 / np.sqrt(k)), fmt)
    bias = (rnd(f, 2 * f) * 0.1).astype(np.float32)
    h = x @ w.T + bias
    e = sum_bound(x, w) + 2.0 ** -24 * np.abs(h)
    ref = O.glu(h, f)
    bound = 1.1 * e[:, :f] * (np.abs(h[:, f:]) + e[:, f:]) + np.abs(h[:, :f]) * e[:, f:] + 8 * 2.0 ** -24 * np.abs(ref)
    ld = -(-f // 8) * 8
    for y_ty in ("f32", "f16", "bf16"):
        z = torch.full((m + 2, ld + 8), 77.0, dtype=DT[y_ty], device=DEV)
        fp4.glu(engine, wq, xq, z[:m, :f], torch.from_numpy(bias).to(DEV))
        fp4.sync(engine)
        check_close(z[:m, :f], ref, bound + out_bound(ref, y_ty) * (1 + 2.0 ** -10))
        assert bool((z[m:] == 77).all()) and bool((z[:, f:] == 77).all())


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("m,n,k", [(300, 1000, 320), (2100, 136, 96), (513, 2048, 512), (1000, 300, 128), (300, 257, 2000), (33, 1000, 1001)])
def test_gemm_into_aligned_rows(engine, fmt, m, n, k):
    xq, x = mat_from(rnd(m + k, m, k), fmt)
    wq, w = mat_from(rnd(n + 2 * k, n, k, dev=0.05), fmt)
    bias = rnd(n, n).astype(np.float32)
    r = x @ w.T + bias
    bound = sum_bound(x, w) + 2.0 ** -24 * np.abs(r)
    ld = -(-n // 8) * 8
    for y_ty in ("f32", "f16", "bf16"):
        y = torch.full((m + 2, ld + 8), 77.0, dtype=DT[y_ty], device=DEV)
        fp4.gemm(engine, wq, xq, y[:m, :n], torch.from_numpy(bias).to(DEV))
        fp4.sync(engine)
        check_close(y[:m, :n], r, bound + out_bound(r, y_ty) * (1 + 2.0 ** -10))
        assert bool((y[m:] == 77).all()) and bool((y[:, n:] == 77).all())


@pytest.mark.parametrize("m", [40, 2100])  # few tokens, CTA pairs
@pytest.mark.parametrize("n", [1, 3, *range(127, 138), 259])
def test_nothing_behind_the_last_column_is_written(engine, m, n):
    k = 96
    xq, x = mat_from(rnd(m, m, k), "nv")
    wv = rnd(n, 2 * n, k, dev=0.2)
    (wq, w), (half, _) = mat_from(wv, "nv"), mat_from(wv[:n], "nv")
    h, e = x @ w.T, sum_bound(x, w)
    ref = O.glu(h, n)
    bound = 1.1 * e[:, :n] * (np.abs(h[:, n:]) + e[:, n:]) + np.abs(h[:, :n]) * e[:, n:] + 8 * 2.0 ** -24 * np.abs(ref)
    for y_ty in ("f32", "f16", "bf16"):
        buf = torch.full((m + 1, -(-n // 8) * 8 + 8), 77.0, dtype=DT[y_ty], device=DEV)
        for f, a, r, b in ((fp4.gemm, half, h[:, :n], e[:, :n] + 2.0 ** -24 * np.abs(h[:, :n])), (fp4.glu, wq, ref, bound)):
            buf.fill_(77.0)
            f(engine, a, xq, buf[:m, :n])
            check_close(buf[:m, :n], r, b + out_bound(r, y_ty) * (1 + 2.0 ** -10))
            assert bool((buf[m:] == 77).all()) and bool((buf[:, n:] == 77).all())
    fp4.sync(engine)
