"""Standalone GEMMs whose operands the kernel before them on the stream has just written.

Every kernel may start while the one before it ends (programmatic dependent launch), and the 4-bit operators let it start
before they write.  What they write, as a bias too, has to be read after they have completed.
"""
import numpy as np
import pytest
import torch

from t0_web_b200 import fp4
from t0_web_b200._lib import Q4_0, Q8_0, check, lib, ptr
from test_gpu_qmatrix import DEV, QMatrix, _weights

pytestmark = pytest.mark.gpu

N, K = 1024, 1024
ROUNDS = 40


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _bias_writers(engine):
    """Calls that write a bias of N values, and what they write in round i."""
    g = torch.Generator(device=DEV).manual_seed(5)
    rnd = lambda *s: torch.randn(*s, device=DEV, generator=g)  # noqa: E731
    fmt = "mx"
    # the last row of a large expansion
    rows = 40000
    big = [fp4.quantize(engine, rnd(rows, N), fp4.Fp4Matrix.empty(fmt, rows, N, DEV)) for _ in range(2)]
    out = torch.empty((rows, N), device=DEV)
    # one token's product, and a token of a batch's
    w = fp4.quantize(engine, rnd(N, 4096) * 0.02, fp4.Fp4Matrix.empty(fmt, N, 4096, DEV))
    one = [fp4.quantize(engine, rnd(1, 4096), fp4.Fp4Matrix.empty(fmt, 1, 4096, DEV)) for _ in range(2)]
    y1 = torch.empty((1, N), device=DEV)
    many = [fp4.quantize(engine, rnd(2048, 4096), fp4.Fp4Matrix.empty(fmt, 2048, 4096, DEV)) for _ in range(2)]
    ym = torch.empty((2048, N), device=DEV)
    return {"expansion": (lambda i: fp4.dequantize(engine, big[i], out), out, out[-1]),
            "token": (lambda i: fp4.gemm(engine, w, one[i], y1), y1, y1[0]),
            "batch": (lambda i: fp4.gemm(engine, w, many[i], ym), ym, ym[-1])}


@pytest.mark.parametrize("writer", ["expansion", "token", "batch"])
@pytest.mark.parametrize("qtype", [Q8_0, Q4_0], ids=["q8_0", "q4_0"])
@pytest.mark.parametrize("m", [1, 16, 300])
def test_bias_written_by_the_kernel_before(engine, writer, qtype, m):
    wb, wd = _weights(qtype, N, K, seed=m)
    x = torch.from_numpy(np.random.default_rng(m).standard_normal((m, K), dtype=np.float32)).to(DEV)
    write, buf, bias = _bias_writers(engine)[writer]
    got = torch.empty((m, N), device=DEV)
    q = QMatrix(engine, qtype, wd, N, K)
    try:
        want = []
        for i in range(2):
            write(i)
            torch.cuda.synchronize()
            check(lib().t0b_qmatrix_gemm(q.h, ptr(x), m, bias.data_ptr(), ptr(got), _stream()))
            torch.cuda.synchronize()
            want.append(got.clone())
        bad = 0
        for r in range(ROUNDS):
            buf.fill_(float("nan"))
            got.fill_(float("nan"))
            torch.cuda.synchronize()
            write(r % 2)
            check(lib().t0b_qmatrix_gemm(q.h, ptr(x), m, bias.data_ptr(), ptr(got), _stream()))
            torch.cuda.synchronize()
            bad += not torch.equal(got, want[r % 2])
        check(lib().t0b_qmatrix_sync(q.h, _stream()))
    finally:
        q.close()
    fp4.sync(engine)
    assert bad == 0, f"{bad} of {ROUNDS}"


@pytest.mark.parametrize("m", [1, 16])
def test_bias_written_by_another_gemm(engine, m):
    """A product's row as the next product's bias, and as a bias of a gated MLP's parts."""
    f = 512
    (_, wd), (_, w0), (_, w2) = _weights(Q8_0, 2 * f, K, 1), _weights(Q8_0, 2 * f, K, 2), _weights(Q8_0, N, f, 3)
    x = torch.from_numpy(np.random.default_rng(m).standard_normal((m, K), dtype=np.float32)).to(DEV)
    b, y = torch.empty((m, 2 * f), device=DEV), torch.empty((m, N), device=DEV)
    q, q0, q2 = (QMatrix(engine, Q8_0, *a) for a in ((wd, 2 * f, K), (w0, 2 * f, K), (w2, N, f)))

    def run(wait):
        check(lib().t0b_qmatrix_gemm(q.h, ptr(x), m, None, ptr(b), _stream()))
        if wait:
            torch.cuda.synchronize()
        check(lib().t0b_qmatrix_swiglu(q0.h, q2.h, ptr(x), m, b[-1].data_ptr(), b[0].data_ptr(), None, ptr(y), _stream()))
        torch.cuda.synchronize()

    try:
        run(True)
        want, bad = y.clone(), 0
        for _ in range(ROUNDS):
            b.fill_(float("nan"))
            y.fill_(float("nan"))
            torch.cuda.synchronize()
            run(False)
            bad += not torch.equal(y, want)
    finally:
        for h in (q, q0, q2):
            h.close()
    assert torch.isfinite(want).all() and bad == 0, f"{bad} of {ROUNDS}"
