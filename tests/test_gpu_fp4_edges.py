"""4-bit operators: corners of the results, of the matrix layout, of error reporting and of the sigmoid.

Bounds of products and gated products: see test_gpu_fp4.py, whose helpers are used.
"""
import ctypes as C
import threading
import time

import numpy as np
import pytest
import torch

import fp4_oracle as O
from t0_web_b200 import fp4, t0_fast
from t0_web_b200._lib import T0B_ERR_DEVICE, T0bError, lib
from test_gpu_fp4 import DEV, DT, FMT, TS, check_close, empty, mat_from, out_bound, rnd, sum_bound

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


# ------------------------------------------------------------ error reporting
class _Word:
    """The engine's device error word of the 4-bit operators, as a tensor."""

    def __init__(self, engine):
        f = lib()["_Z18t0b_engine_fp4_errPK10t0b_engine"]
        f.argtypes, f.restype = [C.c_void_p], C.c_void_p
        self.__cuda_array_interface__ = dict(shape=(1,), typestr="<i4", data=(f(engine.handle), False), version=2)


def error_word(engine):
    return torch.as_tensor(_Word(engine), device=DEV)


def test_error_of_a_kernel_is_reported_once(engine):
    word = error_word(engine)
    assert int(word) == 0
    outcome = torch.zeros(1, dtype=torch.int32, device=DEV)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    wait = lib()["_Z32t0b_launch_bounded_wait_selftestPiS_P11CUstream_st"]
    wait.argtypes = [C.c_void_p] * 3
    assert wait(word.data_ptr(), outcome.data_ptr(), side.cuda_stream) == 0
    with pytest.raises(T0bError) as e:
        fp4.sync(engine, side.cuda_stream)
    assert e.value.status == T0B_ERR_DEVICE and "error code 1" in str(e.value)
    assert int(outcome) == 2
    fp4.sync(engine, side.cuda_stream)
    fp4.sync(engine)


def test_errors_during_a_sync_are_not_lost(engine):
    """An error recorded while another thread reads and clears the word is reported by that call or by the next."""
    word = error_word(engine)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    lost = []
    for i in range(400):
        said = []

        def sync():
            try:
                fp4.sync(engine, a.cuda_stream)
            except T0bError as e:
                said.append(str(e))

        with torch.cuda.stream(a):
            word.fill_(1)
        a.synchronize()
        t = threading.Thread(target=sync)
        t.start()
        end = time.perf_counter() + (i % 100) * 2e-6
        while time.perf_counter() < end:
            pass
        with torch.cuda.stream(b):
            word.fill_(2)
        b.synchronize()
        t.join()
        sync()
        if not any("error code 2" in s for s in said):
            lost.append(i)
    word.zero_()
    torch.cuda.synchronize()
    assert not lost, f"{len(lost)} of 400"


def test_new_engine_has_no_errors_while_the_default_stream_is_busy():
    e = t0_fast.Engine(0)
    word = error_word(e)
    at = word.data_ptr()
    word.fill_(7)
    torch.cuda.synchronize()
    e.close()
    side = torch.cuda.Stream()
    torch.cuda._sleep(400_000_000)  # about 0.2 s on the legacy default stream
    e = t0_fast.Engine(0)
    fp4.sync(e, side.cuda_stream)  # a non-blocking stream: not ordered after the default one
    if error_word(e).data_ptr() != at:
        pytest.skip("the new engine's word lies elsewhere: nothing stale to see")
    torch.cuda.synchronize()
    e.close()


def test_sync_of_a_stream_under_capture_is_refused(engine):
    w, _ = mat_from(rnd(1, 64, 96), "mx")
    x, _ = mat_from(rnd(2, 5, 96), "mx")
    y, want = torch.full((5, 64), float("nan"), device=DEV), torch.empty((5, 64), device=DEV)
    fp4.gemm(engine, w, x, want)
    torch.cuda.synchronize()
    g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(g, stream=s):
        fp4.gemm(engine, w, x, y)
        with pytest.raises(T0bError, match="captured"):
            fp4.sync(engine)
    g.replay()
    fp4.sync(engine)
    assert torch.equal(y, want)


# ---------------------------------------------------------------- the sigmoid
@pytest.mark.parametrize("m", [3, 700])  # both product kernels
@pytest.mark.parametrize("y_ty", ["f32", "bf16"])
def test_glu_small_sigmoids_of_large_values(engine, m, y_ty):
    """Gates down to -210 against up values to 3e38: products in range although the sigmoid alone is not.

    The gates and up values are the biases (x = 0), exact in f32.  Bound: 8 units of 2^-24 for exp, quotient and products,
    half a step of the output type, and two half steps of f32's smallest number where the result is subnormal."""
    f = 640
    rng = np.random.default_rng(7)
    g = np.concatenate([np.linspace(-210, -80, f - 8), [-87, np.nextafter(np.float32(-87), np.float32(-100)), -87.3365, -87.34, -88.8, -103.9,
                                                        -104.5, -120]]).astype(np.float32)
    rng.shuffle(g)
    u = (rng.choice([-1, 1], f) * 10.0 ** rng.uniform(0, 38.4, f)).astype(np.float32)
    w, _ = mat_from(np.zeros((2 * f, 64)), "mx")
    x, _ = mat_from(np.zeros((m, 64)), "mx")
    z = torch.full((m, f), float("nan"), dtype=DT[y_ty], device=DEV)
    fp4.glu(engine, w, x, z, torch.from_numpy(np.concatenate([g, u])).to(DEV))
    fp4.sync(engine)
    g, u = g.astype(np.float64), u.astype(np.float64)
    ref = np.broadcast_to(g / (1 + np.exp(-g)) * u, (m, f))
    check_close(z, ref, 8 * 2.0 ** -24 * np.abs(ref) + 2 * 2.0 ** -150 + out_bound(ref, y_ty) * (1 + 2.0 ** -10)
                + (2.0 ** -134 if y_ty == "bf16" else 0))


def test_glu_mixed_gates_on_both_kernels(engine):
    """Ordinary gates beside large and small ones: the same bits from both product kernels, a group of 32 of one kind or mixed."""
    f = 64 * 8
    rng = np.random.default_rng(8)
    g = rng.standard_normal((8, 64)) * 5
    g[1], g[2], g[3] = rng.uniform(88, 3000, 64), rng.uniform(-150, -88, 64), rng.uniform(-200, 200, 64)
    g[4, 7], g[5, 9], g[6, 11], g[7, 13] = 1e6, 1e30, -87.5, -1e30
    g, u = g.reshape(-1).astype(np.float32), rng.standard_normal(f).astype(np.float32)
    w, _ = mat_from(np.zeros((2 * f, 64)), "nv")
    bias = torch.from_numpy(np.concatenate([g, u])).to(DEV)
    got = []
    for m in (3, 700):
        x, _ = mat_from(np.zeros((m, 64)), "nv")
        got.append(fp4.glu(engine, w, x, torch.full((m, f), float("nan"), device=DEV), bias))
    fp4.sync(engine)
    assert torch.equal(got[1], got[0][:1].expand(700, f)) and torch.equal(got[0], got[0][:1].expand(3, f))
    g, u = g.astype(np.float64), u.astype(np.float64)
    with np.errstate(over="ignore"):
        ref = g / (1 + np.exp(-g)) * u
    check_close(got[0][:1], ref[None], 8 * 2.0 ** -24 * np.abs(ref[None]) + 2 * 2.0 ** -150)


def test_glu_infinite_gates_and_values(engine):
    """silu(-inf) is NaN (-inf / inf) and silu(inf) infinite; a negative gate's finite factor leaves an infinity."""
    f = 64
    inf = float("inf")
    g = torch.tensor([-inf, inf, -100.0, -1e38, float("nan"), 100.0, -50.0, 1e38], device=DEV).repeat(f // 8)
    u = torch.tensor([1.0, 2.0, inf, 3e38, 1.0, -inf, inf, 1.0], device=DEV).repeat(f // 8)
    w, _ = mat_from(np.zeros((2 * f, 64)), "mx")
    for m in (3, 700):
        x, _ = mat_from(np.zeros((m, 64)), "mx")
        z = fp4.glu(engine, w, x, torch.empty((m, f), device=DEV), torch.cat([g, u])).cpu().numpy()
        want = np.tile(np.array([np.nan, inf, -inf, 0, np.nan, -inf, -inf, 1e38], np.float32), f // 8)
        assert np.array_equal(z, np.broadcast_to(want, z.shape), equal_nan=True)


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


# ------------------------------------------------------------ threads, objects
def test_threads_finish_their_work(engine):
    k, n, rounds = 512, 700, 20
    wq, _ = mat_from(rnd(1, n, k), "mx")
    xs = [torch.from_numpy(rnd(i, 5 + 60 * i, k).astype(np.float32)).to(DEV) for i in range(4)]
    want = [fp4.linear(engine, wq, x, empty("mx", len(x), k), torch.empty((len(x), n), device=DEV)).clone() for x in xs]
    torch.cuda.synchronize()
    bad, done = [], [0] * 4

    def work(i):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for _ in range(rounds):
                    y = torch.empty((len(xs[i]), n), device=DEV)
                    fp4.linear(engine, wq, xs[i], empty("mx", len(xs[i]), k), y)
                    fp4.sync(engine)
                    if not torch.equal(y, want[i]):
                        bad.append(i)
                    done[i] += 1
        except Exception as e:  # noqa: BLE001  (an exception ends the thread only)
            bad.append((i, repr(e)))

    ts = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    fp4.sync(engine)
    assert not bad and done == [rounds] * 4


def test_matrices_cannot_be_changed_behind_their_pointers():
    m = fp4.Fp4Matrix.empty("nv", 4, 64, DEV, 2.0 ** -6)
    for name, v in (("codes", m.codes.clone()), ("scales", m.scales.clone()), ("tensor_scale", 0.5), ("rows", 3), ("k", 32), ("format", "mx")):
        with pytest.raises(AttributeError):
            setattr(m, name, v)
    assert m.tensor_scale == 2.0 ** -6 and m._c.codes == m.codes.data_ptr()
    m.label = "a user's own attribute"
    assert m.label


# --------------------------------------------------------------- K slices
@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("k", [257, 513, 1281, 2305, 2600, 2817, 3329, 3585])  # clusters of 1 to 8, slices of unequal length
@pytest.mark.parametrize("m", [1, 5, 40, 64])
def test_every_cluster_size(engine, fmt, m, k):
    n = 130
    xq, x = mat_from(rnd(m + k, m, k), fmt)
    wq, w = mat_from(rnd(k, 2 * n, k, dev=1.5 / np.sqrt(k)), fmt)
    h, e = x @ w.T, sum_bound(x, w)
    e = e + 2.0 ** -24 * np.abs(h)
    y = fp4.gemm(engine, wq, xq, torch.full((m, 2 * n), float("nan"), device=DEV))
    z = fp4.glu(engine, wq, xq, torch.full((m, n), float("nan"), device=DEV))
    fp4.sync(engine)
    check_close(y, h, e)
    zr = O.glu(h, n)
    check_close(z, zr, 1.1 * e[:, :n] * (np.abs(h[:, n:]) + e[:, n:]) + np.abs(h[:, :n]) * e[:, n:] + 9 * 2.0 ** -24 * np.abs(zr))


# ------------------------------------------------------------------ long sums
@pytest.mark.parametrize("fmt", FMT)
def test_longest_rows(engine, fmt):
    """k = 2^20, the longest row there is: quantised, expanded, multiplied, gated."""
    m, n, k = 9, 20, 1 << 20
    xv = rnd(1, m, k).astype(np.float32)
    xd = torch.from_numpy(xv).to(DEV)
    xq = fp4.quantize(engine, xd, empty(fmt, m, k))
    byte, code = O.quantize(xv, fmt, TS[fmt])
    c, s = O.pack(byte, code, fmt)
    assert np.array_equal(xq.codes.cpu().numpy(), c) and np.array_equal(xq.scales.cpu().numpy(), s)
    x = O.values(byte, code, fmt, TS[fmt])
    assert np.array_equal(fp4.dequantize(engine, xq, torch.empty_like(xd)).cpu().numpy(), x)
    wq, w = mat_from(rnd(2, n, k, dev=2.0 ** -10), fmt)
    ref, bound = x @ w.T, sum_bound(x, w)
    y = fp4.gemm(engine, wq, xq, torch.empty((m, n), device=DEV))
    check_close(y, ref, bound + 2.0 ** -24 * np.abs(ref))
    y2 = fp4.linear(engine, wq, xd, empty(fmt, m, k), torch.empty((m, n), device=DEV))
    assert torch.equal(y, y2)
    z = fp4.glu(engine, wq, xq, torch.empty((m, n // 2), device=DEV))
    fp4.sync(engine)
    f = n // 2
    e = bound + 2.0 ** -24 * np.abs(ref)
    zr = O.glu(ref, f)
    check_close(z, zr, 1.1 * e[:, :f] * (np.abs(ref[:, f:]) + e[:, f:]) + np.abs(ref[:, :f]) * e[:, f:] + 9 * 2.0 ** -24 * np.abs(zr))
