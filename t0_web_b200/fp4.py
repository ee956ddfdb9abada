"""4-bit microscaled matrices and their operators (t0b_fp4_* of include/t0b.h).

An `Fp4Matrix` holds a matrix [rows, k] in 4 bits per value and one 8-bit scale
per block of 32 values (format "mx", power-of-two scales) or 16 values ("nv",
8-bit float scales times the matrix's own `tensor_scale`).  Operators take
torch tensors on the engine's device: float32, float16 or bfloat16, unit stride
along the columns, rows any distance apart that does not make them overlap.

    engine = t0_fast.Engine(0)
    w = fp4.Fp4Matrix.empty("nv", n, k, "cuda:0", tensor_scale=2.0 ** -12)
    fp4.quantize(engine, weights, w)                  # [n, k] -> 4 bits, once
    xq = fp4.Fp4Matrix.empty("nv", m, k, "cuda:0", tensor_scale=2.0 ** -6)
    fp4.linear(engine, w, x, xq, y)                   # y = q(x) . w^T
    fp4.sync(engine)                                  # kernel-side errors

Every call queues work on `stream` (a cudaStream_t as an integer; by default
torch's current stream of the engine's device) and returns; arguments that do
not fit raise T0bError (or TypeError) before anything is queued.  As with
torch's own operators, a tensor that is used on another stream than its own
has to outlive that use (`Tensor.record_stream`, or a reference kept until the
stream has passed).
"""
from __future__ import annotations

import ctypes as C

import torch

from ._lib import BF16, F16, F32, FP4_MX, FP4_NV, T0B_ERR_INVALID, Fp4, T0bError, check, lib

FORMATS = {"mx": FP4_MX, "nv": FP4_NV}
BLOCK = {"mx": 32, "nv": 16}
_TYPES = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}


def _shape32(rows: int, k: int):
    """The shape as the C calls take it; ctypes would cut larger numbers to 32 bits, so they become an invalid 0."""
    return tuple(v if -(1 << 31) <= v < 1 << 31 else 0 for v in (rows, k))


def code_bytes(rows: int, k: int) -> int:
    return int(lib().t0b_fp4_code_bytes(*_shape32(rows, k)))


def scale_bytes(fmt: str, rows: int, k: int) -> int:
    return int(lib().t0b_fp4_scale_bytes(FORMATS[fmt], *_shape32(rows, k)))


class Fp4Matrix:
    """A 4-bit matrix over two uint8 tensors (layout: include/t0b.h), which it keeps alive.

    What it holds cannot be set anew: calls go by the pointers taken here.  (The tensors' contents may be written.)"""

    def __init__(self, fmt: str, rows: int, k: int, codes: torch.Tensor, scales: torch.Tensor, tensor_scale: float = 1.0):
        if fmt not in FORMATS:
            raise T0bError(T0B_ERR_INVALID, f"Fp4Matrix: format must be one of {sorted(FORMATS)}, not {fmt!r}")
        need = code_bytes(rows, k), scale_bytes(fmt, rows, k)
        if not need[0]:
            raise T0bError(T0B_ERR_INVALID, f"Fp4Matrix: shape [{rows}, {k}] is empty or too large")
        for name, t, n in (("codes", codes, need[0]), ("scales", scales, need[1])):
            if t.dtype != torch.uint8 or not t.is_contiguous() or t.numel() != n:
                raise T0bError(T0B_ERR_INVALID, f"Fp4Matrix: {name} must be {n} contiguous uint8 values")
            if t.device.type != "cuda" or t.device != codes.device:
                raise T0bError(T0B_ERR_INVALID, f"Fp4Matrix: {name} must be on the codes' CUDA device, not {t.device}")
        self.format, self.rows, self.k, self.tensor_scale = fmt, rows, k, tensor_scale
        self.codes, self.scales = codes, scales
        self._device = codes.device.index
        self._c = Fp4(FORMATS[fmt], rows, k, tensor_scale, codes.data_ptr(), scales.data_ptr())
        self._ref = C.byref(self._c)

    def __setattr__(self, name, value):
        if "_ref" in self.__dict__ and name in self.__dict__:
            raise AttributeError(f"Fp4Matrix: {name} cannot be set, make another matrix")
        object.__setattr__(self, name, value)

    @classmethod
    def empty(cls, fmt: str, rows: int, k: int, device, tensor_scale: float = 1.0) -> "Fp4Matrix":
        """A matrix with memory of its own, not yet written."""
        if fmt not in FORMATS:
            raise T0bError(T0B_ERR_INVALID, f"Fp4Matrix: format must be one of {sorted(FORMATS)}, not {fmt!r}")
        codes = torch.empty(code_bytes(rows, k), dtype=torch.uint8, device=device)
        scales = torch.empty(scale_bytes(fmt, rows, k), dtype=torch.uint8, device=device)
        return cls(fmt, rows, k, codes, scales, tensor_scale)

    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()


def _mat(engine, m: Fp4Matrix):
    if m._device != engine.device:
        raise T0bError(T0B_ERR_INVALID, f"fp4: a matrix is on cuda:{m._device}, the engine on cuda:{engine.device}")
    return m._ref


def _plain(engine, name: str, t: torch.Tensor, rows: int, cols: int):
    """(type id, pointer, row stride) of a plain tensor [rows, cols]."""
    ty = _TYPES.get(t.dtype)
    if ty is None:
        raise T0bError(T0B_ERR_INVALID, f"fp4: {name} must be float32, float16 or bfloat16, not {t.dtype}")
    if t.get_device() != engine.device:  # -1 for host memory
        raise T0bError(T0B_ERR_INVALID, f"fp4: {name} is on {t.device}, the engine on cuda:{engine.device}")
    if t.shape != (rows, cols):
        raise T0bError(T0B_ERR_INVALID, f"fp4: {name} has shape {tuple(t.shape)}, expected ({rows}, {cols})")
    s0, s1 = t.stride()
    if s1 != 1 and cols > 1:
        raise T0bError(T0B_ERR_INVALID, f"fp4: {name} must have unit stride along its columns")
    return ty, t.data_ptr(), s0 if rows > 1 else max(s0, cols)


def _bias(engine, name: str, b, n: int):
    if b is None:
        return None
    if b.dtype != torch.float32 or b.get_device() != engine.device or b.numel() != n or not b.is_contiguous():
        raise T0bError(T0B_ERR_INVALID, f"fp4: {name} must be {n} contiguous float32 values on cuda:{engine.device}")
    return b.data_ptr()


def _stream(engine, stream):
    # the pointer alone: building torch's Stream object costs more than the rest of a small call's checks
    return torch._C._cuda_getCurrentRawStream(engine.device) if stream is None else stream


def quantize(engine, x: torch.Tensor, out: Fp4Matrix, stream=None) -> Fp4Matrix:
    """x [rows, k] to 4 bits."""
    ty, p, ld = _plain(engine, "x", x, out.rows, out.k)
    check(lib().t0b_fp4_quantize(engine._h, ty, p, ld, _mat(engine, out), _stream(engine, stream)))
    return out


def dequantize(engine, m: Fp4Matrix, y: torch.Tensor, stream=None) -> torch.Tensor:
    """The values of m, rounded to y's type."""
    ty, p, ld = _plain(engine, "y", y, m.rows, m.k)
    check(lib().t0b_fp4_dequantize(engine._h, _mat(engine, m), ty, p, ld, _stream(engine, stream)))
    return y


def gemm(engine, w: Fp4Matrix, x: Fp4Matrix, y: torch.Tensor, bias=None, stream=None) -> torch.Tensor:
    """y [x.rows, w.rows] = x . w^T (+ bias)."""
    ty, p, ld = _plain(engine, "y", y, x.rows, w.rows)
    check(lib().t0b_fp4_gemm(engine._h, _mat(engine, w), _mat(engine, x), _bias(engine, "bias", bias, w.rows), ty, p,
                             ld, _stream(engine, stream)))
    return y


def glu(engine, w: Fp4Matrix, x: Fp4Matrix, z, bias=None, stream=None):
    """z = silu(x . gate^T + bg) * (x . up^T + bu), w = gate rows, then up rows;
    z a tensor [x.rows, w.rows / 2] or an Fp4Matrix of that shape (quantised)."""
    b = _bias(engine, "bias", bias, w.rows)
    if isinstance(z, Fp4Matrix):
        ty, p, ld, zq = 0, None, 0, _mat(engine, z)
    else:
        (ty, p, ld), zq = _plain(engine, "z", z, x.rows, w.rows // 2), None
    check(lib().t0b_fp4_glu(engine._h, _mat(engine, w), _mat(engine, x), b, ty, p, ld, zq, _stream(engine, stream)))
    return z


def linear(engine, w: Fp4Matrix, x: torch.Tensor, xq: Fp4Matrix, y: torch.Tensor, bias=None, stream=None) -> torch.Tensor:
    """y = q(x) . w^T (+ bias): quantisation into xq's memory (whose contents
    afterwards are unspecified) and the product in one call."""
    xt, xp, xld = _plain(engine, "x", x, xq.rows, xq.k)
    ty, p, ld = _plain(engine, "y", y, xq.rows, w.rows)
    check(lib().t0b_fp4_linear(engine._h, _mat(engine, w), xt, xp, xld, _mat(engine, xq),
                               _bias(engine, "bias", bias, w.rows), ty, p, ld, _stream(engine, stream)))
    return y


def mlp(engine, w0: Fp4Matrix, w2: Fp4Matrix, x: torch.Tensor, xq: Fp4Matrix, zq: Fp4Matrix, y: torch.Tensor, b0=None,
        b2=None, stream=None) -> torch.Tensor:
    """The gated MLP y = q(silu(q(x) . gate^T + bg) * (q(x) . up^T + bu)) . w2^T + b2
    (the contents of xq and zq afterwards are unspecified)."""
    xt, xp, xld = _plain(engine, "x", x, xq.rows, xq.k)
    ty, p, ld = _plain(engine, "y", y, xq.rows, w2.rows)
    check(lib().t0b_fp4_mlp(engine._h, _mat(engine, w0), _mat(engine, w2), xt, xp, xld, _mat(engine, xq),
                            _mat(engine, zq), _bias(engine, "b0", b0, w0.rows), _bias(engine, "b2", b2, w2.rows), ty, p,
                            ld, _stream(engine, stream)))
    return y


def sync(engine, stream=None) -> None:
    """Wait for the stream and raise any kernel-side error of the engine's 4-bit operators."""
    check(lib().t0b_fp4_sync(engine._h, _stream(engine, stream)))
