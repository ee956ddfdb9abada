"""CPU checks of the 4-bit operators: sizes, refusals, and the oracle against hand-worked blocks."""
import ctypes as C

import numpy as np
import pytest
import torch

import fp4_oracle as O
from t0_web_b200 import fp4
from t0_web_b200._lib import FP4_MX, FP4_NV, T0B_ERR_INVALID, Fp4, T0bError, lib


def test_sizes():
    assert fp4.code_bytes(3, 33) == 3 * 32 and fp4.code_bytes(1, 1) == 16
    assert fp4.scale_bytes("mx", 1, 1) == 512 and fp4.scale_bytes("mx", 129, 129) == 4 * 512
    assert fp4.scale_bytes("nv", 128, 64) == 512 and fp4.scale_bytes("nv", 128, 65) == 1024
    for rows, k in ((0, 5), (5, 0), (-1, 5), (5, -1), (1 << 30, 1), (1, (1 << 20) + 1)):
        assert fp4.code_bytes(rows, k) == 0 and fp4.scale_bytes("mx", rows, k) == 0
    assert lib().t0b_fp4_scale_bytes(7, 4, 4) == 0
    # sizes past 32 bits
    assert fp4.code_bytes((1 << 30) - 1, 1 << 20) == ((1 << 30) - 1) * (1 << 19)


@pytest.mark.parametrize("call", ["quantize", "dequantize", "gemm", "glu", "linear", "mlp", "sync"])
def test_null_engine_is_refused(call):
    m = Fp4(FP4_MX, 4, 4, 1.0, 0, 0)
    r, n = C.byref(m), None
    args = dict(quantize=(0, n, 4, r, n), dequantize=(r, 0, n, 4, n), gemm=(r, r, n, 0, n, 4, n),
                glu=(r, r, n, 0, n, 4, n, n), linear=(r, 0, n, 4, r, n, 0, n, 4, n),
                mlp=(r, r, 0, n, 4, r, r, n, n, 0, n, 4, n), sync=(n,))[call]
    assert getattr(lib(), "t0b_fp4_" + call)(None, *args) == T0B_ERR_INVALID
    assert b"engine is NULL" in lib().t0b_last_error()


def test_matrix_refusals():
    codes, scales = torch.zeros(16 * 4, dtype=torch.uint8), torch.zeros(512, dtype=torch.uint8)
    for args in (("e4m3", 4, 4, codes, scales), ("mx", 0, 4, codes, scales), ("mx", 4, 4, codes[1:], scales),
                 ("mx", 4, 4, codes, scales[:-1]), ("mx", 4, 4, codes.float(), scales), ("mx", 4, 4, codes, scales)):
        with pytest.raises(T0bError):  # the last: not on a CUDA device
            fp4.Fp4Matrix(*args)


def test_header_names_the_formats():
    import os
    import re
    src = open(os.path.join(os.path.dirname(__file__), "..", "include", "t0b.h")).read()
    assert dict(re.findall(r"(T0B_FP4_[MN][XV]) = (\d)", src)) == {"T0B_FP4_MX": str(FP4_MX), "T0B_FP4_NV": str(FP4_NV)}


def test_oracle_by_hand():
    # every midpoint goes to the even index; 5.0 -> 4, above 6 saturates
    x = np.zeros((1, 32))
    x[0, :9] = [4, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 7.9]
    byte, code = O.quantize(x, "mx")
    assert byte[0, 0] == 127 and list(code[0, :9]) == [6, 0, 2, 2, 4, 4, 6, 6, 7]
    assert list(O.values(byte, code, "mx")[0, :9]) == [4, 0, 1, 1, 2, 2, 4, 4, 6]
    byte, code = O.quantize(-x[:, :16], "nv", 2.0 ** -3)
    assert byte[0, 0] == np.argmin(abs(O.E4M3[:127] - 7.9 / 0.75)) and code[0, 8] == 15
    b2, c2 = O.unpack(*O.pack(byte, code, "nv"), 1, 16, "nv")
    assert np.array_equal(b2, byte) and np.array_equal(c2, code)
    assert O.quantize(np.full((1, 3), np.inf), "mx")[0][0, 0] == 255
    assert O.quantize(np.array([[1, np.nan]]), "nv")[0][0, 0] == 127
