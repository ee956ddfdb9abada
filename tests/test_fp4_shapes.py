"""CPU checks of the 4-bit matrices' shapes as Python gives them."""
import pytest
import torch

from t0_web_b200 import fp4
from t0_web_b200._lib import T0bError

WIDE = [(2 ** 32 + 4, 32), (4, 2 ** 32 + 32), (-2 ** 32 + 4, 32), (4, 2 ** 64 + 32), (2 ** 31, 1), (1, 2 ** 31)]


@pytest.mark.parametrize("rows,k", WIDE)
def test_shapes_past_32_bits_have_no_size(rows, k):
    assert fp4.code_bytes(rows, k) == 0
    assert fp4.scale_bytes("mx", rows, k) == 0 and fp4.scale_bytes("nv", rows, k) == 0


@pytest.mark.parametrize("rows,k", WIDE)
def test_shapes_past_32_bits_are_refused(rows, k):
    codes, scales = torch.zeros(64, dtype=torch.uint8), torch.zeros(512, dtype=torch.uint8)  # what [4, 32] needs
    with pytest.raises(T0bError, match="empty or too large"):
        fp4.Fp4Matrix("mx", rows, k, codes, scales)
    with pytest.raises(T0bError, match="empty or too large"):
        fp4.Fp4Matrix.empty("mx", rows, k, "cpu")
