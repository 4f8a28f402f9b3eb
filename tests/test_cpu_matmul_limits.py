"""CPU-only: calls of diga_amd/matmul.py that must be refused although each of their tensors looks right."""
import pytest
import torch

from diga_amd import matmul as M
from diga_amd._lib import DigaError

E4M3 = torch.float8_e4m3fn
WRAP = 1 << 32                                # a 32-bit count of WRAP + n reads n


def meta(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device="meta")


@pytest.mark.parametrize("call", [
    lambda: M.quantize_fp8(meta(1, WRAP + 128)),
    lambda: M.silu_mul_fp8(meta(1, 2 * WRAP + 256)),
    lambda: M.rms_norm_fp8(meta(1, WRAP + 128), meta(WRAP + 128)),
    lambda: M.matmul_fp8(meta(1, WRAP + 128, dtype=E4M3), meta(1, WRAP // 128 + 1, dtype=torch.float32), meta(64, WRAP + 128, dtype=E4M3),
                         meta(1, WRAP // 128 + 1, dtype=torch.float32)),
    lambda: M.matmul_fp8(meta(1, 128, dtype=E4M3), meta(1, 1, dtype=torch.float32), meta(WRAP + 64, 128, dtype=E4M3), meta(WRAP // 128 + 1, 1, dtype=torch.float32)),
    lambda: M.grouped_matmul(meta(1, WRAP + 8), meta(2, 8, WRAP + 8), meta(3, dtype=torch.int32)),
    lambda: M.grouped_matmul(meta(1, 8), meta(2, WRAP + 8, 8), meta(3, dtype=torch.int32)),
    lambda: M.grouped_matmul(meta(1, 8), meta(WRAP + 2, 8, 8), meta(WRAP + 3, dtype=torch.int32)),
])
def test_counts_that_pass_32_bits_are_refused(call):
    with pytest.raises(DigaError, match="more than 2.31 - 1"):
        call()
