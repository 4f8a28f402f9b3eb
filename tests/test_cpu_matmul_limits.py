"""CPU-only: calls of diga_amd/matmul.py that must be refused although each of their tensors looks right."""
import pytest
import torch

from diga_amd import _lib, matmul as M
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


A = 1 << 20                                   # addresses that are never read: every call here is refused before a launch


@pytest.mark.parametrize("change, message", [
    (dict(out=A), "left rows"),
    (dict(out=A + 9 * 512 + 254), "left rows"),                         # the last two bytes of x
    (dict(out=A - 63 * 2), "left rows"),                                # the first two
    (dict(ldo=512, out=A + 256), "left rows"),                          # another stride than x's, inside its range
    (dict(ldo=256, out=A + 512 + 192), "left rows"),                    # x's stride, 64 bytes into its rows
    (dict(ldo=256, out=A + 512 + 448), "left rows"),                    # ... and from the row before
    (dict(M=1, out=A + 254), "left rows"),
    (dict(out=2 * A + 63 * 256 + 254), "weights"),
    (dict(out=2 * A - 9 * 128 - 126), "weights"),
])
def test_products_refuse_outputs_on_their_operands(change, message):
    a = dict(x=A, ldx=512, xs=A, ssm=1, ssb=10, w=2 * A, ldw=256, ws=A, out=3 * A, out_type=0, ldo=64, M=10, N=64, K=256, stream=None)
    a.update(change)
    with pytest.raises(DigaError, match="the output lies on the " + message):
        _lib.call("diga_matmul_fp8", *a.values())
    g = dict(x=a["x"], ldx=a["ldx"] // 2, x_rows=10, type=0, rows=None, w=a["w"], ldw=128, w_stride=64 * 128, offsets=A, groups=2, out=a["out"], out_type=0,
             ldo=a["ldo"], T=a["M"], N=64, K=128, stream=None)
    with pytest.raises(DigaError, match="the output lies on the " + message):
        _lib.call("diga_grouped_matmul", *g.values())
    if "M" not in change and message == "left rows":                    # gathered rows: all of x, however few rows come out
        with pytest.raises(DigaError, match="the output lies on the left rows"):
            _lib.call("diga_grouped_matmul", *{**g, "rows": A, "T": 1, "ldo": 64, "out": A + 9 * 512}.values())


@pytest.mark.parametrize("change", [
    dict(h=A + 2), dict(h=A, ldh=80), dict(h=2 * A + 64 * 3), dict(h=2 * A, ldh=72), dict(h=3 * A - 9 * 128 - 2), dict(h=A + 128 - 2, M=1), dict(h=3 * A, M=1),
])
def test_norm_refuses_a_sum_written_across_its_inputs(change):
    a = dict(x=A, ldx=64, res=2 * A, ldr=64, type=0, weight=3 * A, wtype=0, eps=1e-6, M=10, N=64, q=5 * A, ldq=64, scale=6 * A, ssm=1, ssb=10, h=4 * A, ldh=64,
             stream=None)
    with pytest.raises(DigaError, match="lies across"):
        _lib.call("diga_rms_norm_fp8", *{**a, **change}.values())


@pytest.mark.parametrize("ldx, x_rows", [(1 << 62, 4), (1 << 32, 1), (1 << 61, 8), ((1 << 32) - 16, 2)])
def test_gathered_rows_beyond_4_gib_are_refused_whatever_their_product_wraps_to(ldx, x_rows):
    a = dict(x=A, ldx=ldx, x_rows=x_rows, xs=A, ssm=1, ssb=4, rows=A, w=2 * A, ldw=256, w_stride=64 * 256, ws=A, offsets=A, groups=2, out=3 * A, out_type=0, ldo=64,
             T=1, N=64, K=256, stream=None)
    with pytest.raises(DigaError, match="at most 4 GiB"):
        _lib.call("diga_grouped_matmul_fp8", *a.values())
