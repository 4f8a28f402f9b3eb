"""CPU-only: what 8-bit products with 32-bit outputs refuse."""
import pytest
import torch

from diga_amd import _lib, matmul as M
from diga_amd._lib import DigaError
from test_cpu_matmul import A, f32, grouped_args, product_args


@pytest.mark.parametrize("change, message", [
    (dict(), "no CPU fallback"), (dict(out=f32(3, 64)), "no CPU fallback"), (dict(out=torch.zeros(3, 64, dtype=torch.bfloat16)), "out must be"),
    (dict(out=f32(64, 3).t()), "out must be"), (dict(xs=f32(3, 1)), "rows' scales"),
])
def test_matmul_fp8_to_fp32_refuses(change, message):
    with pytest.raises(DigaError, match=message):
        M.matmul_fp8(**product_args(out_dtype=torch.float32, **change))


@pytest.mark.parametrize("change, message", [(dict(), "no CPU fallback"), (dict(out=f32(4, 64)), "out must be")])
def test_grouped_matmul_fp8_to_fp32_refuses(change, message):
    with pytest.raises(DigaError, match=message):
        M.grouped_matmul_fp8(**grouped_args(out_dtype=torch.float32, **change))


@pytest.mark.parametrize("change, message", [
    (dict(M=-1), "M=-1"), (dict(N=0), "N=0"), (dict(K=(1 << 23) + 1), "K="), (dict(x=None), "null pointer"), (dict(out=None), "null pointer"),
    (dict(ws=None), "null pointer"), (dict(x=A + 8), "multiples of 16"), (dict(ldw=240), "below K"), (dict(ldo=63), "below N"),
    (dict(M=1 << 30, N=1 << 20, ldo=1 << 20), "too many tiles"),
])
def test_c_matmul_fp8_f32_refuses(change, message):
    a = dict(x=A, ldx=256, xs=A, ssm=1, ssb=4, w=A, ldw=256, ws=A, out=A, ldo=64, M=4, N=64, K=256, stream=None)
    with pytest.raises(DigaError, match="diga_matmul_fp8_f32.*" + message):
        _lib.call("diga_matmul_fp8_f32", *{**a, **change}.values())


@pytest.mark.parametrize("change, message", [
    (dict(groups=0), "0 groups"), (dict(offsets=None), "null pointer"), (dict(x_rows=3), "3 left rows for 4"), (dict(w_stride=63 * 256 - 16), "overlap"),
    (dict(rows=A, T=1, ldx=0), "lie 0 bytes apart"), (dict(w_stride=64 * 256 + 8), "multiples of 16"), (dict(xs=None), "null pointer"),
])
def test_c_grouped_matmul_fp8_f32_refuses(change, message):
    a = dict(x=A, ldx=256, x_rows=4, xs=A, ssm=1, ssb=4, rows=None, w=A, ldw=256, w_stride=64 * 256, ws=A, offsets=A, groups=2, out=A, ldo=64, T=4, N=64,
             K=256, stream=None)
    with pytest.raises(DigaError, match="diga_grouped_matmul_fp8_f32.*" + message):
        _lib.call("diga_grouped_matmul_fp8_f32", *{**a, **change}.values())
