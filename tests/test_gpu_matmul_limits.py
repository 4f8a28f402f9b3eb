"""-m gpu: calls of diga_amd/matmul.py at the edge of what it takes."""
import pytest
import torch

import matmul_ref as R
from diga_amd import matmul as M
from diga_amd._lib import DigaError
from test_gpu_matmul import BF16, DEV, E4M3, gen, held, held_weights, rand, sizes_to_offsets

pytestmark = pytest.mark.gpu


def test_more_columns_than_32_bits_count_are_refused():
    with pytest.raises(DigaError, match="more than 2.31 - 1"):
        M.quantize_fp8(torch.empty(1, (1 << 32) + 128, dtype=BF16, device=DEV))


def test_outputs_on_operands_are_refused_and_beside_them_are_not():
    g = gen(1)
    x, w = rand(g, 40, 64).bfloat16(), rand(g, 2, 64, 64).bfloat16()
    off = sizes_to_offsets([30, 10])
    want = M.grouped_matmul(x, w, off)
    for out in (x, w.view(-1, 64)[64:104]):
        before = out.clone()
        with pytest.raises(DigaError, match="the output lies on"):
            M.grouped_matmul(x, w, off, out=out)
        assert torch.equal(out, before)
    wide = torch.zeros(40, 3 * 64, dtype=BF16, device=DEV)              # the left rows in the middle of one matrix, outputs on both sides
    wide[:, 64:128] = x
    for at in (0, 128):
        assert torch.equal(M.grouped_matmul(wide[:, 64:128], w, off, out=wide[:, at : at + 64]), want)
        assert torch.equal(wide[:, 64:128], x)
    both = torch.cat([x, torch.zeros_like(x)])                          # one behind the other
    assert torch.equal(M.grouped_matmul(both[:40], w, off, out=both[40:]), want)
    r = rand(g, 40, 64).bfloat16()
    ones = torch.ones(64, dtype=BF16, device=DEV)
    h = M.rms_norm_fp8(x, ones, r)[2]
    pair = torch.cat([x, r], 1)
    with pytest.raises(DigaError, match="lies across"):
        M.rms_norm_fp8(pair[:, :64], ones, pair[:, 64:], residual_out=pair[:, 32:96])
    assert torch.equal(M.rms_norm_fp8(pair[:, :64], ones, pair[:, 64:], residual_out=pair[:, :64])[2], h) and torch.equal(pair[:, :64], h)
    pair = torch.cat([x, r, x], 1)
    assert torch.equal(M.rms_norm_fp8(pair[:, :64], ones, pair[:, 64:128], residual_out=pair[:, 128:])[2], h) and torch.equal(pair[:, :128], torch.cat([x, r], 1))


def test_one_output_row_between_the_rows_of_its_operands():
    g = gen(2)
    xq, xs = held(g, 1, 256)
    wq, ws = held_weights(g, 32, 256)
    want = M.matmul_fp8(xq, xs, wq, ws)
    rows = torch.zeros(32, 384, dtype=torch.uint8, device=DEV)          # 256 bytes of weights and 128 others a row
    rows[:, :256] = wq.view(torch.uint8)
    got = M.matmul_fp8(xq, xs, rows[:, :256].view(E4M3), ws, out=rows[5:6, 256:320].view(BF16))
    assert torch.equal(got, want)
    R.check_product(want, R.rows_of(xq, xs), R.weights_of(wq, ws), True)
    with pytest.raises(DigaError, match="the output lies on the weights"):
        M.matmul_fp8(xq, xs, rows[:, :256].view(E4M3), ws, out=rows[5:6, 240:304].view(BF16))
