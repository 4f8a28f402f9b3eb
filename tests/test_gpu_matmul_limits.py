"""-m gpu: calls of diga_amd/matmul.py at the edge of what it takes."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

import matmul_ref as R
from diga_amd import matmul as M
from diga_amd._lib import DigaError
from test_gpu_matmul import BF16, DEV, E4M3, NothingShort, gen, held, held_weights, rand, sizes_to_offsets

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


@pytest.mark.parametrize("strided", [False, True])
def test_tensors_with_a_tangent_are_refused(strided):
    """Forward-mode differentiation, on the ordinary call and on the one that goes by the Python checks."""
    g = gen(3)
    x, w, r = rand(g, 6, 256).bfloat16(), rand(g, 128).bfloat16(), rand(g, 6, 128).bfloat16()
    x = x[:, :128] if strided else x[:, :128].contiguous()
    q, s = M.quantize_fp8(x)
    wq, ws = M.quantize_weight_fp8(rand(g, 2, 40, 128))
    off = sizes_to_offsets([2, 4])
    w16 = rand(g, 2, 40, 128).bfloat16()
    eps = 1 if strided else 1e-6
    with fwd.dual_level():
        dual = lambda t: fwd.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: M.rms_norm_fp8(dual(x), w, None, eps), lambda: M.rms_norm_fp8(x, dual(w), None, eps), lambda: M.rms_norm_fp8(x, w, dual(r), eps),
                     lambda: M.silu_mul_fp8(dual(x)), lambda: M.quantize_fp8(dual(x)), lambda: M.matmul_fp8(q, dual(s), wq[0], ws[0]),
                     lambda: M.matmul_fp8(q, s, wq[0], dual(ws[0]), torch.float32), lambda: M.grouped_matmul(dual(x), w16, off),
                     lambda: M.grouped_matmul(x, dual(w16), off), lambda: M.grouped_matmul_fp8(q, dual(s), wq, ws, off)):
            with pytest.raises(DigaError, match="tangent"):
                call()
        with torch.no_grad(), pytest.raises(DigaError, match="tangent"):    # (no_grad leaves forward mode on)
            M.quantize_fp8(dual(x))
        p = dual(x)
        assert torch.equal(M.quantize_fp8(fwd.unpack_dual(p).primal)[0].float(), q.float())
        with fwd._set_fwd_grad_enabled(False):
            assert torch.equal(M.quantize_fp8(p)[0].float(), q.float())


@pytest.mark.parametrize("long_way", [False, True])
def test_a_backward_notices_what_was_written_in_place(monkeypatch, long_way):
    if long_way:
        monkeypatch.setattr(M, "_calls", NothingShort())
    g = gen(4)
    x, r, w = rand(g, 6, 128).bfloat16(), rand(g, 6, 128).bfloat16(), torch.ones(128, dtype=BF16, device=DEV)
    q, s = M.quantize_fp8(x)
    wq, ws = M.quantize_weight_fp8(rand(g, 2, 128, 128))
    w16, off = rand(g, 2, 128, 128).bfloat16(), sizes_to_offsets([2, 4])
    fp32 = torch.float32
    for dtype, write in [(BF16, lambda t: M.rms_norm_fp8(x, w, r, 1e-6, t)), (BF16, lambda t: M.rms_norm_fp8(t, w, r, 1e-6, t)), (BF16, lambda t: M.matmul_fp8(q, s, wq[0], ws[0], out=t)),
                         (fp32, lambda t: M.matmul_fp8(q, s, wq[0], ws[0], fp32, t)), (BF16, lambda t: M.grouped_matmul_fp8(q, s, wq, ws, off, out=t)),
                         (fp32, lambda t: M.grouped_matmul_fp8(q, s, wq, ws, off, None, fp32, t)), (fp32, lambda t: M.grouped_matmul(x, w16, off, None, fp32, t))]:
        saved, leaf = rand(g, 6, 128).to(dtype), torch.ones(6, 128, dtype=dtype, device=DEV, requires_grad=True)
        loss = (leaf * saved).sum()           # the backward needs `saved` as it is now
        write(saved)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    with torch.inference_mode():
        kept = torch.empty(6, 128, dtype=BF16, device=DEV)
        M.matmul_fp8(q, s, wq[0], ws[0], out=kept)
    again = torch.empty_like(kept)
    M.matmul_fp8(q, s, wq[0], ws[0], out=kept)                          # outside as well: nothing can have saved it
    assert torch.equal(kept, M.matmul_fp8(q, s, wq[0], ws[0], out=again))
