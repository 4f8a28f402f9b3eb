"""-m gpu: 8-bit products with 32-bit outputs (diga_amd/matmul.py) against plain 64-bit forms.

Tolerance: tests/matmul_ref.py's of products summed in 32 bits.  The operands become bf16 without an error; the matrix pipe keeps 24
bits below the largest of 8 products, so each of a block's 128 products costs at most 2^-23 of the largest, two of them the place
of the other's rounding; a block then takes one FMA and the product of its two scales."""
import pytest
import torch

import matmul_ref as R
from diga_amd import matmul as M
from test_gpu_matmul import BF16, DEV, E4M3, FP32, GROUPS, PRODUCTS, check_groups, gen, held, held_weights, rand, sizes_to_offsets

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m, n, k", [*PRODUCTS, (2048, 2050, 1032), (3000, 1500, 384)])
@pytest.mark.parametrize("odd", [False, True])
def test_matmul_fp8_to_fp32(m, n, k, odd):
    g = gen(m + 3 * n + 5 * k)
    xq, xs = held(g, m, k, odd)
    wq, ws = held_weights(g, n, k)
    out = None
    if odd:                                   # an output inside a wider one, its rows not on 16 bytes
        wide = torch.full((m, n + 7), -7.0, device=DEV)
        out = wide[:, 3 : 3 + n]
    got = M.matmul_fp8(xq, xs, wq, ws, FP32, out)
    assert got.dtype == FP32 and got.shape == (m, n)
    R.check_product(got, R.rows_of(xq, xs), R.weights_of(wq, ws))
    if out is not None:
        assert got is out and (wide[:, :3] == -7).all() and (wide[:, 3 + n :] == -7).all()
    assert torch.equal(got, M.matmul_fp8(xq, xs, wq, ws, FP32))


@pytest.mark.parametrize("sizes, n, k", GROUPS)
@pytest.mark.parametrize("gather", [False, True])
def test_grouped_fp8_to_fp32(sizes, n, k, gather):
    g = gen(sum(sizes) + n + k)
    e, used = len(sizes), sum(sizes)
    t = used + 3                              # rows behind the last group
    xr = max(1, t // 3) if gather else t
    rows = torch.randint(0, xr, (t,), generator=g, device=DEV, dtype=torch.int32) if gather else None
    if gather and used > 4:
        rows[1], rows[used - 1] = -1, xr      # indices outside: rows of zeros
    off = sizes_to_offsets(sizes)
    before = torch.full((t, n), -3.0, device=DEV)
    out = before.clone()
    xq, xs = held(g, xr, k, odd_rows=gather)
    wq, ws = held_weights(g, e, n, k)
    assert M.grouped_matmul_fp8(xq, xs, wq, ws, off, rows, FP32, out) is out
    check_groups(out, before, R.rows_of(xq, xs), R.weights_of(wq, ws), off.tolist(), rows)


@pytest.mark.parametrize("m", [1, 20, 70, 600])
def test_every_e4m3_value_comes_through(m):
    codes = torch.arange(256, dtype=torch.uint8, device=DEV)
    codes[[0x7F, 0xFF]] = 0                   # the NaNs
    x = codes.view(E4M3).expand(m, 256).contiguous()
    w = torch.eye(256, device=DEV).to(E4M3)
    xs, ws = torch.full((m, 2), 2.0 ** -3, device=DEV), torch.ones(2, 2, device=DEV)
    assert torch.equal(M.matmul_fp8(x, xs, w, ws, FP32), x.float() * 2.0 ** -3)
    assert torch.equal(M.matmul_fp8(w, ws.repeat_interleave(128, 0), x, torch.full((-(-m // 128), 2), 2.0 ** -3, device=DEV), FP32), x.t().float() * 2.0 ** -3)
    x.view(torch.uint8)[m - 1, 255] = 0xFF
    got = M.matmul_fp8(x, xs, w, ws, FP32)
    assert torch.isnan(got[m - 1]).all() and torch.isfinite(got[: m - 1]).all()


def test_products_that_cancel_keep_24_bits():
    """256 * 256 - 256 * 256 + 2^-4 * 2^-4 side by side: the least part is 2^-24 of the largest."""
    m, k = 300, 256
    x, w = torch.zeros(m, k, device=DEV), torch.zeros(64, k, device=DEV)
    x[:, 8], x[:, 9], x[:, 10] = 256.0, -256.0, 2.0 ** -4
    w[:, 8], w[:, 9], w[:, 10] = 256.0, 256.0, 2.0 ** -4
    ones = lambda r: torch.ones(r, 2, device=DEV)  # noqa: E731
    for rows in (1, 33, m):
        got = M.matmul_fp8(x[:rows].to(E4M3), ones(rows), w.to(E4M3), ones(1), FP32)
        assert (got == 2.0 ** -8).all()


def test_fp32_outputs_in_a_graph_and_empty():
    g = gen(5)
    xq, xs = held(g, 70, 520)
    wq, ws = held_weights(g, 3, 200, 520)
    off = sizes_to_offsets([30, 0, 40])
    run = lambda: (M.matmul_fp8(xq, xs, wq[0], ws[0], FP32), M.grouped_matmul_fp8(xq, xs, wq, ws, off, out_dtype=FP32))  # noqa: E731
    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run()
    for _ in range(3):
        xs.mul_(1.5)
        torch.cuda.synchronize()
        graph.replay()
        want = run()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
    empty = M.matmul_fp8(xq[:0], xs[:0], wq[0], ws[0], FP32)
    assert empty.shape == (0, 200) and empty.dtype == FP32
    half = M.matmul_fp8(xq, xs, wq[0], ws[0], BF16)           # the 16-bit output, of the e4m3 pipe, is the same to its rounding and that pipe's cut
    off = (half.double() - run()[0].double()).norm() / run()[0].double().norm()
    assert off <= 2.0 ** -8 + 2.0 ** -12
