"""-m gpu: every output of the matrix products (diga_amd/matmul.py) within its bound (tests/matmul_bounds.py), the last rows and columns among them."""
import pytest
import torch

import matmul_ref as R
from diga_amd import matmul as M
from matmul_bounds import check_every
from test_gpu_matmul import BF16, DEV, FP16, FP32, GROUPS, PRODUCTS, gen, held, held_weights, rand, sizes_to_offsets

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m, n, k", [*PRODUCTS, (517, 999, 2050), (2741, 1000, 520)])
@pytest.mark.parametrize("t", [BF16, FP16, FP32])
def test_matmul_fp8_every_output(m, n, k, t):
    g = gen(m + 3 * n + 5 * k)
    xq, xs = held(g, m, k, t == FP16)
    wq, ws = held_weights(g, n, k)
    ws *= 0.02
    check_every(M.matmul_fp8(xq, xs, wq, ws, t), R.rows_of(xq, xs), R.weights_of(wq, ws), t != FP32)


def check_groups(got, x, w, off, rows=None, fp8=False, what=""):
    """The groups' rows against one product each; indices outside take rows of zeros."""
    for e in range(w.shape[0]):
        a, b = off[e], off[e + 1]
        xe = x[a:b]
        if rows is not None:
            r = rows[a:b].long()
            xe = torch.where(((r >= 0) & (r < x.shape[0]))[:, None], x[r.clamp(0, x.shape[0] - 1)], 0.0)
        if a < b:
            check_every(got[a:b], xe, w[e], fp8, what=what)


@pytest.mark.parametrize("sizes, n, k", GROUPS)
@pytest.mark.parametrize("kind", ["fp8", "fp8 to fp32", "bf16", "fp16"])
@pytest.mark.parametrize("gather", [False, True])
def test_grouped_every_output(sizes, n, k, kind, gather):
    g = gen(sum(sizes) + n + k)
    t = sum(sizes) + 3
    xr = max(1, t // 3) if gather else t
    rows = torch.randint(-1, xr + 1, (t,), generator=g, device=DEV, dtype=torch.int32) if gather else None
    off = sizes_to_offsets(sizes)
    if kind.startswith("fp8"):
        xq, xs = held(g, xr, k)
        wq, ws = held_weights(g, len(sizes), n, k)
        got = M.grouped_matmul_fp8(xq, xs, wq, ws, off, rows, BF16 if kind == "fp8" else FP32)
        x, w = R.rows_of(xq, xs), R.weights_of(wq, ws)
    else:
        xi, wi = (v.to({"bf16": BF16, "fp16": FP16}[kind]) for v in (rand(g, xr, k), rand(g, len(sizes), n, k)))
        got, x, w = M.grouped_matmul(xi, wi, off, rows), xi.double(), wi.double()
    check_groups(got, x, w, off.tolist(), rows, kind == "fp8")
