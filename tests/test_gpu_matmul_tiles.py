"""-m gpu: every tile of the matrix products, at the sizes for which the rule takes it and, asked for, around each change of its loop: K steps, a last one
that ends inside its 128 bytes, rows and columns that leave waves without outputs, uneven and gathered groups."""
import pytest
import torch

import matmul_ref as R
from diga_amd import matmul as M
from diga_amd._lib import DigaError, call
from matmul_bounds import check_every
from matmul_tiles import TAKEN, TILES, codes
from test_gpu_matmul import BF16, DEV, FP16, FP32, gen, held, held_weights, rand, sizes_to_offsets
from test_gpu_matmul_every import check_groups

pytestmark = pytest.mark.gpu


@pytest.fixture
def use_tile():
    yield lambda tile: call("diga_matmul_use_tile", tile)
    call("diga_matmul_use_tile", -1)


def product(kind, m, n, k, sizes, gather, what):
    """One product of this kind, checked at every output; what lies round the result stays as it was."""
    fp8, g = "fp8" in kind, gen(m + 3 * n + 5 * k)
    out_t = {"fp8": BF16, "fp8 to fp32": FP32, "bf16": BF16, "fp16": FP16}[kind.removeprefix("grouped ")]
    wide = torch.full((m + 1, n + 5), -7.0, dtype=out_t, device=DEV)
    out = wide[:m, 2 : 2 + n]
    if not sizes:
        xq, xs = held(g, m, k, odd_rows=gather)
        wq, ws = held_weights(g, n, k)
        ws *= 0.05
        M.matmul_fp8(xq, xs, wq, ws, out_t, out)
        check_every(out, R.rows_of(xq, xs), R.weights_of(wq, ws), out_t != FP32, what=what)
    else:
        xr = max(1, 2 * m // 3) if gather else m
        rows = torch.randint(-1, xr + 1, (m,), generator=g, device=DEV, dtype=torch.int32) if gather else None
        off, e = sizes_to_offsets(sizes), len(sizes)
        if fp8:
            xq, xs = held(g, xr, k)
            wq, ws = held_weights(g, e, n, k)
            ws *= 0.05
            M.grouped_matmul_fp8(xq, xs, wq, ws, off, rows, out_t, out)
            x, w = R.rows_of(xq, xs), R.weights_of(wq, ws)
        else:
            kp = -(-k // 8) * 8                # what lies behind a row must not matter
            xi, wi = (torch.full((*s, kp), float("nan"), dtype=out_t, device=DEV)[..., :k] for s in ((xr,), (e, n)))
            xi.copy_(rand(g, xr, k))
            wi.copy_(0.05 * rand(g, e, n, k))
            M.grouped_matmul(xi, wi, off, rows, out_t, out)
            x, w = xi.double(), wi.double()
        check_groups(out, x, w, off.tolist(), rows, fp8 and out_t != FP32, what)
        assert (out[sum(sizes) :] == -7).all(), what
    assert (wide[:, :2] == -7).all() and (wide[:, 2 + n :] == -7).all() and (wide[m] == -7).all(), what


@pytest.mark.parametrize("tile", range(12))
@pytest.mark.parametrize("kind", TAKEN)
def test_tile_that_the_rule_takes(kind, tile):
    if tile == len(TAKEN[kind]):
        return
    groups, m, n, k = TAKEN[kind][tile]
    assert call("diga_matmul_tile_of", *codes(kind), groups, m, m, n, k) == tile
    sizes = [(m + g) // groups for g in range(groups)]
    if groups and m // groups > 8:             # uneven ones of the same number
        sizes[0] += sizes[1] // 3
        sizes[1] -= sizes[1] // 3 + 2
    for gather in ([False, True] if groups and k < 1500 else [False]):
        product(kind, m, n, k, sizes, gather, (tile, kind, gather))


@pytest.mark.parametrize("tile", range(12))
@pytest.mark.parametrize("kind", TAKEN)
def test_tile_at_its_edges(use_tile, kind, tile):
    bm, bn, steps = TILES[tile]
    use_tile(tile)
    if "fp32" in kind and tile == 11:
        with pytest.raises(DigaError, match="too many tiles"):
            product(kind, 300, 300, 128, [100, 200] if "grouped" in kind else [], False, "refused")
        return
    step = 128 if "fp8" in kind else 64
    for nk in steps:
        for k in (nk * step, nk * step - step + (16 if nk % 2 else 5), nk * step - 3):
            what = (tile, kind, k)
            if "grouped" not in kind:
                for m, n in ((1, 1), (bm, bn), (2 * bm + 17, 2 * bn + 33), (bm - 3, 3 * bn - 5)):
                    product(kind, m, n, k, [], nk == steps[-1], (*what, m, n))
            else:
                for sizes, n in (([1], 1), ([bm + 3, 0, 1, 2 * bm, 17], bn + 33), ([0, bm - 1], 2 * bn - 9)):
                    product(kind, sum(sizes) + 2, n, k, sizes, nk % 2 == 0, (*what, sizes, n))
