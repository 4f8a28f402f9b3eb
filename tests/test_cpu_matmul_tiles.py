"""CPU-only: which tile the products' rule takes, so that the GPU tests' sizes go on reaching every one."""
import threading

import pytest

from diga_amd._lib import DigaError, call
from matmul_tiles import TAKEN, TILES, codes


@pytest.mark.parametrize("kind", TAKEN)
def test_every_tile_is_taken_by_the_tests_sizes(kind):
    assert len(TILES) == 12
    for tile, (groups, m, n, k) in enumerate(TAKEN[kind]):
        assert call("diga_matmul_tile_of", *codes(kind), groups, m, m, n, k) == tile, (tile, groups, m, n, k)


def test_an_asked_tile_is_taken_by_the_calling_thread_only():
    size = (3, 0, 0, 100, 100, 200, 300)
    rule = call("diga_matmul_tile_of", *size)
    seen = []
    try:
        for tile in range(12):
            call("diga_matmul_use_tile", tile)
            assert call("diga_matmul_tile_of", *size) == tile
        other = threading.Thread(target=lambda: seen.append(call("diga_matmul_tile_of", *size)))
        other.start()
        other.join()
        with pytest.raises(DigaError, match="too many tiles"):          # (no 256 x 256 tile for sums of 32 bits)
            call("diga_matmul_tile_of", 3, 2, *size[2:])
        for bad in (-2, 12):
            with pytest.raises(DigaError, match="diga_matmul_use_tile"):
                call("diga_matmul_use_tile", bad)
    finally:
        call("diga_matmul_use_tile", -1)
    assert seen == [rule] and call("diga_matmul_tile_of", *size) == rule


@pytest.mark.parametrize("args, message", [
    ((2, 0, 1, 1, 1, 1, 1), "unknown type 2"), ((0, 0, 0, 1, 1, 1, 1), "0 groups"), ((3, 0, 4097, 1, 1, 1, 1), "4097 groups"), ((3, 0, 0, 0, 1, 1, 1), "M=0"),
    ((3, 0, 0, 1, 1, 0, 1), "N=0"), ((0, 0, 1, 1, 1, 1, (1 << 22) + 1), "K="), ((3, 0, 0, 1 << 30, 1 << 30, 1 << 20, 16), "too many tiles"),
])
def test_tile_of_refuses(args, message):
    with pytest.raises(DigaError, match=message):
        call("diga_matmul_tile_of", *args)
