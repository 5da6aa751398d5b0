"""The tile and the splits of an 8-bit product, chosen on the host."""

import ctypes

import pytest

import ien
from test_gpu_multiply8_tiles import CASES

CUS, WORKSPACE = 256, 8 << 20
TILES = [(256, 256), (128, 128), (64, 128), (64, 64)]


def choice(rows, n, chunks, exact=False, add=False, workspace=WORKSPACE):
    """(tile, splits)."""
    f = ien.load()._ZN3ien16multiply8_choiceEilllibb
    f.argtypes = [ctypes.c_int, ctypes.c_long, ctypes.c_long, ctypes.c_long, ctypes.c_int, ctypes.c_bool, ctypes.c_bool]
    return divmod(f(CUS, workspace, rows, n, chunks, exact, add), 64)


@pytest.mark.parametrize("exact", [False, True])
@pytest.mark.parametrize("add", [False, True])
def test_choices_are_launchable(exact, add):
    for rows in (1, 2, 63, 64, 65, 300, 4096, 10625, 98304, 1 << 20, 1 << 33):
        for n in (1, 64, 129, 1536, 8192):
            for chunks in (1, 2, 9, 36, 72, 1000):
                for workspace in (0, WORKSPACE):
                    tile, splits = choice(rows, n, chunks, exact, add, workspace)
                    tm, tn = TILES[tile]
                    tiles = -(-rows // tm) * -(-n // tn)
                    assert splits >= 1 and (splits == 1 or tiles * splits * tm * tn <= workspace)
                    deep = -(-chunks // splits)  # every split has blocks to add
                    assert (splits - 1) * deep < chunks


def test_choices():
    assert choice(8192, 8192, 64)[0] == 0  # matrix-bound: the largest tile
    assert choice(64, 64, 72)[1] > 1  # one tile: its depth in splits
    assert choice(4096, 512, 36) == (2, 1)  # a tile for every CU
    assert choice(98304, 256, 18, add=True) == (1, 1)  # residuals under another workgroup's products


def test_the_gpu_tests_take_every_tile():
    for add in (False, True):
        taken = {choice(rows, n, -(-k // 128), add=add)[0] for rows, k, n in CASES}
        assert taken >= ({1, 2, 3} if add else {0, 1, 2, 3})
