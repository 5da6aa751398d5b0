"""The sizes of the launches of the 8-bit entry points and of the norm (host code,
no GPU): a launch counts its lanes in 32 bits, whatever sizes it is for."""

import ctypes

import pytest

from internal import _function

LANES = 1 << 32  # the first count that no launch can have


@pytest.mark.parametrize("blocks", [1, 16, 17, 393216, 2**24, 2**28 - 16, 2**28 - 15, 2**28, 2**28 + 1, 2**40, 2**62])
def test_quantize8(blocks):
    grid = _function("_ZN3ien14quantize8_gridEl", ctypes.c_long, restype=ctypes.c_uint)(blocks)
    assert 1 <= grid and grid * 256 < LANES
    assert grid == min(-(-blocks // 16), 1 << 20)  # one turn, but for more than 2 GiB of blocks


class NormPlan(ctypes.Structure):
    """eight_bits.h NormPlan."""
    _fields_ = [(n, ctypes.c_long) for n in ("one", "span", "px", "chunks", "chunk", "lanes", "groups", "images")]


CUS, WORKSPACE = 256, 8 << 20  # MI355X; the context's workspace in floats


def norm_plan(images, pixels, c, groups, y_bytes):
    f = _function("_ZN3ien9norm_planEillliii", ctypes.c_int, ctypes.c_long, ctypes.c_long, ctypes.c_long, ctypes.c_int,
                  ctypes.c_int, ctypes.c_int, restype=NormPlan)
    return f(CUS, WORKSPACE, images, pixels, c, groups, y_bytes)


@pytest.mark.parametrize("y_bytes", [1, 2, 4])
@pytest.mark.parametrize("c,groups", [(1, 1), (7, 1), (8, 1), (64, 8), (512, 32), (640, 32), (2056, 8), (4090, 10), (4104, 1), (8184, 1023),
                                      (8191, 8191), (8192, 1), (8192, 64), (8192, 1024), (8192, 8192)])
def test_group_norm(c, groups, y_bytes):
    for images in (1, 2, 255, 256, 257, 65535, 65536, 65537, 2**20 - 1):
        for pixels in (1, 2, 8, 9, 512, 513, 5000, 2**20 + 1, 2**32, 2**40 - 1):
            p = norm_plan(images, pixels, c, groups, y_bytes)
            assert 1 <= p.images <= images and 64 <= p.lanes <= 1024 and p.lanes % 64 == 0
            assert p.images * p.groups * p.lanes < LANES
            assert p.chunks * p.chunk >= pixels and (p.chunks - 1) * p.chunk < pixels
            assert p.span % (c // groups) == 0 and c % p.span == 0
            if p.one:
                assert p.groups == c // p.span and p.px * -(-p.span // 8) <= p.lanes
                assert 68 * p.lanes + 8 * p.span // (c // groups) <= 160 << 10  # LDS
            else:
                assert p.groups == p.chunks and p.chunk <= 1 << 30 and 8 * p.lanes + 8 * groups <= 160 << 10
                # (One image's parts fit the workspace, but where no card's memory holds it.)
                if pixels * c < 2**40:
                    assert 2 * p.images * p.chunks * groups <= WORKSPACE


def multiply8_plan(rows, n, chunks, exact, add):
    choice = _function("_ZN3ien16multiply8_choiceEilllibb", ctypes.c_int, ctypes.c_long, ctypes.c_long, ctypes.c_long,
                       ctypes.c_int, ctypes.c_bool, ctypes.c_bool)
    tile, splits = divmod(choice(CUS, WORKSPACE, rows, n, chunks, exact, add), 64)
    return tile, splits, _function("_ZN3ien14multiply8_partEil", ctypes.c_int, ctypes.c_long, restype=ctypes.c_long)(tile, n)


@pytest.mark.parametrize("exact", [False, True])
@pytest.mark.parametrize("add", [False, True])
def test_multiply8(exact, add):
    tiles = [(256, 256), (128, 128), (64, 128), (64, 64)]
    for rows in (1, 64, 65, 4096, 2**20, 2**24, 2**27 + 1, 2**30, 2**33, 2**40 - 1):
        for n in (1, 8, 64, 65, 129, 8192, 100000, 2**22 - 1):
            for chunks in (1, 9, 64, 1000):
                tile, splits, part = multiply8_plan(rows, n, chunks, exact, add)
                tm, tn = tiles[tile]
                assert part >= tm and part % tm == 0
                across = -(-n // tn)
                assert -(-min(part, rows) // tm) * across * splits * 512 < LANES
                if -(-rows // tm) * across <= 2**21:
                    assert part >= rows  # one launch


def test_a_part_of_a_norm_for_each_cu():
    for pixels, c, chunks in ((6144, 640, 256), (16384, 512, 256), (4096, 512, 128), (131072, 64, 256)):
        assert norm_plan(1, pixels, c, 32, 2).chunks == chunks
    assert norm_plan(4, 16384, 512, 32, 2).chunks == 64
