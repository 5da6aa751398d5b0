"""That the GPU tests of the 8-bit products take every path that a size chooses."""

from test_eight_bits_launches import multiply8_plan
from test_gpu_multiply8_paths import MAPS, ROWS

# Tiles 0 .. 3: 256 x 256, 128 x 128, 64 x 128, 64 x 64.


def paths(cases):
    """{(exact, add, tile, in splits)} of (rows, n, blocks deep)."""
    out = set()
    for exact in (False, True):
        for add in (False, True):
            for case in cases:
                tile, splits, _ = multiply8_plan(*case, exact, add)
                out.add((exact, add, tile, splits > 1))
    return out


# (Exact sums with a residual take no tile of 256 x 256: see below.)
WHOLE = {(e, a, t, False) for e in (False, True) for a in (False, True) for t in range(4)} - {(True, True, 0, False)}


def test_rows():
    split = {(e, a, t, True) for e in (False, True) for a in (False, True) for t in (1, 2, 3)}
    assert paths([(r, n, -(-k // 128)) for r, k, n in ROWS]) == WHOLE | split


def test_maps():
    got = paths([(b * -(-h // s) * -(-w // s), n, 9 * -(-c // 128)) for b, h, w, s, c, n in MAPS])
    assert got >= WHOLE and any(s for _, _, _, s in got)


def test_no_exact_residual_of_the_largest_tile():
    for rows in (4096, 16384, 2**17, 2**20, 2**24):
        for n in (264, 512, 2048, 8192, 65536):
            for chunks in (1, 4, 16, 64, 256, 1000):
                assert multiply8_plan(rows, n, chunks, True, True)[0] != 0
