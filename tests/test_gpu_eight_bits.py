"""Rows in 8 bits and their products against their definitions in 64 bits.

What is written in 8 bits is compared bit for bit.  Products of small whole
numbers under power-of-two scales are exact in f32 whatever the order of the
sums, so those outputs are compared for equality; those of real numbers to
half a step of the output (2^-11 of the value in f16, 2^-24 in f32) and one
step of f32 for each sum, 2^-23 k times the sum of the products' magnitudes.
"""

import numpy as np
import pytest

import eight_bits as E

pytestmark = pytest.mark.gpu

ACTS = {"none": 0, "relu": 1, "gelu": 2, "sigmoid": 4, "silu": 5}


def cuda(x):
    import torch

    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def strided(x, extra, fill=float("nan")):
    """x (numpy rows) on the GPU, `extra` more columns between its rows."""
    import torch

    t = torch.full((x.shape[0], x.shape[1] + extra), fill, dtype=cuda(x[:1]).dtype, device="cuda")
    t[:, :x.shape[1]] = cuda(x)
    return t[:, :x.shape[1]]


def rows8_of(data, scales, k, extra=0):
    """Bytes and scales as the library takes them; bytes past the row's blocks are NaN."""
    import ien
    import torch

    d = torch.full((data.shape[0], data.shape[1] + extra), 127, dtype=torch.uint8, device="cuda")
    d[:, :data.shape[1]] = cuda(data)
    s = torch.full((data.shape[0], 4 * -(-scales.shape[1] // 4)), 255, dtype=torch.uint8, device="cuda")
    s[:, :scales.shape[1]] = cuda(scales)
    return ien.Rows8(data.shape[0], k, data=d[:, :data.shape[1]], scales=s)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("rows,k,extra", [(1, 1, 0), (3, 128, 0), (5, 127, 0), (7, 129, 3), (77, 768, 0), (33, 640, 8),
                                          (2, 5000, 0), (1000, 96, 0), (4099, 264, 8), (1, 8192, 0)])
def test_quantize8(ctx, dtype, rows, k, extra):
    import ien
    import torch

    rng = np.random.default_rng(rows + k)
    x = (rng.standard_normal((rows, k)) * 2.0 ** rng.integers(-12, 12, (rows, k))).astype(dtype)
    x.flat[:: 11] = 0
    want, scales = E.quantize(x)
    q = ien.Rows8(rows, k)
    q.data.fill_(99)
    ien.quantize8(ctx, strided(x, extra), q)
    assert np.array_equal(q.data.cpu().numpy(), want)
    assert np.array_equal(q.scales[:, :scales.shape[1]].cpu().numpy(), scales)
    y = torch.empty(rows, k, dtype=torch.float32, device="cuda")
    ien.dequantize8(ctx, q, y)
    assert np.array_equal(y.cpu().numpy(), E.values(want, scales, k).astype(np.float32))
    wide = torch.full((rows, k + extra), 7.0, dtype=torch.float16, device="cuda")
    ien.dequantize8(ctx, q, wide[:, :k])
    with np.errstate(over="ignore"):
        assert np.array_equal(wide[:, :k].cpu().numpy(), E.values(want, scales, k).astype(np.float16))
    assert bool((wide[:, k:] == 7.0).all())


def test_quantize8_every_half(ctx):
    """Every f16 value alone in its block, and beside the largest one."""
    import ien

    h = np.arange(65536, dtype=np.uint16).view(np.float16).astype(np.float32)
    for beside in (0.0, 65504.0, 1.0):
        x = np.zeros((65536, 2), np.float32)
        x[:, 0], x[:, 1] = h, beside
        want, scales = E.quantize(x)
        for t in (cuda(x), cuda(x.astype(np.float16))):
            q = ien.Rows8(65536, 2)
            ien.quantize8(ctx, t, q)
            got = q.data.cpu().numpy()
            nan = np.isnan(E.E4M3[want])
            assert np.array_equal(np.isnan(E.E4M3[got]), nan) and np.array_equal(got[~nan], want[~nan])
            assert np.array_equal(q.scales[:, :1].cpu().numpy(), scales)


def test_quantize8_ends_of_f32(ctx):
    """Subnormal, largest and infinite values: the scale goes by the finite
    ones, at least 2^-127."""
    import ien

    top = np.finfo(np.float32).max
    x = np.zeros((8, 130), np.float32)
    x[0, :3] = [1e-45, -3e-45, 1.2e-38]
    x[1, :3] = [top, -top, 1.0]
    x[2, :3] = [np.inf, 2.0, -3.0]
    x[3, :3] = [np.nan, -np.inf, 0.0]
    x[4, 5], x[4, 129] = 448.0, 449.0
    x[5, 7], x[5, 128] = 1.75 * 2.0**-100, np.nextafter(np.float32(1.75 * 2.0**-100), np.float32(1))
    x[6, :2] = [2.0**-118, 2.0**-140]
    x[7, 128] = -0.0
    want, scales = E.quantize(x)
    q = ien.Rows8(8, 130)
    ien.quantize8(ctx, cuda(x), q)
    nan = np.isnan(E.E4M3[want])
    got = q.data.cpu().numpy()
    assert np.array_equal(np.isnan(E.E4M3[got]), nan) and np.array_equal(got[~nan], want[~nan])
    assert np.array_equal(q.scales[:, :2].cpu().numpy(), scales)


def whole_rows(rng, rows, k):
    """Whole numbers within 4 as bytes, under scales of 1 or 2 a block."""
    v = rng.integers(-4, 5, (rows, k)).astype(np.float64)
    blocks = -(-k // 128)
    data = E.to_bytes(np.concatenate([v, np.zeros((rows, -k % 128))], 1))
    return data, rng.integers(127, 129, (rows, blocks)).astype(np.uint8)


def whole_weights(rng, taps, c, n):
    """Whole numbers within 4 (exact in 8 bits), mostly small sums."""
    return rng.integers(-4, 5, (taps * c, n)).astype(np.float32)


def check_whole(ctx, rng, x, data, scales, k, w, taps, outs, call, f16=True):
    """f32 outputs equal to the whole numbers, f16 ones to their rounding."""
    import ien
    import torch

    n = w.shape[1]
    b = rng.integers(-9, 10, n).astype(np.float32)
    add = rng.integers(-9, 10, (outs, n)).astype(np.float32)
    m = ien.Matrix8(ctx, w, b, taps=taps)
    want = x @ E.weights(w, taps) + b + add
    assert np.abs(want).max() < 2**24
    q = rows8_of(data, scales, k, 16)
    for dtype in (torch.float32, torch.float16):
        for extra in (0, 3):
            y = torch.full((outs, n + extra), 5.0, dtype=dtype, device="cuda")
            call(q, m, y[:, :n], strided(add.astype(np.float16 if dtype == torch.float16 else np.float32), extra))
            got = y[:, :n].float().cpu().numpy()
            with np.errstate(over="ignore"):
                assert np.array_equal(got, want.astype(np.float16 if dtype == torch.float16 else np.float32).astype(np.float32))
            assert bool((y[:, n:] == 5.0).all())
    m.free()


# One row, a few, odd ones and many; k inside, at and past a block's end; n of one output,
# odd ones, and over the widest tile; deep sums.
ROWS = [(1, 1, 1), (1, 128, 128), (2, 130, 3), (1, 1280, 5120), (5, 64, 40), (17, 384, 96), (31, 2000, 77),
        (33, 257, 256), (64, 512, 8), (100, 1152, 136), (128, 128, 128), (129, 129, 129), (200, 4096, 64),
        (257, 1000, 520), (1000, 300, 33), (4096, 384, 1536), (3, 9000, 24), (700, 2048, 264), (2049, 640, 1288)]


@pytest.mark.parametrize("rows,k,n", ROWS)
def test_multiply8_whole_numbers(ctx, rows, k, n):
    import ien

    rng = np.random.default_rng(rows * 7 + k + n)
    data, scales = whole_rows(rng, rows, k)
    x = E.values(data, scales, k)
    w = whole_weights(rng, 1, k, n)
    check_whole(ctx, rng, x, data, scales, k, w, 1, rows,
                lambda q, m, y, add: ien.multiply8(ctx, q, m, y, add=add))


MAPS = [(1, 1, 1, 1, 16, 8), (1, 1, 1, 2, 16, 8), (2, 3, 5, 1, 40, 24), (3, 5, 3, 2, 130, 40), (1, 1, 300, 1, 64, 16),
        (1, 300, 1, 2, 64, 16), (2, 7, 9, 2, 128, 128), (1, 64, 64, 1, 128, 64), (1, 33, 47, 1, 256, 136),
        (1, 40, 56, 2, 320, 320), (4, 16, 16, 1, 512, 256), (1, 85, 125, 1, 96, 128), (5, 2, 2, 1, 640, 3)]


@pytest.mark.parametrize("taps", [9, 1])
@pytest.mark.parametrize("images,h,w,step,c,n", MAPS)
def test_conv8_whole_numbers(ctx, taps, images, h, w, step, c, n):
    import ien

    rng = np.random.default_rng(h * w + c + n)
    data, scales = whole_rows(rng, images * h * w, c)
    x = E.values(data, scales, c)
    x = E.patches(x, images, h, w, step) if taps == 9 else \
        x.reshape(images, h, w, c)[:, ::step, ::step].reshape(-1, c)
    check_whole(ctx, rng, x, data, scales, c, whole_weights(rng, taps, c, n), taps, x.shape[0],
                lambda q, m, y, add: ien.conv8(ctx, q, images, h, w, m, y, step=step, add=add))


@pytest.mark.parametrize("dtype", ["float16", "float32"])
@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("rows,k,n", [(1, 300, 72), (65, 512, 136), (300, 1280, 320), (1500, 200, 260)])
def test_multiply8_real_numbers(ctx, rows, k, n, act, dtype):
    import ien
    import torch

    rng = np.random.default_rng(k + n)
    data, scales = E.quantize(rng.standard_normal((rows, k)) * 2.0 ** rng.integers(-6, 6, (rows, 1)))
    w = (rng.standard_normal((k, n)) / np.sqrt(k)).astype(np.float32)
    b = rng.standard_normal(n).astype(np.float32)
    m = ien.Matrix8(ctx, w, b)
    y = torch.empty(rows, n, dtype=getattr(torch, dtype), device="cuda")
    ien.multiply8(ctx, rows8_of(data, scales, k), m, y, act=ACTS[act])
    x, w8 = E.values(data, scales, k), E.weights(w, 1)
    v = x @ w8 + b
    want = E.activate(v, act)
    # The sums' error through the activation, the activation's own (exponentials
    # of arguments off by one step: |v| 2^-23 of the value; the error function to 4
    # steps) and the output's rounding (below f16's smallest normal, half of 2^-24).
    half = 2.0**-11 if dtype == "float16" else 2.0**-24
    tol = (E.SLOPE[act] * (k + 2) * 2.0**-23 * (np.abs(x) @ np.abs(w8) + np.abs(b))
           + (4 + np.abs(v)) * 2.0**-23 * np.abs(want) + half * np.abs(want) + (2.0**-25 if half == 2.0**-11 else 0)
           + (4 * 2.0**-23 * np.abs(v) if act == "gelu" else 2.0**-23))
    assert (np.abs(y.double().cpu().numpy() - want) <= tol).all()
    m.free()


def test_multiply8_weights_in_f16_and_no_bias(ctx):
    import ien
    import torch

    rng = np.random.default_rng(1)
    data, scales = whole_rows(rng, 70, 140)
    w = whole_weights(rng, 1, 140, 24)
    q = rows8_of(data, scales, 140)
    for weights in (w, w.astype(np.float16)):
        m = ien.Matrix8(ctx, weights)
        y = torch.empty(70, 24, device="cuda")
        ien.multiply8(ctx, q, m, y)
        assert np.array_equal(y.cpu().numpy(), (E.values(data, scales, 140) @ w).astype(np.float32))


@pytest.mark.parametrize("taps,shape,c,n", [(1, (1, 1, 900), 700, 200), (9, (2, 31, 29), 256, 72)])
def test_multiply8_part_of_the_rows(ctx, taps, shape, c, n):
    """Rows row0 .. alone, onto their place of a map: the bits of the whole
    product, and nothing outside them."""
    import ien
    import torch

    rng = np.random.default_rng(c)
    rows = shape[0] * shape[1] * shape[2]
    data, scales = E.quantize(rng.standard_normal((rows, c)))
    q = rows8_of(data, scales, c)
    m = ien.Matrix8(ctx, rng.standard_normal((taps * c, n)).astype(np.float32), taps=taps)
    whole = torch.empty(rows, n, device="cuda")
    run = (lambda y, r: ien.multiply8(ctx, q, m, y, row0=r)) if taps == 1 else \
        (lambda y, r: ien.conv8(ctx, q, *shape, m, y, row0=r))
    run(whole, 0)
    for r, count in ((0, 1), (17, 300), (rows - 5, 5), (rows, 0)):
        y = torch.full((rows + 2, n), 9.0, device="cuda")
        run(y[r + 1:r + 1 + count], r)
        # (Tiles and splits of the sums go by the rows of a call: f32 sums of other orders.)
        near = torch.allclose(y[r + 1:r + 1 + count], whole[r:r + count], rtol=2.0**-23 * taps * c, atol=2.0**-23 * taps * c * 40)
        assert near and bool((y[:r + 1] == 9.0).all()) and bool((y[r + 1 + count:] == 9.0).all())


def test_multiply8_in_place_and_again(ctx):
    """add = out accumulates; the same call on the same inputs gives the same
    bits (deep sums in splits among them)."""
    import ien
    import torch

    rng = np.random.default_rng(2)
    for rows, k, n in ((64, 9216, 64), (1, 5120, 1280), (3000, 512, 512)):
        data, scales = E.quantize(rng.standard_normal((rows, k)))
        q = rows8_of(data, scales, k)
        m = ien.Matrix8(ctx, rng.standard_normal((k, n)).astype(np.float32))
        old = torch.randn(rows, n, device="cuda").half()
        want = torch.empty_like(old)
        ien.multiply8(ctx, q, m, want, add=old, act=ien.ACT_SILU)
        for _ in range(5):
            y = old.clone()
            ien.multiply8(ctx, q, m, y, add=y, act=ien.ACT_SILU)
            assert torch.equal(y, want)


def test_multiply8_nan_and_infinity_stay_in_their_row(ctx):
    import ien
    import torch

    rng = np.random.default_rng(3)
    x = rng.standard_normal((300, 300)).astype(np.float32)
    x[7, 299], x[150, 0] = np.nan, np.inf
    w = rng.standard_normal((300, 96)).astype(np.float32)
    w[5, 40] = np.nan
    m = ien.Matrix8(ctx, w)
    q = ien.Rows8(300, 300)
    ien.quantize8(ctx, cuda(x), q)
    y = torch.empty(300, 96, device="cuda")
    ien.multiply8(ctx, q, m, y)
    want = np.zeros((300, 96), bool)
    want[[7, 150]] = want[:, 40] = True
    assert np.array_equal(np.isnan(y.cpu().numpy()), want)


def test_multiply8_scales_far_apart(ctx):
    """Blocks under scales from 2^-60 to 2^60 of the rows and of the weights."""
    import ien
    import torch

    rng = np.random.default_rng(4)
    data, _ = whole_rows(rng, 40, 512)
    scales = rng.integers(67, 188, (40, 4)).astype(np.uint8)
    w = whole_weights(rng, 1, 512, 48) * np.repeat(2.0 ** rng.integers(-60, 60, (4, 48)), 128, 0).astype(np.float32)
    y = torch.empty(40, 48, device="cuda")
    ien.multiply8(ctx, rows8_of(data, scales, 512), ien.Matrix8(ctx, w), y)
    x, w8 = E.values(data, scales, 512), E.weights(w, 1)
    tol = 514 * 2.0**-23 * (np.abs(x) @ np.abs(w8))
    assert (np.abs(y.double().cpu().numpy() - x @ w8) <= tol).all()


def test_multiply8_other_stream_and_graph(ctx):
    """A call on another stream of the context, and one in a captured graph that
    is replayed with eager work in between (the split sums' counters return to
    zero in the kernels)."""
    import ien
    import torch

    rng = np.random.default_rng(5)
    cases = []
    for rows, k, n in ((64, 9216, 64), (1, 2560, 640), (1500, 512, 256)):
        data, scales = E.quantize(rng.standard_normal((rows, k)))
        q = rows8_of(data, scales, k)
        m = ien.Matrix8(ctx, rng.standard_normal((k, n)).astype(np.float32))
        want = torch.empty(rows, n, device="cuda").half()
        ien.multiply8(ctx, q, m, want)
        cases.append((q, m, want))
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    L = ien.load()
    ys = [torch.zeros_like(c[2]) for c in cases]
    torch.cuda.synchronize()
    try:
        ien.check(L.ien_set_stream(ctx.h, other.cuda_stream))
        for (q, m, _), y in zip(cases, ys):
            ien.multiply8(ctx, q, m, y)
        other.synchronize()
        assert all(torch.equal(y, c[2]) for y, c in zip(ys, cases))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=other):
            for (q, m, _), y in zip(cases, ys):
                ien.multiply8(ctx, q, m, y)
    finally:
        ien.check(L.ien_set_stream(ctx.h, None))
    for _ in range(4):
        for y in ys:
            y.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(y, c[2]) for y, c in zip(ys, cases))
        again = torch.empty_like(ys[0])
        ien.multiply8(ctx, cases[0][0], cases[0][1], again)
        torch.cuda.synchronize()
        assert torch.equal(again, cases[0][2])
