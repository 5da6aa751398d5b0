"""Every tile of the 8-bit products, whole and with its depth in splits, with a
residual and without, of rows and of maps, with fast and with exact sums.

Products of whole numbers within 4 under scales of 1 and 2: their sums are under
2^24 and exact whatever their order, and no product lies 2^7 under a neighbour, so
the fast sums are exact too."""

import pytest

pytestmark = pytest.mark.gpu

# (rows, k, n)
ROWS = [(5981, 128, 1288), (65530, 4000, 136), (32769, 128, 264), (16390, 256, 2056), (8299, 24000, 200), (5554, 8000, 72), (5557, 6000, 72),
        (1001, 128, 2056), (501, 100, 2056), (1, 16000, 2056), (3, 8000, 4096), (3, 2000, 24), (1, 16, 8)]
# (images, height, width, step, c, n)
MAPS = [(2, 129, 127, 1, 128, 264), (1, 255, 257, 1, 200, 136), (1, 254, 258, 1, 128, 136), (1, 91, 90, 1, 128, 200), (4, 182, 90, 2, 120, 72),
        (1, 131, 126, 1, 100, 264), (3, 40, 31, 2, 256, 40), (1, 3, 3, 1, 128, 24), (1, 9, 7, 1, 520, 24)]


def whole(rows, c, taps, n):
    """Whole rows and weights on the GPU: bytes, scales, their values, numpy weights."""
    import numpy as np
    import torch

    import eight_bits as E

    g = torch.Generator(device="cuda").manual_seed(rows + c + n)
    v = torch.randint(-4, 5, (rows, c), generator=g, device="cuda")
    table = torch.from_numpy(E.to_bytes(np.arange(-4.0, 5.0))).cuda()
    blocks = -(-c // 128)
    data = torch.zeros(rows, 128 * blocks, dtype=torch.uint8, device="cuda")
    data[:, :c] = table[v + 4]
    scales = torch.full((rows, 4 * -(-blocks // 4)), 255, dtype=torch.uint8, device="cuda")
    scales[:, :blocks] = torch.randint(127, 129, (rows, blocks), generator=g, device="cuda").to(torch.uint8)
    x = v.double() * (scales[:, :blocks].double() - 126).repeat_interleave(128, 1)[:, :c]
    w = np.random.default_rng(c + n).integers(-4, 5, (taps * c, n)).astype(np.float32)
    return data, scales, x, w


def check(ctx, rows, c, n, taps, want_of, call):
    import ien
    import torch

    data, scales, x, w = whole(rows, c, taps, n)
    want = want_of(x, torch.from_numpy(w).cuda().double())
    del x
    outs = want.shape[0]
    bias = torch.arange(n, device="cuda") % 17 - 8
    old = torch.arange(outs * n, device="cuda").reshape(outs, n) % 23 - 11
    q, m = ien.Rows8(rows, c, data=data, scales=scales), ien.Matrix8(ctx, w, bias.float().cpu().numpy(), taps=taps)
    want += bias
    for add in (False, True):
        if add:
            want += old
        assert bool((want.abs() < 2**24).all())
        for dtype, exact in ((torch.float16, False), (torch.float16, True), (torch.float32, True)):
            y = torch.full((outs, n + 5), float("nan"), dtype=dtype, device="cuda")
            call(q, m, y[:, :n], dict(exact=exact, add=old.to(dtype) if add else None))
            assert torch.equal(y[:, :n], want.float().to(dtype)) and bool(y[:, n:].isnan().all())
    m.free()


@pytest.mark.parametrize("rows,k,n", ROWS)
def test_rows(ctx, rows, k, n):
    import ien

    check(ctx, rows, k, n, 1, lambda x, w: x @ w, lambda q, m, y, more: ien.multiply8(ctx, q, m, y, **more))


@pytest.mark.parametrize("images,h,w,step,c,n", MAPS)
def test_maps(ctx, images, h, w, step, c, n):
    import ien
    import torch

    def want_of(x, weights):
        p = torch.zeros(images, h + 2, w + 2, c, dtype=torch.float64, device="cuda")
        p[:, 1:-1, 1:-1] = x.reshape(images, h, w, c)
        return sum(p[:, t // 3:t // 3 + h:step, t % 3:t % 3 + w:step].reshape(-1, c) @ weights[t * c:(t + 1) * c].contiguous()
                   for t in range(9))

    check(ctx, images * h * w, c, n, 9, want_of, lambda q, m, y, more: ien.conv8(ctx, q, images, h, w, m, y, step=step, **more))
