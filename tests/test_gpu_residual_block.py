"""The residual block that runs group norm into 8 bits and 8-bit convolutions
together, against its steps in 64 bits.

Values next to a border of e4m3 may fall on its other side (f32 statistics),
which moves a value by a sixteenth: the map between the halves is compared by
its norm, 2^-11 for its own rounding and 2^-10 for those; the result likewise."""

import numpy as np
import pytest

import eight_bits as E

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("images,h,w,c,groups", [(1, 16, 24, 128, 32), (2, 13, 9, 96, 8), (1, 40, 33, 256, 16)])
def test_residual_block(ctx, images, h, w, c, groups):
    import torch

    from residual_block import ResidualBlock8

    rng = np.random.default_rng(c)
    x = rng.standard_normal((images * h * w, c)).astype(np.float16)
    convs = [((rng.standard_normal((9 * c, c)) / np.sqrt(9 * c)).astype(np.float32), rng.standard_normal(c).astype(np.float32))
             for _ in range(2)]
    gains = [((1 + 0.2 * rng.standard_normal(c)).astype(np.float32), rng.standard_normal(c).astype(np.float32))
             for _ in range(2)]
    block = ResidualBlock8(ctx, c, groups, [tuple(torch.from_numpy(g).cuda() for g in p) for p in gains], convs)
    xt = torch.from_numpy(x).cuda()
    y = block.run(xt, images, h, w).double().cpu().numpy()
    again = block.run(xt, images, h, w, torch.empty_like(xt)).double().cpu().numpy()
    assert np.array_equal(y, again)

    def half(v, gain, conv):
        n, _ = E.group_norm(v, images, groups, *gain, 1e-5, "silu")
        q = E.values(*E.quantize(n), c)
        return E.patches(q, images, h, w, 1) @ E.weights(conv[0], 9) + conv[1]

    mid = half(x, gains[0], convs[0]).astype(np.float16)
    want = x.astype(np.float64) + half(mid, gains[1], convs[1])
    assert np.linalg.norm(y - want) <= (2.0**-11 + 2.0**-10) * np.linalg.norm(want)
    block.free()


def test_the_command(ctx, capsys):
    """Both operands of a product are off by at most a sixteenth of themselves,
    evenly spread: some 4% of a sum, 6% after two in a row."""
    import residual_block
    import torch

    assert residual_block.main(20, 28, 128, 32) < 0.1
    assert "us a block" in capsys.readouterr().out
    assert torch.cuda.current_stream() == ctx.stream  # (the command's own context left it as it was)
