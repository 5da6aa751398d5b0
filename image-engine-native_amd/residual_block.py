"""A residual block of an image decoder or U-Net with its convolutions in 8
bits, x + conv(silu(norm(conv(silu(norm(x)))))): group norms that write rows
in 8 bits, and 3 x 3 convolutions of those.

  python image-engine-native_amd/residual_block.py [height width channels groups]

runs one with random weights on the GPU, and prints how far it is from the
block in f32 and how long it takes.
"""

import pathlib
import sys

if __name__ == "__main__":
    sys.path.insert(0, str(pathlib.Path(__file__).resolve().parent))

import ien


class ResidualBlock8:
    """The weights (f32 or f16 numpy, (9 c) x c with the taps row-major and
    the channels fastest, and c biases) of two convolutions, quantised once,
    and the f32 gains (gamma, beta: torch, on the GPU) of two group norms.

    The first run of each number of rows makes the two maps between its steps
    (3 c bytes a row, and the scales); they stay the block's until free(), so a
    captured run has them for as long as the block lives.  Runs share them:
    like all calls of a context, which share its workspace, those of one block
    follow each other, a graph's replays among them."""

    def __init__(self, ctx, c, groups, norms, convs, eps=1e-5):
        self.ctx, self.c, self.groups, self.norms, self.eps = ctx, c, groups, norms, eps
        self.convs = [ien.Matrix8(ctx, w, b, taps=9) for w, b in convs]
        self._work = {}  # rows: the map in 8 bits, the map between the halves

    def run(self, x, images, height, width, out=None):
        """f16 or f32 rows x channels (a pixel a row, one map after the other)
        into `out` (or a new tensor; not x itself), in the order of the
        context's stream."""
        import torch

        rows = x.shape[0]
        if rows not in self._work:
            self._work[rows] = (ien.Rows8(rows, self.c, device=x.device),
                                torch.empty(rows, self.c, dtype=torch.float16, device=x.device))
        q, h = self._work[rows]
        out = torch.empty_like(x) if out is None else out
        shape = images, height, width
        ien.group_norm(self.ctx, x, images, self.groups, *self.norms[0], q, eps=self.eps, act=ien.ACT_SILU)
        ien.conv8(self.ctx, q, *shape, self.convs[0], h)
        ien.group_norm(self.ctx, h, images, self.groups, *self.norms[1], q, eps=self.eps, act=ien.ACT_SILU)
        ien.conv8(self.ctx, q, *shape, self.convs[1], out, add=x)
        return out

    def free(self):
        self._work.clear()
        for m in self.convs:
            m.free()


def main(height=64, width=64, c=512, groups=32):
    import numpy as np
    import torch
    import torch.nn.functional as F

    ctx = ien.Context(0)
    rng = np.random.default_rng(0)
    convs = [((rng.standard_normal((9 * c, c)) / np.sqrt(9 * c)).astype(np.float32),
              (0.1 * rng.standard_normal(c)).astype(np.float32)) for _ in range(2)]
    norms = [(1 + 0.2 * torch.randn(c, device="cuda"), 0.2 * torch.randn(c, device="cuda")) for _ in range(2)]
    x = torch.randn(height * width, c, device="cuda").half()
    block = ResidualBlock8(ctx, c, groups, norms, convs)
    y = block.run(x, 1, height, width)

    branch = x.float().t().reshape(1, c, height, width)
    for (w, b), (gamma, beta) in zip(convs, norms):
        branch = F.silu(F.group_norm(branch, groups, gamma, beta))
        w = torch.from_numpy(w).cuda().reshape(3, 3, c, c).permute(3, 2, 0, 1)
        branch = F.conv2d(branch, w, torch.from_numpy(b).cuda(), padding=1)
    want = branch.reshape(c, -1).t()
    error = ((y.float() - x.float() - want).norm() / want.norm()).item()

    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    for _ in range(20):
        block.run(x, 1, height, width, y)
    start.record()
    for _ in range(200):
        block.run(x, 1, height, width, y)
    end.record()
    torch.cuda.synchronize()
    print(f"{height} x {width} x {c}: {start.elapsed_time(end) * 5:.1f} us a block, its branch {100 * error:.1f}% from the "
          "one in f32")
    block.free()
    ctx.close()
    return error


if __name__ == "__main__":
    main(*map(int, sys.argv[1:]))
