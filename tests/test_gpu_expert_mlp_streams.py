"""First runs of the block's sizes while torch's current stream, which is not the
context's, still has work queued: equal to runs on an idle GPU."""

import numpy as np
import pytest

from test_gpu_eight_bits import cuda
from test_gpu_expert_mlp import block_of, weights_of

pytestmark = pytest.mark.gpu


def test_first_runs_behind_other_work():
    import ien
    import torch

    rng = np.random.default_rng(6)
    own, other = ien.Context(0), ien.Context(0)
    assert torch.cuda.current_stream() == other.stream
    w = weights_of(rng, 100, 160, 6, True)
    block, check = block_of(own, w, 100, 2, True), block_of(own, w, 100, 2, True)
    a = torch.randn(4096, 4096, device="cuda") / 64
    for tokens in (1, 40, 700):
        x = cuda(rng.standard_normal((tokens, 100)).astype(np.float16))
        want = check.run(x)
        torch.cuda.synchronize()
        for out in (torch.zeros_like(x), None):
            torch.cuda.synchronize()
            b = a
            for _ in range(20):
                b = a @ b
            got = block.run(x, out=out)
            torch.cuda.synchronize()
            assert torch.equal(got, want)
    for c in (block, check):
        c.free()
    other.close()
    own.close()
