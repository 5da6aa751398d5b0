"""The second half of a transformer block whose MLP is one of many for each
token, x + sum of weight expert(norm(x)) over the experts that a router chooses:
a root-mean-square norm into f16 and 8 bits, the router's product and choice, and
the experts' two products in 8 bits.

  python image-engine-native_amd/expert_mlp.py [tokens channels hidden experts top]

runs one with random weights on the GPU, and prints how far it is from the block
in f32 and how long it takes.
"""

import pathlib
import sys

if __name__ == "__main__":
    sys.path.insert(0, str(pathlib.Path(__file__).resolve().parent))

import ien


class ExpertMlp8:
    """gamma: the norm's f32 gains (torch, on the GPU; or None).  router: c x
    experts weights and biases of the logits (numpy, kept in f16 and f32; biases
    or None; its product is of the norm in f16).  first, second: the experts' weights and biases, as Experts8 takes
    them (gated: first has 2 hidden columns).  how: the choice, as keywords of
    ien.route.

    The first run of each number of tokens, which is not a captured one, makes
    what lies between its steps; it stays the block's until free(), so a captured
    run has it for as long as the block lives.  A program of many sizes keeps to
    a few, by parts or padding, or frees the block.  An f16 stream is rounded once,
    at its end.  Runs of a number of tokens share it: they follow each other, a
    graph's replays among them."""

    def __init__(self, ctx, c, top, gamma, router, first, second, gated=True, act=ien.ACT_SILU, eps=1e-6, how=None):
        import numpy as np

        self.ctx, self.c, self.top, self.gamma, self.act, self.eps, self.how = ctx, c, top, gamma, act, eps, how or {}
        # (Products over rows take whole 16s of channels: zeros past c, here and in the rows.)
        self.router = ien.Matrix(ctx, np.pad(np.asarray(router[0], np.float16), ((0, -c % 16), (0, 0))), router[1])
        self.first, self.second = ien.Experts8(ctx, *first, gated=gated), ien.Experts8(ctx, *second)
        if not (len(router[0]) == self.first.c == self.second.n == c and self.first.n == self.second.c
                and self.router.n == self.first.experts == self.second.experts):
            raise ValueError(f"a router of {len(router[0])} x {self.router.n}, experts of {self.first.experts} x {self.first.c} x "
                             f"{self.first.n} and {self.second.experts} x {self.second.c} x {self.second.n} for {c} channels")
        self._work = {}  # tokens and type: the norm in f16 and 8 bits, the logits, the routes, the hidden rows, the products

    def run(self, x, add=None, out=None):
        """f16 or f32 rows x channels x (+ add, a branch that joins the stream first), in
        the order of the context's stream, into `out` (or a new tensor; x itself
        too)."""
        import torch

        if x.dim() != 2 or x.shape[1] != self.c or x.get_device() != self.ctx.device:  # (before anything is kept for its size)
            raise ValueError(f"rows of {self.c} channels on GPU {self.ctx.device} expected, not {tuple(x.shape)} on {x.device}")
        tokens, made = x.shape[0], out is None
        out = torch.empty_like(x) if made else out
        if tokens == 0:
            return out
        key = tokens, x.dtype
        if key not in self._work:
            routes = ien.Routes(tokens, self.first.experts, self.top, device=x.device)
            self._work[key] = (torch.zeros(tokens, self.router.k, dtype=torch.float16, device=x.device),
                               ien.Rows8(tokens, self.c, device=x.device),
                               torch.empty(tokens, self.router.n, dtype=torch.float32, device=x.device), routes,
                               ien.Rows8(tokens * self.top, self.first.n, device=x.device),
                               ien.expert_parts(routes, self.second, torch.float32))
            made = True
        if made:
            ien.settle(self.ctx)
        norm, q, logits, routes, hidden, parts = self._work[key]
        ien.rms_norm(self.ctx, x, self.gamma, norm[:, :self.c], q, add=add, eps=self.eps)
        ien.multiply_ex(self.ctx, ien.rows_input(norm, self.router.k), 0, tokens, self.router, logits, self.router.n, out_f32=True)
        ien.route(self.ctx, logits, routes, **self.how)
        ien.experts_in8(self.ctx, q, routes, self.first, hidden, act=self.act)
        # (The two addends again, not their sum as x's type: an f16 stream is rounded once.)
        ien.experts_out8(self.ctx, hidden, routes, self.second, parts, out, add=x, branch=add)
        return out

    def free(self):
        self._work.clear()
        for m in (self.router, self.first, self.second):
            m.free()


def main(tokens=4096, c=384, hidden=768, experts=16, top=2):
    import numpy as np
    import torch
    import torch.nn.functional as F

    ctx = ien.Context(0)
    g = torch.Generator(device="cuda")
    g.manual_seed(0)
    rand = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    gamma = 1 + 0.2 * rand(c)
    router = (rand(c, experts) / c**0.5).half()
    first = rand(experts, c, 2 * hidden) / c**0.5, 0.1 * rand(experts, 2 * hidden)
    second = rand(experts, hidden, c) / hidden**0.5, 0.1 * rand(experts, c)
    x = rand(tokens, c).half()
    block = ExpertMlp8(ctx, c, top, gamma, (router.cpu().numpy(), None), first, second)
    y = block.run(x)

    n = x.float() * torch.rsqrt((x.float() ** 2).mean(1, keepdim=True) + block.eps) * gamma
    index = block._work[tokens, x.dtype][3].index.long()  # (the same experts: two that are close may be chosen either way)
    weight = torch.softmax((n.half().float() @ router.float()).gather(1, index), 1)
    branch = torch.zeros_like(n)
    for e in range(experts):
        t, slot = torch.nonzero(index == e, as_tuple=True)
        v = n[t] @ first[0][e] + first[1][e]
        v = F.silu(v[:, :hidden]) * v[:, hidden:]
        branch[t] += weight[t, slot, None] * (v @ second[0][e] + second[1][e])
    error = ((y.float() - x.float() - branch).norm() / branch.norm()).item()

    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    for _ in range(20):
        block.run(x, out=y)
    start.record()
    for _ in range(200):
        block.run(x, out=y)
    end.record()
    torch.cuda.synchronize()
    print(f"{tokens} x {c}, {top} of {experts} experts of {hidden}: {start.elapsed_time(end) * 5:.1f} us a block, its branch "
          f"{100 * error:.1f}% from the one in f32")
    block.free()
    ctx.close()
    return error


if __name__ == "__main__":
    main(*map(int, sys.argv[1:]))
