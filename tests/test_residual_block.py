"""The residual block's buffers, without a GPU: what a captured run works in stays
the block's when another size is run."""

import functools
import weakref

import torch

import ien


def test_buffers_of_a_size_stay(monkeypatch):
    import residual_block

    used = []
    monkeypatch.setattr(ien, "Rows8", functools.partial(ien.Rows8, device="cpu"))
    monkeypatch.setattr(ien, "Matrix8", lambda *a, **k: None)
    monkeypatch.setattr(ien, "group_norm", lambda ctx, x, images, groups, gamma, beta, y, **k: used.append(y.data))
    monkeypatch.setattr(ien, "conv8", lambda ctx, q, images, h, w, m, out, **k: used.append(out))
    block = residual_block.ResidualBlock8(None, 40, 8, [(None, None)] * 2, [(None, None)] * 2)

    def buffers(rows):
        used.clear()
        block.run(torch.zeros(rows, 40, dtype=torch.float16), 1, 1, rows)
        q, h, again, out = used
        assert again is q and h.shape == (rows, 40) and h.dtype == torch.float16 and q.shape[0] == rows
        return q.data_ptr(), h.data_ptr(), weakref.ref(q), weakref.ref(h)

    first, second = buffers(30), buffers(40)
    used.clear()
    assert all(b[i]() is not None for b in (first, second) for i in (2, 3))
    assert buffers(30)[:2] == first[:2] and buffers(40)[:2] == second[:2]
