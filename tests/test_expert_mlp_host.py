"""The block's buffers and what comes before their first use, without a GPU."""

import pytest
import torch

import expert_mlp
import ien

CTX = type("Context", (), dict(h=None, device=0))()


class Experts:
    def __init__(self, ctx, experts, c, n, gated=False):
        self.ctx, self.experts, self.c, self.n, self.h = ctx, experts, c, n // 2 if gated else n, None


class Router:
    def __init__(self, ctx, w, bias):
        self.k, self.n = w.shape


@pytest.fixture
def seen(monkeypatch):
    """What a run does, in order: tensors made, waits for torch's stream, the framework's calls."""
    seen = []

    def logged(name, f):
        return lambda *a, **k: (seen.append(name), f(*a, **k))[1]

    stream = type("Stream", (), dict(cuda_stream=4096, synchronize=lambda self: seen.append("wait")))()
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: stream)
    for name in ("zeros", "empty", "empty_like"):
        monkeypatch.setattr(torch, name, logged("made", getattr(torch, name)))
    monkeypatch.setattr(ien, "Matrix", Router)
    monkeypatch.setattr(ien, "Experts8", Experts)
    monkeypatch.setattr(ien, "expert_parts", lambda routes, matrix, dtype: torch.empty(8))
    for name in ("rms_norm", "multiply_ex", "route", "experts_in8", "experts_out8"):
        monkeypatch.setattr(ien, name, logged("call", lambda *a, **k: None))
    monkeypatch.setattr(ien, "rows_input", lambda x, stride: None)
    return seen


class OnGpu(torch.Tensor):
    """A host tensor that says it is on GPU 0."""

    def get_device(self):
        return 0


def rows(tokens, c=24):
    return torch.zeros(tokens, c, dtype=torch.float16).as_subclass(OnGpu)


def block(c=24):
    return expert_mlp.ExpertMlp8(CTX, c, 2, None, (torch.zeros(c, 4).numpy(), None), (4, c, 64), (4, 32, c))


def test_nothing_made_is_used_before_torchs_stream_is_done_with_it(seen):
    """The first run of a size, a later one with a new result, and one that makes nothing."""
    b, x = block(), rows(6)
    for out, makes in ((x, True), (None, True), (x, False)):
        seen.clear()
        b.run(x, out=out)
        assert ("made" in seen) == makes and "call" in seen
        if makes:
            last = max(i for i, name in enumerate(seen) if name == "made")
            assert "wait" in seen[last:seen.index("call")], seen
        else:
            assert "wait" not in seen


def test_what_is_refused_leaves_nothing(seen):
    """Rows that are not on the context's GPU, or not the block's: nothing of theirs is kept, and the same number of tokens
    runs afterwards."""
    b = block()
    for x in (torch.zeros(6, 24, dtype=torch.float16), rows(6, 23), rows(6)[0], rows(6)[:, None]):
        with pytest.raises(ValueError):
            b.run(x)
        assert not b._work and "call" not in seen
    b.run(rows(6))
    assert list(b._work) == [(6, torch.float16)] and "call" in seen
