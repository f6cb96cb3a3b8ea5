"""What the embedding, the 8-bit product and the draft verification refuse,
and their collectives: no GPU needed."""

from __future__ import annotations

import types

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from nmce import _lib as L
    return L.load()


def test_embedding_argument_errors_before_launch(lib):
    p = 4096  # a fake, aligned device address; never dereferenced
    fwd = lib.nmce_embedding_fwd
    assert fwd(p, 4, p, 7, 8, 8, 8, 0, 1.0, p, 0, 8, None) == -1
    assert fwd(p, 4, p, 0, 8, 8, 8, 0, 1.0, p, 2, 8, None) == -1
    assert fwd(p, -1, p, 0, 8, 8, 8, 0, 1.0, p, 0, 8, None) == -2
    assert fwd(p, 4, p, 0, 0, 8, 8, 0, 1.0, p, 0, 8, None) == -2
    assert fwd(p, 4, p, 0, 8, 0, 8, 0, 1.0, p, 0, 8, None) == -2
    assert fwd(p, 4, p, 0, 8, 8, 7, 0, 1.0, p, 0, 8, None) == -2
    assert fwd(p, 4, p, 0, 8, 8, 8, 0, 1.0, p, 0, 7, None) == -2
    assert fwd(p, 1 << 31, p, 0, 8, 8, 8, 0, 1.0, p, 0, 8, None) == -2
    assert fwd(p, 4, p, 0, 1 << 31, 8, 8, 0, 1.0, p, 0, 8, None) == -2
    assert fwd(p + 4, 4, p, 0, 8, 8, 8, 0, 1.0, p, 0, 8, None) == -3
    assert fwd(p, 4, p + 2, 0, 8, 8, 8, 0, 1.0, p, 0, 8, None) == -3
    assert fwd(p, 4, p, 1, 8, 8, 8, 0, 1.0, p + 1, 1, 8, None) == -3
    assert fwd(None, 4, p, 0, 8, 8, 8, 0, 1.0, p, 0, 8, None) == -4
    assert fwd(p, 4, p, 0, 8, 8, 8, 0, 1.0, None, 0, 8, None) == -4
    assert fwd(None, 0, None, 0, 8, 8, 8, 0, 1.0, None, 0, 8, None) == 0
    bwd, size = lib.nmce_embedding_bwd, lib.nmce_embedding_bwd_workspace_bytes
    ws = size(4, 8, 8)
    assert ws > 0 and size(-1, 8, 8) == size(4, 0, 8) == size(4, 8, 0) == size(1 << 31, 8, 8) == -1
    assert size(0, 8, 8) >= 0 and size((1 << 31) - 1, 8, 8) > 0
    assert bwd(p, 4, p, 3, 8, 8, 8, 0, 1.0, p, 0, p, ws, None) == -1
    assert bwd(p, 4, p, 0, 7, 8, 8, 0, 1.0, p, 0, p, ws, None) == -2
    assert bwd(p, 4, p, 0, 8, 8, 8, 0, 1.0, p + 8, 0, p, ws, None) == -3
    assert bwd(p, 4, None, 0, 8, 8, 8, 0, 1.0, p, 0, p, ws, None) == -4
    assert bwd(p, 4, p, 0, 8, 8, 8, 0, 1.0, None, 0, p, ws, None) == -4
    assert bwd(p, 4, p, 0, 8, 8, 8, 0, 1.0, p, 0, p, ws - 1, None) == -6
    assert bwd(p, 4, p, 0, 8, 8, 8, 0, 1.0, p, 0, None, ws, None) == -6
    assert bwd(p, 4, p, 0, 8, 8, 8, 0, 1.0, p, 0, p + 8, ws, None) == -6


def test_embedding_refusals():
    import nmce
    ctx = nmce.ParallelContext.single()
    w, t = torch.randn(10, 8), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="no CPU path"):
        nmce.vocab_parallel_embedding(t, w, 0, 10, ctx)
    with pytest.raises(RuntimeError, match="no CPU path"):
        nmce._VocabParallelEmbedding.apply(w, t, 0, 10, 1.0, torch.float32)
    cfg = types.SimpleNamespace(vocab_size=1001, n_embd=8)
    two = nmce.ParallelContext(rank=1, world_size=2, tp_size=2, tp_rank=1, pp_size=1, pp_rank=0,
                               dp_size=1, dp_rank=0)
    with pytest.raises(ValueError, match="not divisible"):
        nmce.VocabParallelEmbedding(cfg, two)
    cfg.vocab_size = 1000
    emb = nmce.VocabParallelEmbedding(cfg, two)
    assert emb.weight.shape == (500, 8) and emb.weight.tensor_parallel_sharded is True
    assert emb.vocab_range() == (500, 1000)
    with pytest.raises(RuntimeError, match="no CPU path"):
        emb(t)


def test_embedding_refuses_shapes_and_types():
    """The checks behind the device's, on stand-ins that claim a GPU."""
    from nmce import embedding

    class Fake:
        def __init__(self, shape, dtype, device="cuda:0"):
            self.shape, self.dtype, self.device = torch.Size(shape), dtype, torch.device(device)
            self.is_cuda = self.device.type == "cuda"

        def dim(self):
            return len(self.shape)

    f32, i64 = torch.float32, torch.int64
    w, t = Fake((10, 8), f32), Fake((3,), i64)
    check = embedding._check_embedding
    check(t, w, 0, 10, f32)
    with pytest.raises(RuntimeError, match="tokens on"):
        check(Fake((3,), i64, "cpu"), w, 0, 10, f32)
    with pytest.raises(RuntimeError, match="tokens on"):
        check(Fake((3,), i64, "cuda:1"), w, 0, 10, f32)
    with pytest.raises(TypeError, match="int64"):
        check(Fake((3,), torch.int32), w, 0, 10, f32)
    with pytest.raises(TypeError, match="unsupported"):
        check(t, Fake((10, 8), torch.float16), 0, 10, f32)
    with pytest.raises(TypeError, match="unsupported"):
        check(t, w, 0, 10, torch.float16)
    with pytest.raises(ValueError, match="vocabulary rows"):
        check(t, w, 0, 11, f32)
    with pytest.raises(ValueError, match="vocabulary rows"):
        check(t, Fake((0, 8), f32), 0, 0, f32)
    for shape in ((10,), (10, 0), (2, 5, 8)):
        with pytest.raises(ValueError, match="must be"):
            check(t, Fake(shape, f32), 0, 10, f32)
