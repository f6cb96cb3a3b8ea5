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


def test_embedding_refusals(lib):
    import nmce
    from nmce import _lib as L
    ctx = nmce.ParallelContext.single()
    w, t = torch.randn(10, 8), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="no CPU path"):
        nmce.vocab_parallel_embedding(t, w, 0, 10, ctx)
    with pytest.raises(RuntimeError, match="no CPU path"):
        L.autograd_ext().embedding(w, t, 0, 1.0, True)
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


def test_int8_argument_errors_before_launch(lib):
    p = 4096
    quant = lib.nmce_quantize_rows
    assert quant(p, 2, 4, 8, 8, p, 16, p, None) == -1
    assert quant(p, 0, -1, 8, 8, p, 16, p, None) == -2
    assert quant(p, 0, 4, 0, 8, p, 16, p, None) == -2
    assert quant(p, 0, 4, 8, 7, p, 16, p, None) == -2
    assert quant(p, 0, 4, 8, 8, p, 7, p, None) == -2
    assert quant(p + 2, 0, 4, 8, 8, p, 16, p, None) == -3
    assert quant(p, 0, 4, 8, 8, p, 16, p + 2, None) == -3
    assert quant(p, 0, 4, 8, 8, None, 16, p, None) == -4
    assert quant(None, 0, 0, 8, 8, None, 16, None, None) == 0
    size, lin = lib.nmce_int8_linear_workspace_bytes, lib.nmce_int8_linear
    assert size(-1, 8) == size(4, 0) == size(4, 131073) == -1 and size(0, 8) >= 0
    ws = size(4, 32)
    assert lin(p, 9, 4, 32, 32, p, 10, 32, p, p, 0, 10, p, ws, None) == -1
    assert lin(p, 0, 4, 32, 32, p, 10, 32, p, p, 9, 10, p, ws, None) == -1
    assert lin(p, 0, 4, 32, 31, p, 10, 32, p, p, 0, 10, p, ws, None) == -2
    assert lin(p, 0, 4, 32, 32, p, 0, 32, p, p, 0, 10, p, ws, None) == -2
    assert lin(p, 0, 4, 32, 32, p, 10, 16, p, p, 0, 10, p, ws, None) == -2
    assert lin(p, 0, 4, 32, 32, p, 10, 1 << 23, p, p, 0, 10, p, ws, None) == -2
    assert lin(p, 0, 4, 32, 32, p, 10, 32, p, p, 0, 9, p, ws, None) == -2
    assert lin(p, 0, 4, 131073, 131073, p, 10, 131088, p, p, 0, 10, p, 1 << 40, None) == -2
    assert lin(p, 0, 4, 32, 32, p + 8, 10, 32, p, p, 0, 10, p, ws, None) == -3
    assert lin(p, 0, 4, 32, 32, p, 10, 40, p, p, 0, 10, p, ws, None) == -3
    assert lin(p, 0, 4, 32, 32, p, 10, 32, p, p + 2, 0, 10, p, ws, None) == -3
    assert lin(p, 0, 4, 32, 32, None, 10, 32, p, p, 0, 10, p, ws, None) == -4
    assert lin(p, 0, 4, 32, 32, p, 10, 32, p, p, 0, 10, p, ws - 1, None) == -6
    assert lin(p, 0, 4, 32, 32, p, 10, 32, p, p, 0, 10, None, ws, None) == -6
    assert lin(None, 0, 0, 32, 32, None, 10, 32, None, None, 0, 10, None, 0, None) == 0


def test_int8_refusals_without_a_gpu():
    import nmce
    x = torch.randn(4, 32)
    with pytest.raises(RuntimeError, match="no CPU path"):
        nmce.quantize_rows(x)
    with pytest.raises(RuntimeError, match="no CPU path"):
        nmce.int8_linear(x, torch.zeros(3, 32, dtype=torch.int8), torch.ones(3))
    cfg = types.SimpleNamespace(vocab_size=1000, n_embd=30, sequence_parallel=False)
    two = nmce.ParallelContext(rank=1, world_size=2, tp_size=2, tp_rank=1, pp_size=1, pp_rank=0,
                               dp_size=1, dp_rank=0)
    head = nmce.Int8ParallelLMHead(cfg, two)
    assert head.weight_q.shape == (500, 32) and head.vocab_range() == (500, 1000)
    assert sorted(head.state_dict()) == ["weight_q", "weight_scale"]
    assert not list(head.parameters())
    with pytest.raises(RuntimeError, match="no CPU path"):
        head(torch.randn(2, 30))


def test_int8_weight_rows():
    """Which weights the product reads as they lie (no device needed)."""
    from nmce.int8 import _weight_rows
    base = torch.randint(-128, 128, (10, 48), dtype=torch.int8)
    pad = (-base.data_ptr()) % 16
    assert pad == 0
    for w, same in ((base, True), (base[:, :33], True), (base[:, 16:40], True),
                    (base[:, 8:40], False), (base[:, 32:47], True), (base.t(), False),
                    (base[:1, :33], True), (base[:1].expand(10, 48), False),
                    (base[:, :40].contiguous(), False), (base[3:7:2], True)):
        got, ld = _weight_rows(w)
        assert (got is w) == same, (w.shape, w.stride())
        assert ld % 16 == 0 and ld >= w.shape[1]
        assert torch.equal(got[:, :w.shape[1]], w)
    far = torch.zeros((1 << 23) + 48, dtype=torch.int8).as_strided((2, 48), (1 << 23, 1))
    assert _weight_rows(far)[0] is not far and _weight_rows(far)[1] == 48
    # the last row ends with the storage, inside 16 bytes
    tight = torch.zeros(9 * 48 + 33, dtype=torch.int8).as_strided((10, 33), (48, 1))
    assert _weight_rows(tight)[0] is not tight


def test_verify_argument_errors_before_launch(lib):
    import ctypes
    from nmce import _lib as L
    p = 4096

    def batch(**kwargs):
        fields = dict(target=p, draft=p, draft_tokens=p, accept_u=p, sample_u=p, temperature=None,
                      target_batch_stride=40, target_row_stride=10, draft_batch_stride=30,
                      draft_row_stride=10, batch=2, drafts=3, vocab_local=10, vocab_start=0,
                      vocab_total=10, temperature_all=1.0, dtype=0)
        fields.update(kwargs)
        return L.VerifyBatch(**fields)

    def stats(out=p, **kwargs):
        b = batch(**kwargs)
        return lib.nmce_verify_stats(ctypes.addressof(b), out, None)

    assert lib.nmce_verify_slabs(0) == -1 and lib.nmce_verify_slabs(1) == 1
    assert lib.nmce_verify_slabs(8192) == 1 and lib.nmce_verify_slabs(8193) == 2
    assert lib.nmce_verify_workspace_bytes(-1) == -1 and lib.nmce_verify_workspace_bytes(0) == 0
    assert lib.nmce_verify_stats(None, p, None) == -4
    assert stats(dtype=2) == -1
    for bad in (dict(batch=-1), dict(drafts=-1), dict(vocab_local=0), dict(vocab_start=-1),
                dict(vocab_start=1), dict(vocab_total=9), dict(batch=1 << 22, drafts=1),
                dict(batch=1 << 20, vocab_local=80000, vocab_total=80000),
                dict(vocab_local=1 << 31, vocab_total=1 << 31)):
        assert stats(**bad) == -2, bad
    assert stats(target=None) == stats(draft_tokens=None) == stats(accept_u=None) == -4
    assert stats(sample_u=None) == stats(out=None) == -4
    assert stats(target=p + 2) == stats(draft=p + 1) == stats(dtype=1, target=p + 1) == -3
    assert stats(batch=0, target=None) == 0
    b = batch()
    at, ws = ctypes.addressof(b), lib.nmce_verify_workspace_bytes(2)
    assert lib.nmce_verify_masses(at, p, 0, p, p, p, p, p, ws, None) == -5
    assert lib.nmce_verify_masses(at, None, 1, p, p, p, p, p, ws, None) == -4
    assert lib.nmce_verify_masses(at, p, 1, p, p, p, None, p, ws, None) == -4
    assert lib.nmce_verify_masses(at, p, 1, p, p, p, p, p, ws - 1, None) == -6
    assert lib.nmce_verify_pick(at, p, 2, 2, p, ws, p, p, p, None) == -5
    assert lib.nmce_verify_pick(at, p, 2, 1, p, ws, p, p, None, None) == -4  # ranks need picked
    assert lib.nmce_verify_pick(at, p, 1, 0, p, 0, p, p, None, None) == -6
    assert lib.nmce_verify_finish(None, p, ws, 2, 3, p, p, None) == -4
    assert lib.nmce_verify_finish(p, p, ws, -1, 3, p, p, None) == -2
    assert lib.nmce_verify_finish(p, p, 0, 2, 3, p, p, None) == -6
    assert lib.nmce_verify_finish(None, None, 0, 0, 3, None, None, None) == 0


def test_verify_has_no_cpu_path():
    import nmce
    with pytest.raises(RuntimeError, match="no CPU path"):
        nmce.vocab_parallel_verify_drafts(
            torch.zeros(1, 2, 5), torch.zeros(1, 1, dtype=torch.int64), None, torch.zeros(1, 1),
            torch.zeros(1), 0, 5, nmce.ParallelContext.single())


def test_int8_products_keep_their_wait_states(tmp_path):
    """The 8-bit products run on the GEMM core, whose MFMAs are inline asm: in the
    generated code no VALU instruction writes one's source within two wait states
    before it, and none touches its result within 16 behind it (as for the bf16
    products). The few tokens' kernel uses the builtin, which the compiler
    schedules itself."""
    import re
    import subprocess

    from _util import mfma_hazards
    from nmce import _build
    asm = tmp_path / "int8.s"
    subprocess.run([_build.hipcc(), *_build.HIPCC_FLAGS, "-S", "--cuda-device-only",
                    str(_build.CSRC_DIR / "nmce_int8.hip"), "-o", str(asm)], check=True,
                   capture_output=True)
    bodies = re.findall(r"^_Z\w*int8_linear_kernel\w*:(.*?)\.end_amdhsa_kernel", asm.read_text(),
                        re.S | re.M)
    assert len(bodies) == 3
    for body in bodies:
        mfmas, offenders = mfma_hazards(body)
        assert mfmas >= 384 and not offenders, offenders[:5]


def test_int8_head_keeps_its_types_under_casts():
    """A cast of the served model reaches its buffers too: the 8-bit rows and their
    fp32 scales stay as they are, to the bit, and only move."""
    import nmce
    cfg = types.SimpleNamespace(vocab_size=40, n_embd=30)
    head = nmce.Int8ParallelLMHead(cfg, nmce.ParallelContext.single())
    g = torch.Generator().manual_seed(0)
    head.weight_q.copy_(torch.randint(-127, 128, head.weight_q.shape, generator=g))
    head.weight_scale.copy_(torch.rand(40, generator=g))
    q, scale = head.weight_q.clone(), head.weight_scale.clone()
    model = torch.nn.Sequential(torch.nn.Linear(4, 4), head)
    for cast in (lambda m: m.to(torch.bfloat16), lambda m: m.half(), lambda m: m.bfloat16(),
                 lambda m: m.double(), lambda m: m.type(torch.bfloat16), lambda m: m.float(),
                 lambda m: m.to("cpu", torch.float16)):
        cast(model)
        for name, want in (("weight_q", q), ("weight_scale", scale)):
            held = getattr(head, name)
            assert held.dtype == want.dtype and torch.equal(held, want), name
            assert model.state_dict()["1." + name] is not None
    assert model[0].weight.dtype == torch.float16
    # a move and a cast in one, and memory of its own
    head.to("meta", torch.bfloat16)
    assert head.weight_scale.is_meta and head.weight_scale.dtype == torch.float32
    head.to_empty(device="cpu")
    assert head.weight_q.dtype == torch.int8 and head.weight_scale.shape == (40,)


def test_tensors_that_want_a_derivative_are_refused():
    """What the kernels without one ask of each of their tensors (no device needed)."""
    from torch.autograd import forward_ad
    from nmce import _lib as L
    t = torch.randn(3)
    L.refuse_gradient(t, "x", "they have")
    leaf = torch.randn(3, requires_grad=True)
    with pytest.raises(RuntimeError, match="nmce: x requires grad, but they have no backward"):
        L.refuse_gradient(leaf, "x", "they have")
    with torch.no_grad():
        L.refuse_gradient(leaf, "x", "they have")
    with forward_ad.dual_level():
        L.refuse_gradient(t, "x", "they have")
        dual = forward_ad.make_dual(t, torch.ones(3))
        for mode in (torch.enable_grad, torch.no_grad):
            with mode(), pytest.raises(RuntimeError, match="forward-mode tangent"):
                L.refuse_gradient(dual, "x", "they have")
        L.refuse_gradient(forward_ad.unpack_dual(dual).primal, "x", "they have")
        with torch.inference_mode():  # where torch's own operators drop tangents
            assert forward_ad.unpack_dual(dual * 2).tangent is None
            L.refuse_gradient(dual, "x", "they have")


def test_verify_refuses_another_ranks_shard():
    """The shards' running sums are joined in the order of the ranks: a shard that is
    not the rank's own would give other tokens (stand-ins that claim a GPU)."""
    import dataclasses
    import nmce
    from nmce import verify

    class Fake:
        is_cuda, device, requires_grad, dtype = True, torch.device("cuda:0"), False, torch.float32

        def __init__(self, *shape, dtype=torch.float32):
            self.shape, self.dtype = torch.Size(shape), dtype

        def dim(self):
            return len(self.shape)

    one = nmce.ParallelContext.single()
    args = (Fake(2, 4, 50), Fake(2, 3, dtype=torch.int64), None, Fake(2, 3), Fake(2))
    for tp, rank, start, ok in ((1, 0, 0, True), (1, 0, 50, False), (2, 0, 0, True),
                                (2, 1, 50, True), (2, 1, 0, False), (2, 0, 50, False),
                                (4, 2, 100, True), (4, 2, 101, False), (4, 2, 99, False),
                                (4, 1, 100, False), (2, 1, 100, False)):
        ctx = dataclasses.replace(one, tp_size=tp, tp_rank=rank)
        if ok:
            verify._check_verify(*args, start, start + 50, ctx, 1.0)
        else:
            with pytest.raises(ValueError, match="is not rank"):
                verify._check_verify(*args, start, start + 50, ctx, 1.0)


def test_verify_starts_that_would_overflow(lib):
    """A start near 2^63 is refused as outside the vocabulary: its sum with the
    shard's size is not formed."""
    import ctypes
    from nmce import _lib as L
    p = 4096
    for start in ((1 << 63) - 1, (1 << 63) - 9, 1 << 62, 1 << 31, 11):
        b = L.VerifyBatch(p, None, p, p, p, None, 40, 10, 0, 0, 2, 3, 10, start, 20, 1.0, 0)
        assert lib.nmce_verify_stats(ctypes.addressof(b), p, None) == -2, start


def test_a_cast_reaches_other_buffers_of_the_head():
    import nmce
    head = nmce.Int8ParallelLMHead(types.SimpleNamespace(vocab_size=8, n_embd=16),
                                   nmce.ParallelContext.single())
    head.register_buffer("mine", torch.ones(3))
    head.to(torch.bfloat16)
    assert head.mine.dtype == torch.bfloat16 and head.weight_scale.dtype == torch.float32
