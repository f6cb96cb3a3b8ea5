"""What the adjusted logits, the top logits and their distillation refuse: no GPU needed."""

from __future__ import annotations

import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from nmce import _lib as L
    return L.load()


class Fake:
    """A stand-in that claims a GPU, for the checks behind the device's."""

    def __init__(self, shape, dtype, device="cuda:0"):
        self.shape, self.dtype, self.device = torch.Size(shape), dtype, torch.device(device)
        self.is_cuda = self.device.type == "cuda"
        self.requires_grad = False

    def dim(self):
        return len(self.shape)


F32, BF, I64 = torch.float32, torch.bfloat16, torch.int64


def _adjust_batch(**kw):
    from nmce import _lib as L
    p = 4096  # a fake, aligned device address; never dereferenced
    a = L.AdjustBatch()
    fields = dict(logits=p, out=2 * p, prompt=p, output=p, drafts=p, bias_ids=p, bias=p, allowed=p,
                  logits_batch_stride=30, logits_row_stride=10, out_batch_stride=30,
                  out_row_stride=10, prompt_stride=4, output_stride=4, drafts_stride=2,
                  bias_ids_stride=4, bias_stride=4, allowed_batch_stride=3, allowed_row_stride=1,
                  n_prompt=4, n_output=4, n_bias=4, batch=2, rows=3, vocab_local=10, vocab_start=0,
                  vocab_total=10, repetition_all=1.0, dtype=0)
    fields.update(kw)
    for name, value in fields.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("change,status", [
    (dict(dtype=2), -1), (dict(batch=-1), -2), (dict(rows=0), -2), (dict(vocab_local=0), -2),
    (dict(vocab_start=-1), -2), (dict(vocab_start=1), -2), (dict(vocab_total=9), -2),
    (dict(vocab_total=1 << 31), -2), (dict(n_prompt=-1), -2), (dict(n_output=-1), -2),
    (dict(n_output=(1 << 29) + 1), -2), (dict(n_bias=-1), -2), (dict(n_bias=8193), -2),
    (dict(batch=1 << 22), -2), (dict(rows=(1 << 22) + 1), -2), (dict(logits=None), -4),
    (dict(out=None), -4), (dict(prompt=None), -4), (dict(output=None), -4), (dict(drafts=None), -4),
    (dict(bias_ids=None), -4), (dict(bias=None), -4), (dict(logits=4098), -3),
    (dict(out=4097, dtype=1), -3), (dict(allowed=4098), -3),
    (dict(out=4096, out_row_stride=11), -2), (dict(out=4096, out_batch_stride=31), -2),
    (dict(batch=0, logits=None), 0)])
def test_adjust_argument_errors_before_launch(lib, change, status):
    a = _adjust_batch(**change)
    assert lib.nmce_adjust_logits(ctypes.addressof(a), None) == status
    assert lib.nmce_adjust_logits(None, None) == -4


def test_adjust_refuses_shapes_and_types():
    import nmce
    from nmce import adjust
    ctx = nmce.ParallelContext.single()
    good = dict(logits=Fake((2, 3, 40), F32), vocab_start=0, vocab_end=40, ctx=ctx,
                prompt=Fake((2, 9), I64), output=Fake((2, 0), I64), drafts=Fake((2, 2), I64),
                penalties=(("repetition_penalty", 1.5), ("frequency_penalty", Fake((2,), F32)),
                           ("presence_penalty", 0.0)),
                bias_ids=Fake((2, 4), I64), bias_values=Fake((2, 4), F32),
                allowed=Fake((2, 3, 2), torch.int32))

    def check(**kw):
        adjust._check_adjust(**{**good, **kw})

    check()
    check(prompt=None, output=None, bias_ids=None, bias_values=None, allowed=None)
    with pytest.raises(RuntimeError, match="no CPU path"):
        check(logits=Fake((2, 3, 40), F32, "cpu"))
    with pytest.raises(TypeError, match="unsupported"):
        check(logits=Fake((2, 3, 40), torch.float16))
    for shape in ((2, 40), (2, 0, 40), (2, 3, 0), (1, 2, 3, 40)):
        with pytest.raises(ValueError, match="must be"):
            check(logits=Fake(shape, F32))
    for start, end in ((0, 41), (1, 40), (-1, 39), (1, 41)):
        with pytest.raises(ValueError, match="shard"):
            check(vocab_start=start, vocab_end=end)
    with pytest.raises(ValueError, match="draft_tokens"):
        check(drafts=None)
    with pytest.raises(ValueError, match="come together"):
        check(bias_ids=None)
    with pytest.raises(ValueError, match="come together"):
        check(bias_values=None)
    for name, shape, dtype in (("prompt", (3, 9), I64), ("prompt", (9,), I64),
                               ("output", (2,), I64), ("drafts", (2, 3), I64),
                               ("bias_values", (2, 5), F32), ("allowed", (2, 3, 1), torch.int32),
                               ("allowed", (2, 1, 2), torch.int32)):
        with pytest.raises(ValueError, match="must be"):
            check(**{name: Fake(shape, dtype)})
    for name, shape, dtype in (("prompt", (2, 9), torch.int32), ("output", (2, 1), F32),
                               ("drafts", (2, 2), torch.int32), ("bias_ids", (2, 4), torch.int32),
                               ("bias_values", (2, 4), BF), ("allowed", (2, 3, 2), I64)):
        with pytest.raises(TypeError, match="must be"):
            check(**{name: Fake(shape, dtype)})
        with pytest.raises(RuntimeError, match="on cuda:1"):
            check(**{name: Fake(shape, dtype, "cuda:1")})
    with pytest.raises(ValueError, match="at most 8192"):
        check(bias_ids=Fake((2, 8193), I64), bias_values=Fake((2, 8193), F32))
    for name, value in (("repetition_penalty", 0.0), ("repetition_penalty", -1.0),
                        ("repetition_penalty", float("nan")),
                        ("frequency_penalty", float("inf")), ("presence_penalty", float("nan"))):
        with pytest.raises(ValueError, match=name):
            check(penalties=((name, value),))
    with pytest.raises(ValueError, match="must be"):
        check(penalties=(("frequency_penalty", Fake((3,), F32)),))
    with pytest.raises(TypeError, match="must be"):
        check(penalties=(("frequency_penalty", Fake((2,), torch.float64)),))


def test_adjust_has_no_cpu_path():
    import nmce
    with pytest.raises(RuntimeError, match="no CPU path"):
        nmce.vocab_parallel_adjust_logits(torch.zeros(1, 1, 8), 0, 8, nmce.ParallelContext.single())


def test_top_argument_errors_before_launch(lib):
    p = 4096
    size = lib.nmce_top_workspace_bytes
    ws = size(4, 100, 10)
    assert ws > 0 and size(0, 100, 10) >= 0
    assert size(-1, 100, 10) == size((1 << 22) + 1, 100, 10) == size(4, 0, 10) == -1
    assert size(4, 1 << 31, 10) == size(4, 100, 0) == size(4, 100, 513) == -1

    def top(logits=p, dtype=0, n=4, v=100, ld=100, start=0, k=10, t=1.0, lists=None, values=p,
            ids=p, norm=p, space=p, size_=ws):
        return lib.nmce_top_logits(logits, dtype, n, v, ld, start, k, t, lists, values, ids, norm,
                                   space, size_, None)

    assert top(dtype=2) == -1
    for bad in (dict(n=-1), dict(n=(1 << 22) + 1), dict(v=0), dict(v=1 << 31), dict(ld=99),
                dict(start=-1), dict(start=(1 << 31) - 100), dict(k=0), dict(k=513), dict(k=101),
                dict(t=0.0), dict(t=-1.0), dict(t=float("nan")), dict(t=1e31), dict(t=1e-31)):
        assert top(**bad) == -2, bad
    assert top(logits=p + 2) == top(logits=p + 1, dtype=1) == -3
    for name in ("logits", "values", "ids", "norm"):
        assert top(**{name: None}) == -4
    assert top(space=None) == top(space=p + 8) == top(size_=ws - 1) == -6
    assert top(n=0, logits=None) == 0
    assert top(lists=p, k=101, values=None, ids=None, norm=None, size_=0) == -6
    merge = lib.nmce_top_merge
    assert merge(p, 2, 3, 4, 10, 1.0, p, p, p, None) == -1
    assert merge(p, 2, 0, -1, 10, 1.0, p, p, p, None) == -2
    assert merge(p, 2, 0, 4, 513, 1.0, p, p, p, None) == -2
    assert merge(p, 0, 0, 4, 10, 1.0, p, p, p, None) == -5
    assert merge(None, 2, 0, 4, 10, 1.0, p, p, p, None) == -4
    assert merge(None, 2, 0, 0, 10, 1.0, None, p, p, None) == 0


def test_top_refuses_shapes_and_types():
    import nmce
    from nmce import top
    ctx = nmce.ParallelContext.single()

    def check(logits=Fake((2, 40), F32), k=5, start=0, end=40, ctx=ctx, t=1.0):
        top._check_top(logits, k, start, end, ctx, t)

    check()
    check(Fake((40,), BF))
    with pytest.raises(RuntimeError, match="no CPU path"):
        check(Fake((2, 40), F32, "cpu"))
    with pytest.raises(TypeError, match="unsupported"):
        check(Fake((2, 40), torch.float16))
    for shape in ((), (2, 0)):
        with pytest.raises(ValueError, match="must be"):
            check(Fake(shape, F32), end=0)
    for start, end in ((0, 41), (1, 41), (-1, 39)):
        with pytest.raises(ValueError, match="shard"):
            check(start=start, end=end)
    for k in (0, -3, 41):
        with pytest.raises(ValueError, match="k must be"):
            check(k=k)
    with pytest.raises(ValueError, match="k must be"):
        check(Fake((2, 1000), F32), k=513, end=1000)
    for t in (0.0, -1.0, 1e-31, 1e31, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="temperature"):
            check(t=t)
    with pytest.raises(RuntimeError, match="no CPU path"):
        nmce.vocab_parallel_top_logits(torch.zeros(2, 8), 2, 0, 8, ctx)


def _distill_batch(**kw):
    from nmce import _lib as L
    p = 4096
    a = L.DistillBatch()
    fields = dict(logits=p, teacher_logits=p, teacher_ids=p, teacher_log_normalizer=p, ld=100,
                  teacher_ld=8, ids_ld=8, n_rows=4, vocab_local=100, vocab_start=0,
                  vocab_total=100, temperature=1.0, k=8, dtype=0, teacher_dtype=0)
    fields.update(kw)
    for name, value in fields.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("change,status", [
    (dict(dtype=2), -1), (dict(teacher_dtype=-1), -1), (dict(n_rows=-1), -2),
    (dict(n_rows=(1 << 22) + 1), -2), (dict(vocab_local=0), -2), (dict(vocab_start=-1), -2),
    (dict(vocab_start=1), -2), (dict(vocab_total=99), -2), (dict(vocab_total=(1 << 31) - 1), -2),
    (dict(ld=99), -2), (dict(k=0), -2), (dict(k=1025), -2), (dict(teacher_ld=-1), -2),
    (dict(ids_ld=-1), -2), (dict(temperature=0.0), -2), (dict(temperature=1e-7), -2),
    (dict(temperature=float("nan")), -2), (dict(temperature=1e7), -2), (dict(logits=None), -4),
    (dict(teacher_logits=None), -4), (dict(teacher_ids=None), -4), (dict(logits=4098), -3),
    (dict(logits=4097, dtype=1), -3), (dict(teacher_logits=4098), -3),
    (dict(n_rows=0, logits=None), 0)])
def test_distill_argument_errors_before_launch(lib, change, status):
    p, size = 4096, lib.nmce_distill_state_bytes(4, 8)
    a = _distill_batch(**change)
    assert lib.nmce_distill_stats(ctypes.addressof(a), p, size, p, None) == status


def test_distill_steps_refuse_before_launch(lib):
    p, state = 4096, lib.nmce_distill_state_bytes
    size = state(4, 8)
    assert size > 0 and state(0, 8) >= 0
    assert state(-1, 8) == state((1 << 22) + 1, 8) == state(4, 0) == state(4, 1025) == -1
    good = _distill_batch()
    stats = lib.nmce_distill_stats
    assert stats(None, p, size, p, None) == -4
    assert stats(ctypes.addressof(good), p, size, None, None) == -4
    for space, bytes_ in ((None, size), (p + 8, size), (p, size - 1)):
        assert stats(ctypes.addressof(good), space, bytes_, p, None) == -6
    def one(batch=good, g=2 * p, ldg=100, space=p, bytes_=size, loss=p, mean=p, expect=p, assumed=p,
            div=4.0):
        return lib.nmce_distill_fwd_bwd(ctypes.addressof(batch), g, ldg, space, bytes_, loss, mean,
                                        expect, assumed, div, None)

    assert one(_distill_batch(dtype=5)) == -1
    for bad in (dict(batch=_distill_batch(vocab_total=200)), dict(ldg=99), dict(div=0.0),
                dict(batch=_distill_batch(vocab_start=100, vocab_total=200)),
                dict(batch=_distill_batch(vocab_local=65537, vocab_total=65537, ld=65537),
                     ldg=65537),
                dict(batch=_distill_batch(dtype=1, vocab_local=131073, vocab_total=131073,
                                          ld=131073), ldg=131073),
                dict(g=p, ldg=104), dict(batch=_distill_batch(n_rows=(1 << 22) + 1))):
        assert one(**bad) == -2, bad
    for name in ("g", "loss", "expect", "assumed"):
        assert one(**{name: None}) == -4
    assert one(g=2 * p + 2) == one(g=2 * p + 4) == one(ldg=101) == -3
    assert one(space=None) == one(space=p + 8) == one(bytes_=size - 1) == -6
    assert one(_distill_batch(n_rows=0), g=None) == 0
    combine = lib.nmce_distill_combine
    assert combine(p, size, -1, 8, 1.0, p, 1, p, p, None) == -2
    assert combine(p, size, 4, 0, 1.0, p, 1, p, p, None) == -2
    assert combine(p, size, 4, 8, 0.0, p, 1, p, p, None) == -2
    assert combine(p, size, 4, 8, 1.0, p, 0, p, p, None) == -5
    assert combine(p, size, 4, 8, 1.0, None, 1, p, p, None) == -4
    assert combine(p, size, 4, 8, 1.0, p, 1, None, p, None) == -4
    assert combine(p, size - 1, 4, 8, 1.0, p, 1, p, None, None) == -6
    assert combine(None, 0, 0, 8, 1.0, None, 1, None, None, None) == 0

    def bwd(x=p, g=2 * p, dtype=0, n=4, v=100, ld=100, ldg=100, k=8, t=1.0, space=p, bytes_=size,
            go=p, stride=0, div=4.0):
        return lib.nmce_distill_bwd(x, g, dtype, n, v, ld, ldg, k, t, space, bytes_, go, stride,
                                    div, None, None, None)

    assert bwd(dtype=3) == -1
    for bad in (dict(n=-1), dict(v=0), dict(ld=99), dict(ldg=99), dict(k=0), dict(k=1025),
                dict(stride=-1), dict(div=0.0), dict(div=float("nan")), dict(t=0.0),
                dict(g=p, ldg=101)):
        assert bwd(**bad) == -2, bad
    assert bwd(x=None) == bwd(g=None) == bwd(go=None) == -4
    assert bwd(x=p + 2) == bwd(g=p + 1, dtype=1) == -3
    assert bwd(space=None) == bwd(space=p + 4) == bwd(bytes_=size - 1) == -6
    assert bwd(n=0, x=None) == 0


def test_distillation_refuses_shapes_and_types():
    import nmce
    from nmce import distill
    ctx = nmce.ParallelContext.single()
    good = dict(logits=Fake((2, 3, 40), F32), teacher_logits=Fake((2, 3, 5), BF),
                teacher_ids=Fake((2, 3, 5), I64), normalizer=Fake((2, 3), F32), vocab_start=0,
                vocab_end=40, ctx=ctx, temperature=1.0, reduction="mean")

    def check(**kw):
        distill._check_distillation(**{**good, **kw})

    check()
    check(normalizer=None, reduction="none", temperature=2)
    with pytest.raises(RuntimeError, match="no CPU path"):
        check(logits=Fake((2, 3, 40), F32, "cpu"))
    with pytest.raises(TypeError, match="unsupported"):
        check(logits=Fake((2, 3, 40), torch.float16))
    with pytest.raises(ValueError, match="must be"):
        check(logits=Fake((2, 3, 0), F32), vocab_end=0)
    for start, end in ((0, 41), (1, 41), (-1, 39)):
        with pytest.raises(ValueError, match="shard"):
            check(vocab_start=start, vocab_end=end)
    for shape in ((2, 3), (3, 2, 5), (6, 5), (5,)):
        with pytest.raises(ValueError, match="not a list"):
            check(teacher_logits=Fake(shape, F32))
    for k in (0, 1025):
        with pytest.raises(ValueError, match="1 to 1024"):
            check(teacher_logits=Fake((2, 3, k), F32), teacher_ids=Fake((2, 3, k), I64))
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        check(teacher_logits=Fake((2, 3, 5), torch.float16))
    with pytest.raises(TypeError, match="int64"):
        check(teacher_ids=Fake((2, 3, 5), torch.int32))
    with pytest.raises(ValueError, match="must be"):
        check(teacher_ids=Fake((2, 3, 4), I64))
    with pytest.raises(ValueError, match="must be"):
        check(normalizer=Fake((2, 3, 1), F32))
    with pytest.raises(TypeError, match="must be"):
        check(normalizer=Fake((2, 3), BF))
    for name, shape, dtype in (("teacher_logits", (2, 3, 5), F32), ("teacher_ids", (2, 3, 5), I64),
                               ("normalizer", (2, 3), F32)):
        with pytest.raises(RuntimeError, match="on cuda:1"):
            check(**{name: Fake(shape, dtype, "cuda:1")})
    for t in (0.0, -1.0, 1e-7, 1e7, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="temperature"):
            check(temperature=t)
    with pytest.raises(ValueError, match="reduction"):
        check(reduction="sum")
    teacher = Fake((2, 3, 5), F32)
    teacher.requires_grad = True
    with pytest.raises(RuntimeError, match="requires grad"):
        check(teacher_logits=teacher)
    with torch.no_grad():
        check(teacher_logits=teacher)
    x, t, ids = torch.zeros(2, 8), torch.zeros(2, 3), torch.zeros(2, 3, dtype=I64)
    with pytest.raises(RuntimeError, match="no CPU path"):
        nmce.vocab_parallel_distillation_loss(x, t, ids, 0, 8, ctx)
    from nmce import _lib as L
    with pytest.raises(RuntimeError, match="no CPU path"):
        L.autograd_ext().distill(x, t, ids, None, 1.0, True, False)
    with pytest.raises(RuntimeError, match="no CPU path"):
        L.autograd_ext().distill_mean(x, t, ids, None, torch.ones(1), 1.0, False)
