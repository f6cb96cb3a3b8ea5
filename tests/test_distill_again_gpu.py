"""Lists that name an id again: its probabilities are one class's, in the loss too.

The reference merges each list first, in 64 bits: an id's logits become one, T log of the sum
of exp(t / T). What the kernels' 64-bit sums and logarithms add to the loss (2^-45 of it at
most) is nothing beside the slacks of the sums over the vocabulary."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

import test_distill_gpu as distill

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32
INF = float("inf")


def _merged(t, ids, temperature, v):
    """Lists of different ids, the first place of each, in 64 bits."""
    t2, ids2 = torch.full(t.shape, -INF, dtype=torch.float64), torch.full_like(ids, -1)
    for i in range(ids.shape[0]):
        for j, at in enumerate(dict.fromkeys(a for a in ids[i].tolist() if 0 <= a < v)):
            ids2[i, j] = at
            t2[i, j] = temperature * torch.logsumexp(t[i][ids[i] == at].double() / temperature, 0)
    return t2, ids2


_plain = distill._reference


def _reference(x, t, ids, norm, temperature, total=None):
    return _plain(x, *_merged(t, ids, temperature, x.shape[1]), norm, temperature)


@pytest.fixture
def check(monkeypatch):
    monkeypatch.setattr(distill, "_reference", _reference)
    return distill._check


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF])
def test_an_id_that_comes_again(check, dtype, tail):
    g = torch.Generator().manual_seed(4)
    x = (torch.randn(5, 300, generator=g) * 2).to(dtype)
    ids = torch.tensor([[7, 7, 7, 9], [1, 2, 1, 2], [299, 0, 299, -1], [5, 5, 5, 5],
                        [8, 9, 10, 8]])
    t = torch.randn(5, 4, generator=g)
    t[4] = torch.tensor([1.0, 2.0, -INF, -INF])
    check(x, t, ids, torch.logsumexp(t, 1) + 0.5 if tail else None)
    many = torch.randint(0, 40, (5, 700), generator=g)
    t = torch.randn(5, 700, generator=g)
    check(x, t, many, torch.logsumexp(t, 1) + 0.1 if tail else None)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("k", [1024, 513, 512, 65, 64, 63, 2])
def test_long_lists_of_few_ids(check, k, tail):
    """One id, two in turn, half of them twice, and one twice at the list's ends."""
    g = torch.Generator().manual_seed(k)
    x = torch.randn(4, 2000, generator=g)
    t = torch.randn(4, k, generator=g)
    j = torch.arange(k)
    ids = torch.stack([torch.full((k,), 1999), j % 2 * 7, j % ((k + 1) // 2), j])
    ids[3, k - 1] = 0
    check(x, t, ids, torch.logsumexp(t.double(), 1).float() + 0.25 if tail else None)


@pytest.mark.parametrize("dtype,teacher", [(F32, BF), (BF, F32)])
@pytest.mark.parametrize("temperature", [0.25, 7.5])
def test_temperatures_and_teacher_types(check, dtype, teacher, temperature):
    g = torch.Generator().manual_seed(3)
    x, t, ids, norm = distill._inputs(6, 5003, 40, dtype, g, teacher, temperature)
    ids[:, 30:] = ids[:, :10]
    check(x, t, ids, norm + 0.5, temperature)
    check(x, t, ids, None, temperature)


@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_a_certain_student_of_a_teacher_in_halves(reduction):
    """The list [5, 5] of equal logits and a student that is sure of 5: no divergence. (The
    exponentials of the list's side are off by 2^-45, which 1e-12 is well above.)"""
    x = torch.full((1, 64), -INF)
    x[0, 5] = 1.0
    d = x.to(DEV).requires_grad_(True)
    loss = distill._loss(d, torch.ones(1, 2), torch.tensor([[5, 5]]), reduction=reduction)
    assert abs(float(loss.detach().sum())) <= 1e-12
    grad, = torch.autograd.grad(loss.sum(), d)
    assert not bool(grad.any())


def test_a_divergence_is_not_negative():
    """At the teacher's own distribution it is 0: off by the two logarithms of fp32 sums of
    8 and 9 terms, 2^-24 (3 D + 9) each with D, the mean distance from the maximum, below 4."""
    g = torch.Generator().manual_seed(8)
    z = torch.randn(20, 8, generator=g)
    again = torch.cat([z, z - 1.0, z + 0.5], 1)
    ids = torch.arange(8).repeat(20, 3)
    x = torch.full((20, 3000), -INF)
    x[:, :8] = z
    loss = distill._loss(x.to(DEV), again, ids, reduction="none").cpu()
    assert bool((loss.abs() <= 2 * 2.0 ** -24 * (3 * 4 + 9)).all())


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("ranks", [2, 5])
def test_over_shards(ranks, dtype, tail):
    """Each shard's statistics, and the losses and gradients from all: alike on every rank,
    also on those that hold none of an id's places."""
    from nmce import _lib as L
    lib = L.load()
    g = torch.Generator().manual_seed(ranks)
    n, per, k = 6, 301, 90
    v = ranks * per
    x, t, ids, norm = distill._inputs(n, v, k, dtype, g)
    ids[:, 60:] = ids[:, :30]
    ids[5] = per - 1
    norm = norm + 0.5 if tail else None
    want, slack, grad, grad_slack = _reference(x, t, ids, norm, 1.0)
    stream = L.stream_handle(torch.device(DEV))
    td, idd, nd = t.to(DEV), ids.to(DEV), None if norm is None else norm.to(DEV)
    size = lib.nmce_distill_state_bytes(n, k)
    stats = torch.empty(ranks, n, 5, dtype=torch.float64, device=DEV)
    mine, states = [], []
    for r in range(ranks):
        mine.append(x[:, r * per:(r + 1) * per].contiguous().to(DEV))
        states.append(torch.empty(size, dtype=torch.uint8, device=DEV))
        batch = L.DistillBatch(mine[r].data_ptr(), td.data_ptr(), idd.data_ptr(),
                               None if nd is None else nd.data_ptr(), per, k, k, n, per, r * per,
                               v, 1.0, k, L.dtype_code(dtype), L.dtype_code(F32))
        L.check(lib.nmce_distill_stats(ctypes.addressof(batch), states[r].data_ptr(), size,
                                       stats[r].data_ptr(), stream), "stats")
    one = torch.ones(1, device=DEV)
    losses, grads = [], []
    for r in range(ranks):
        loss = torch.empty(n, device=DEV)
        L.check(lib.nmce_distill_combine(states[r].data_ptr(), size, n, k, 1.0, stats.data_ptr(),
                                         ranks, loss.data_ptr(), None, stream), "combine")
        out = torch.empty_like(mine[r])
        L.check(lib.nmce_distill_bwd(mine[r].data_ptr(), out.data_ptr(), L.dtype_code(dtype), n,
                                     per, per, per, k, 1.0, states[r].data_ptr(), size,
                                     one.data_ptr(), 0, 1.0, None, None, stream), "bwd")
        losses.append(loss)
        grads.append(out)
    assert all(torch.equal(a, losses[0]) for a in losses)
    distill._within(losses[0], want, slack, F32, "loss")
    distill._within(torch.cat(grads, 1), grad, grad_slack, dtype, "gradient")


def test_nothing_and_too_much():
    """Repeated ids of a teacher's -inf logits, of a NaN, and of a normaliser that is none."""
    t = torch.tensor([[1.0, -INF, -INF], [-INF, -INF, -INF], [0.0, math.nan, 0.0],
                      [0.0, 0.0, 1.0]])
    ids = torch.tensor([[3, 4, 4], [4, 4, 4], [2, 2, 5], [6, 6, 6]])
    x = torch.linspace(-1.0, 1.0, 32).expand(4, 32).contiguous()
    lp = torch.log_softmax(x.double(), 1)
    loss = distill._loss(x.to(DEV), t, ids, reduction="none").double().cpu()
    # (32 terms: two sums' steps as above.)
    slack = 2.0 ** -24 * 40
    assert abs(float(loss[0]) + float(lp[0, 3])) <= slack
    assert float(loss[1]) == 0.0  # no teacher
    assert math.isnan(float(loss[2]))
    assert abs(float(loss[3]) + float(lp[3, 6])) <= slack
    norm = torch.tensor([1.5, -INF, 1.0, 1e4])
    loss = distill._loss(x.to(DEV), t, ids, norm, reduction="none").double().cpu()
    p = math.exp(-0.5)
    rest = 1.0 - p
    s = 1.0 - float(lp[0, 3].exp()) - float(lp[0, 4].exp())
    want = p * (math.log(p) - float(lp[0, 3])) + rest * (math.log(rest) - math.log(s))
    assert abs(float(loss[0]) - want) <= slack
    assert float(loss[1]) == 0.0 and math.isnan(float(loss[2]))
    s = 1.0 - float(lp[3, 6].exp())
    assert abs(float(loss[3]) + math.log(s)) <= slack  # all of it is the rest's
