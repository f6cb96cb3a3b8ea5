"""The distillation loss and its gradient against the definition in 64 bits, on the CPU.

A sum of exponentials over V terms in fp32 is off by delta = 2^-24 (3 D + V / 4096 + 8)
relative to itself: its arguments (x - m) c carry three roundings, which weigh in by
their share (D = the mean distance from the maximum, over T), a thread adds up to
V / 4096 + 2 vectors, three roundings of the tree and one and a half steps of the
exponential, and the merges. The loss takes the logarithms of two such sums, times P
and r, and one rounding. An element of the gradient is a difference of two terms
(P q and p, or P q and r q / s), each off by delta and its own exponential's
2^-24 (3 |x - m| / T + 3), then rounded to the logits' type."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32
INF, NAN = float("inf"), float("nan")
STEP = 2.0 ** -24


def _spread(e, z):
    """Mean distance from the maximum of the weights e = exp(z)."""
    return (e * torch.where(e > 0, -z, 0.0)).sum(-1) / e.sum(-1).clamp(min=1e-300)


def _reference(x, t, ids, norm, temperature, total=None):
    """(loss, its slack, gradient, its slack) per token, of fp64 rows [n, V]."""
    x, t, ids = x.double(), t.double(), ids.clone()
    n, v = x.shape
    z = x / temperature
    loss, loss_slack = torch.zeros(n, dtype=torch.float64), torch.zeros(n, dtype=torch.float64)
    grad = torch.zeros(n, v, dtype=torch.float64)
    slack = torch.zeros(n, v, dtype=torch.float64)
    for i in range(n):
        held = (ids[i] >= 0) & (ids[i] < v)
        if not bool(held.any()):
            continue
        at, te = ids[i][held], t[i][held] / temperature
        if norm is None:
            if bool((te == -INF).all()):
                continue
            lp = te - torch.logsumexp(te, 0)
            r = 0.0
        else:
            lp = te - float(norm[i])
            r = max(1.0 - float(torch.exp(lp).sum()), 0.0)
        p = torch.exp(lp)
        row = z[i]
        if bool(torch.isnan(row).any()) or bool((row == INF).any()) or bool((row == -INF).all()):
            loss[i], grad[i] = NAN, NAN
            continue
        m = row.max()
        e = torch.exp(row - m)
        listed = torch.zeros(v, dtype=torch.bool)
        listed[at] = True
        q = e / e.sum()
        delta = STEP * (3 * float(_spread(e, row - m)) + v / 4096 + 8)
        lq = row - m - torch.log(e.sum())
        use = p > 0
        one = float((p[use] * (lp[use] - lq[at][use])).sum())
        d_out = 0.0
        zo = torch.where(listed, -INF, row)  # (relative to their own maximum: no underflow)
        mo = zo.max()
        rest = r > 0 and float(mo) > -INF
        if rest:
            eo = torch.exp(zo - mo)
            log_s = float(mo - m + torch.log(eo.sum()) - torch.log(e.sum()))
            one += r * (math.log(r) - log_s)
            d_out = STEP * (3 * float(_spread(eo, zo - mo)) + v / 4096 + 8)
            share = r * eo / eo.sum()
        big = float(p.sum()) + (r if rest else 0.0)
        loss[i] = one
        loss_slack[i] = STEP * abs(one) + (big + r) * (delta + d_out)
        dense = torch.zeros(v, dtype=torch.float64).index_add_(0, at, p)
        g = big * q - dense
        size = big * q * (delta + STEP * (3 * (m - row).clamp(max=100.0) + 4)) + dense * 2 * STEP
        if rest:
            g = g - share
            size = size + share * (d_out + delta + STEP * (3 * (mo - zo).clamp(0.0, 100.0) + 4))
        grad[i] = g / temperature
        slack[i] = torch.where(q == 0, 0.0, size) / temperature + dense * STEP
    return loss, loss_slack, grad, slack


def _within(got, want, slack, dtype, what):
    got = got.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    same = got == want
    odd = ~torch.isfinite(want)
    assert bool(same[odd & ~torch.isnan(want)].all()), what
    info = torch.finfo(dtype)
    bound = slack + (want.abs() + slack) * info.eps / 2 + 2.0 ** -125
    ok = ((got - want).abs() <= bound) | same | odd
    assert bool(ok.all()), (what, float(((got - want).abs() / bound)[~ok].max()))


def _loss(x, t, ids, norm=None, temperature=1.0, **kw):
    import nmce
    return nmce.vocab_parallel_distillation_loss(
        x, t.to(DEV), ids.to(DEV), 0, x.shape[-1], nmce.ParallelContext.single(),
        teacher_log_normalizer=None if norm is None else norm.to(DEV), temperature=temperature,
        **kw)


def _check(x, t, ids, norm=None, temperature=1.0):
    """Per-token losses with their own upstream values, and the mean."""
    n, v = x.shape
    loss, loss_slack, grad, slack = _reference(x, t, ids, norm, temperature)
    up = torch.linspace(-1.0, 2.0, n) + 0.3
    d = x.to(DEV).requires_grad_(True)
    got = _loss(d, t, ids, norm, temperature, reduction="none")
    assert got.dtype == F32 and got.shape == (n,)
    _within(got.detach(), loss, loss_slack, F32, "loss")
    g, = torch.autograd.grad(got, d, up.to(DEV))
    assert g.dtype == x.dtype
    w = up.double()[:, None]
    # (the upstream value over T is one rounding, the product another)
    _within(g, torch.where(torch.isnan(grad), grad, grad * w),
            (slack + 3 * STEP * grad.abs().nan_to_num()) * w.abs(), x.dtype, "gradient")
    mean = _loss(d, t, ids, norm, temperature)
    assert mean.shape == ()
    if not bool(torch.isfinite(loss).all()):
        return
    want = loss.mean()
    assert abs(float(mean.detach()) - float(want)) <= float(loss_slack.mean()) + \
        STEP * (abs(float(want)) + 4 * float(loss.abs().mean()))
    g, = torch.autograd.grad(mean * 0.5, d)
    _within(g, grad * (0.5 / n), (slack + 4 * STEP * grad.abs()) * (0.5 / n), x.dtype, "mean")
    again = _loss(d, t, ids, norm, temperature)
    one, = torch.autograd.grad(again, d)
    _within(one, grad / n, (slack + 4 * STEP * grad.abs()) / n, x.dtype, "mean")
    # Without a gradient, and by two passes: sums in another order, within the same bound.
    slack_mean = float(loss_slack.mean()) + STEP * (abs(float(want)) + 4 * float(
        loss.abs().mean()))
    with torch.no_grad():
        other = _loss(d, t, ids, norm, temperature)
    two = _loss(d, t, ids, norm, temperature, one_pass=False)
    assert abs(float(other) - float(want)) <= slack_mean and torch.equal(two.detach(), other)
    g, = torch.autograd.grad(two, d)
    _within(g, grad / n, (slack + 4 * STEP * grad.abs()) / n, x.dtype, "two passes")


def _inputs(n, v, k, dtype, g, teacher_dtype=F32, temperature=1.0, spread=2.0):
    x = (torch.randn(n, v, generator=g) * spread).to(dtype)
    t = x.float() + torch.randn(n, v, generator=g) * 0.7
    values, ids = torch.topk(t, k, dim=1)
    norm = torch.logsumexp(t.double() / temperature, dim=1).float()
    values = values.to(teacher_dtype)
    if n > 3:
        ids[1] = -1  # no teacher
        ids[2, (k + 1) // 2:] = -1  # a shorter list
    return x, values, ids, norm


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("n,v,k", [
    (1, 1, 1), (2, 2, 1), (3, 2, 2), (5, 7, 3), (4, 64, 64), (6, 63, 5), (7, 1000, 20),
    (3, 1025, 1000), (9, 4099, 64), (4, 8192, 63), (5, 8193, 65), (70, 300, 17), (4, 16391, 128),
    (5, 50257, 20), (4, 65537, 512), (4, 100277, 50), (4, 131072, 64), (4, 131073, 64),
    (4, 151936, 1024)])
def test_against_the_definition(n, v, k, dtype, tail):
    g = torch.Generator().manual_seed(n + v + k)
    x, t, ids, norm = _inputs(n, v, k, dtype, g)
    _check(x, t, ids, norm if tail else None)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("temperature", [0.25, 2.0, 7.5])
@pytest.mark.parametrize("dtype,teacher", [(F32, BF), (BF, BF), (BF, F32)])
def test_temperatures_and_teacher_types(dtype, teacher, temperature, tail):
    g = torch.Generator().manual_seed(3)
    x, t, ids, norm = _inputs(6, 5003, 40, dtype, g, teacher, temperature)
    _check(x, t, ids, norm if tail else None, temperature)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF])
def test_an_id_that_comes_again(dtype, tail):
    g = torch.Generator().manual_seed(4)
    x = (torch.randn(5, 300, generator=g) * 2).to(dtype)
    ids = torch.tensor([[7, 7, 7, 9], [1, 2, 1, 2], [299, 0, 299, -1], [5, 5, 5, 5],
                        [8, 9, 10, 8]])
    t = torch.randn(5, 4, generator=g)
    t[4] = torch.tensor([1.0, 2.0, -INF, -INF])
    norm = torch.logsumexp(t, 1) + 0.5 if tail else None
    _check(x, t, ids, norm)
    # a long list of few ids
    many = torch.randint(0, 40, (5, 700), generator=g)
    t = torch.randn(5, 700, generator=g)
    _check(x, t, many, torch.logsumexp(t, 1) + 0.1 if tail else None)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_lists_that_are_the_whole_vocabulary(dtype):
    g = torch.Generator().manual_seed(5)
    x = (torch.randn(4, 200, generator=g) * 2).to(dtype)
    t = torch.randn(4, 200, generator=g)
    ids = torch.stack([torch.randperm(200, generator=g) for _ in range(4)])
    _check(x, t, ids)
    # what rounding leaves for the rest has no class to go to
    _check(x, t, ids, torch.logsumexp(t, 1) + torch.tensor([0.0, 1e-6, 0.5, -1e-6]))


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF])
def test_masked_infinite_and_missing(dtype, tail):
    g = torch.Generator().manual_seed(6)
    v = 9000
    x, t, ids, norm = _inputs(16, v, 8, dtype, g)
    ids[1:3] = ids[4:6]
    x[0] = -INF  # no distribution
    x[1, 17] = NAN
    x[2, 100] = INF
    x[3, ids[3, 0]] = INF
    x[4, ids[4, 2]] = NAN
    x[5, ids[5, 1]] = -INF  # the teacher's token is masked: an infinite loss
    x[6] = -INF
    x[6, ids[6]] = 1.0  # nothing outside the list
    x[7, torch.arange(v) % 2 == 0] = -INF
    x[7, ids[7]] = torch.arange(8.0).to(dtype)
    x[8] = torch.finfo(dtype).min
    x[8, ids[8, :3]] = 0.0
    ids[9] = torch.tensor([-1, v, 2 ** 40, -2 ** 40, v + 1, -7, 2 ** 31, 2 ** 32])  # none
    x[10], ids[10] = NAN, -1  # no teacher: nothing matters
    t[11, 2:] = -INF
    x[12, ids[12, 0]] += 100.0  # a confident student
    x[13, v - 1] += 200.0  # one that is confident elsewhere
    t[14] = -INF
    x[15] = 0.0
    _check(x, t, ids, norm if tail else None)


@pytest.mark.parametrize("tail", [False, True])
def test_against_differences(tail):
    """(L(z + h v) - L(z - h v)) / 2h = <dL, v> + h^2 / 6 L''' with |L'''| at most 2 for
    |v| <= 1 (third moments of two distributions), and the losses' roundings over h."""
    g = torch.Generator().manual_seed(7)
    n, v, k, h = 6, 2000, 30, 0.05
    x, t, ids, norm = _inputs(n, v, k, F32, g)
    norm = norm if tail else None
    d = x.to(DEV).requires_grad_(True)
    loss = _loss(d, t, ids, norm, reduction="none")
    grad, = torch.autograd.grad(loss.sum(), d)
    for _ in range(4):
        w = torch.rand(n, v, generator=g) * 2 - 1
        up, down = (_loss((x + s * h * w).to(DEV), t, ids, norm, reduction="none").double()
                    for s in (1, -1))
        slope = (grad.double().cpu() * w).sum(1)
        err = ((up - down).cpu() / (2 * h) - slope).abs()
        assert bool((err <= h * h / 6 * 2 + (loss.detach().cpu() + 20) * 1e-6 / h).all())


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("inplace", [True, False])
def test_in_place_and_strides(dtype, inplace):
    """Logits as an op's output, with padding between rows, and not viewable as rows."""
    g = torch.Generator().manual_seed(8)
    x, t, ids, norm = _inputs(6, 5001, 20, dtype, g)
    loss, loss_slack, grad, slack = _reference(x, t, ids, norm, 1.0)
    for reduction in ("none", "mean"):
        scale = 1.0 / 6 if reduction == "mean" else 1.0
        for layout in ("plain", "padded", "turned"):
            leaf = torch.zeros(6, 5001, dtype=dtype, device=DEV, requires_grad=True)
            if layout == "plain":
                y = leaf + x.to(DEV)
            elif layout == "padded":
                wide = torch.nn.functional.pad(leaf + x.to(DEV), (3, 12))
                y = wide[:, 3:5004]
            else:
                y = (leaf.t() + x.to(DEV).t()).contiguous().t()
            keep = y.detach().clone()
            out = _loss(y, t, ids, norm, reduction=reduction, inplace=inplace)
            if reduction == "none":
                _within(out.detach(), loss, loss_slack, F32, "loss")
            if not inplace:
                assert torch.equal(y.detach(), keep)
            out.sum().backward()
            _within(leaf.grad, grad * scale, (slack + 4 * STEP * grad.abs()) * scale, dtype,
                    (reduction, layout))
            if not inplace:
                assert torch.equal(y.detach(), keep)
    if inplace:
        leaf = x.to(DEV).requires_grad_(True)
        with pytest.raises(ValueError, match="leaf"):
            _loss(leaf, t, ids, norm, inplace=True)


def test_shapes_and_empty():
    g = torch.Generator().manual_seed(9)
    x, t, ids, norm = _inputs(6, 700, 9, BF, g)
    want = _loss(x.to(DEV), t, ids, norm, reduction="none")
    got = _loss(x.view(2, 3, 700).to(DEV), t.view(2, 3, 9), ids.view(2, 3, 9), norm.view(2, 3),
                reduction="none")
    assert got.shape == (2, 3) and torch.equal(got.view(-1), want)
    one = _loss(x[0].to(DEV), t[0], ids[0], norm[0], reduction="none")
    assert one.shape == () and torch.equal(one, want[0])
    # one list for all tokens, lists in the columns' order and among others
    same = _loss(x.to(DEV), t[:1].expand(6, 9), ids[:1].expand(6, 9), norm[:1].expand(6),
                 reduction="none")
    assert torch.equal(same, _loss(x.to(DEV), t[:1].repeat(6, 1), ids[:1].repeat(6, 1),
                                   norm[:1].repeat(6), reduction="none"))
    wide = torch.full((6, 20), 3, dtype=torch.int64)
    wide[:, 5:14] = ids
    assert torch.equal(_loss(x.to(DEV), t.t().contiguous().t(), wide.to(DEV)[:, 5:14], norm,
                             reduction="none"), want)
    x0 = torch.empty(0, 700, device=DEV, requires_grad=True)
    out = _loss(x0, t[:0], ids[:0], norm[:0], reduction="none")
    assert out.shape == (0,)
    assert torch.autograd.grad(out.sum(), x0)[0].shape == (0, 700)


def test_a_second_backward_and_no_second_derivative():
    g = torch.Generator().manual_seed(10)
    x, t, ids, norm = _inputs(5, 3001, 12, F32, g)
    d = x.to(DEV).requires_grad_(True)
    for reduction in ("mean", "none"):
        loss = _loss(d, t, ids, norm, reduction=reduction).sum()
        first, = torch.autograd.grad(loss, d, retain_graph=True)
        keep = first.clone()
        second, = torch.autograd.grad(loss, d, torch.tensor(3.0, device=DEV), retain_graph=True)
        third, = torch.autograd.grad(loss, d)
        assert torch.equal(first, keep) and torch.equal(third, keep)
        bound = 4 * STEP * (3 * keep).abs() + 1e-37
        assert bool(((second - 3 * keep).abs() <= bound).all())
        with pytest.raises(RuntimeError):
            grad, = torch.autograd.grad(_loss(d, t, ids, norm, reduction=reduction).sum(), d,
                                        create_graph=True)
            grad.sum().backward()


def test_two_losses_of_the_same_logits():
    """Cross entropy and distillation on one head's output, weighted, in one backward."""
    import nmce
    g = torch.Generator().manual_seed(11)
    ctx = nmce.ParallelContext.single()
    x, t, ids, norm = _inputs(8, 4000, 16, F32, g)
    target = torch.randint(0, 4000, (8,), generator=g)
    _, _, grad, slack = _reference(x, t, ids, norm, 1.0)
    leaf = x.to(DEV).requires_grad_(True)
    for _ in range(3):  # (the upstream values that the forwards assume change once)
        y = leaf * 1.0
        loss = 0.25 * nmce.vocab_parallel_cross_entropy(y, target.to(DEV), 0, 4000, ctx) + \
            0.75 * _loss(y, t, ids, norm)
        got, = torch.autograd.grad(loss, leaf)
        q = torch.softmax(x.double(), 1)
        want = 0.25 / 8 * (q - torch.nn.functional.one_hot(target, 4000)) + 0.75 / 8 * grad
        size = 0.75 / 8 * slack + STEP * (100 * q + 8 * want.abs()) / 8
        _within(got, want, size, F32, "sum")


def test_another_stream_and_captured():
    import nmce
    g = torch.Generator().manual_seed(12)
    ctx = nmce.ParallelContext.single()
    x, t, ids, norm = (a.to(DEV) for a in _inputs(12, 20000, 30, BF, g))

    def step(logits, tt, ii, nn, reduction):
        loss = nmce.vocab_parallel_distillation_loss(logits, tt, ii, 0, 20000, ctx,
                                                     teacher_log_normalizer=nn,
                                                     reduction=reduction)
        return loss.detach(), torch.autograd.grad(loss.sum(), logits)[0]

    for reduction in ("mean", "none"):
        logits = x.clone().requires_grad_(True)
        want = step(logits, t, ids, norm, reduction)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = step(logits, t, ids, norm, reduction)
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        static = [a.clone() for a in (t, ids, norm)]
        with torch.cuda.stream(side):
            step(logits, *static, reduction)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(logits, *static, reduction)
        for seed in range(3):
            new = _inputs(12, 20000, 30, BF, torch.Generator().manual_seed(seed))
            with torch.no_grad():
                for a, b in zip([logits] + static, new):
                    a.copy_(b)
            graph.replay()
            torch.cuda.synchronize()
            eager = step(logits, *static, reduction)
            assert all(torch.equal(a, b) for a, b in zip(out, eager))


@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_saved_tensor_hooks(reduction):
    """Tensors kept on the host, or handed back as copies; others are refused."""
    g = torch.Generator().manual_seed(13)
    x, t, ids, norm = _inputs(5, 2001, 9, F32, g)
    d = x.to(DEV).requires_grad_(True)

    def run(pack, unpack):
        with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
            loss = _loss(d, t, ids, norm, reduction=reduction).sum()
        return torch.autograd.grad(loss, d)[0]

    want = run(lambda a: a, lambda a: a)
    assert torch.equal(run(lambda a: a.cpu(), lambda a: a.to(DEV)), want)
    assert torch.equal(run(lambda a: a, lambda a: a.t().contiguous().t() if a.dim() == 2 else
                           a.clone()), want)
    with pytest.raises(RuntimeError, match="hooks"):
        run(lambda a: a, lambda a: a.cpu())
    with pytest.raises(RuntimeError, match="hooks"):
        run(lambda a: a, lambda a: a[:1] if a.dim() else a.double())


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("v", [4000, 4001])
def test_in_place_of_rows_that_share_memory(v, dtype):
    """An expanded tensor's gradient does not fit its storage: it goes into a buffer."""
    g = torch.Generator().manual_seed(15)
    x, t, ids, norm = _inputs(4, v, 6, dtype, g)
    leaf = x[:1].to(DEV).requires_grad_(True)
    for one_pass in (True, False):
        for up in (1.0, 0.5, 0.5, 1.0):  # (assumed or not)
            got = []
            for inplace in (True, False):
                y = (leaf * 1.0).expand(4, v)
                y.retain_grad()
                loss = _loss(y, t, ids, norm, inplace=inplace, one_pass=one_pass)
                (loss * up).backward()
                got.append(y.grad)
            assert torch.equal(y, leaf.expand(4, v)) and torch.equal(*got)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_a_teacher_whose_row_was_masked(dtype):
    """What the top logits of a row of only -inf are: no teacher."""
    import nmce
    ctx = nmce.ParallelContext.single()
    g = torch.Generator().manual_seed(16)
    teacher = torch.randn(5, 300, generator=g)
    teacher[2] = -INF
    t, ids, norm = nmce.vocab_parallel_top_logits(teacher.to(DEV), 8, 0, 300, ctx)
    assert float(norm[2]) == -INF
    x = torch.randn(5, 300, generator=g).to(dtype)
    d = x.to(DEV).requires_grad_(True)
    rest = torch.tensor([0, 1, 3, 4])
    for reduction in ("none", "mean"):
        loss = _loss(d, t, ids, norm, reduction=reduction)
        grad, = torch.autograd.grad(loss.sum(), d)
        assert not bool(grad[2].any()) and bool(torch.isfinite(loss).all())
        if reduction == "none":
            assert float(loss.detach()[2]) == 0.0
            want, slack, _, _ = _reference(x[rest], t.cpu()[rest], ids.cpu()[rest],
                                           norm.cpu()[rest], 1.0)
            _within(loss.detach()[rest.to(DEV)], want, slack, F32, "loss")


@pytest.mark.parametrize("n", [1023, 1025, 9000, 70000])
def test_means_of_many_tokens(n):
    """In the loss's own workgroup, and of as many rows as there are, in a captured graph too:
    a sum in 64 bits of fp32 losses, rounded once."""
    g = torch.Generator().manual_seed(n)
    v = 40
    x, t, ids, norm = (a.to(DEV) for a in _inputs(n, v, 3, F32, g))
    d = x.clone().requires_grad_(True)

    def run():
        one = _loss(d, t, ids, norm)
        two = _loss(d, t, ids, norm, one_pass=False)
        return one, two, torch.autograd.grad(one, d)[0], torch.autograd.grad(two, d)[0]

    def check(out):
        each = _loss(d, t, ids, norm, reduction="none").detach().double()
        one, two, g1, g2 = (o.detach().double() for o in out)
        # The one-pass losses are sums in another order. Of 40 logits the mean distance from
        # the largest is at most 2, so _reference's slacks are at most |loss| + 60 and 64 steps.
        size = 2 * STEP * (float(each.abs().mean()) + 60)
        assert abs(float(two - each.mean())) <= STEP * abs(float(each.mean())) + 1e-12
        assert abs(float(one - each.mean())) <= size
        assert bool(((g1 - g2).abs() <= 2 * STEP * 64 / n).all())

    check(run())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for seed in range(3):
        with torch.no_grad():
            d.copy_(torch.randn(n, v, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        check(out)


def test_an_upstream_hint_and_its_miss():
    g = torch.Generator().manual_seed(17)
    x, t, ids, norm = _inputs(6, 5000, 7, F32, g)
    leaf = x.to(DEV).requires_grad_(True)
    want, = torch.autograd.grad(_loss(leaf, t, ids, norm, one_pass=False), leaf)
    for inplace in (False, True):
        hint = torch.ones(1, device=DEV)
        for start, up in ((1.0, 1.0), (1.0, 4.0), (4.0, 4.0), (math.inf, 2.0), (0.0, 2.0),
                          (math.nan, -0.5), (2.0, 0.0)):
            hint.fill_(start)
            y = leaf * 1.0
            loss = _loss(y, t, ids, norm, upstream_hint=hint, inplace=inplace)
            got, = torch.autograd.grad(loss, leaf, torch.tensor(up, device=DEV))
            assert float(hint) == up
            # (_reference's slack: at most 128 steps where 3 x the mean distance from the
            # largest of 5000 logits, two sums and their elements come together; two sides)
            bound = 2 * 128 * STEP * abs(up) / 6 + 4 * STEP * (want * up).abs()
            assert bool(((got - want * up).abs() <= bound).all()), (inplace, start, up)


def test_threads_on_streams_of_their_own():
    """Two callers at once, of one call site, under different upstream values."""
    import threading
    g = torch.Generator().manual_seed(18)
    data = [_inputs(64, 30000, 20, BF, g) for _ in range(2)]
    data = [tuple(a.to(DEV) for a in d) for d in data]
    ups = (1.0, 8.0)

    def grad_of(i, one_pass):
        x, t, ids, norm = data[i]
        d = x.detach().requires_grad_(True)
        loss = _loss(d, t, ids, norm, one_pass=one_pass)
        return torch.autograd.grad(loss, d, torch.tensor(ups[i], device=DEV))[0]

    # A value that the forward assumed and one written again: the same formula.
    want = [grad_of(i, True) for i in range(2)]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(12):
                got = grad_of(i, True)
                ok = (got.float() - want[i].float()).abs() <= 2.0 ** -7 * want[i].float().abs() + \
                    1e-6 * ups[i] / 64
                if not bool(ok.all()):
                    wrong.append(i)
        stream.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not wrong


@pytest.mark.parametrize("mean", [False, True])
@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF])
def test_the_ranks_node_is_the_single_one(dtype, inplace, mean):
    """The node of several ranks, of one: the same kernels, storage and refusals."""
    from nmce.distill import _VocabParallelDistillation as Node
    g = torch.Generator().manual_seed(20)
    n, v = 6, 3003
    x, t, ids, norm = (a.to(DEV) for a in _inputs(n, v, 11, dtype, g))
    up = torch.tensor(0.75, device=DEV) if mean else \
        torch.linspace(-1.0, 2.0, n, device=DEV)
    wide = torch.zeros(n, v + 5, dtype=dtype, device=DEV)
    wide[:, :v] = x
    for rows in (lambda y: y, lambda y: y.t().contiguous().t(), lambda y: y.view(2, 3, v)):
        got = []
        for node in (True, False):
            leaf = wide.clone().requires_grad_(True)
            y = rows((leaf * 1.0)[:, :v])
            lead = y.shape[:-1]
            args = [t.view(*lead, 11), ids.view(*lead, 11), norm.view(lead)]
            if node:
                loss = Node.apply(y, *args, 0, None, 1, 1.0, mean, inplace)
            else:
                loss = _loss(y, *args, reduction="mean" if mean else "none", inplace=inplace,
                             one_pass=False)
            grad, = torch.autograd.grad(loss, leaf, up.view(loss.shape), retain_graph=True)
            got.append((loss.detach(), grad))
            if inplace and y._version:  # the logits hold the gradient now
                with pytest.raises(RuntimeError):
                    torch.autograd.grad(loss, leaf, up.view(loss.shape))
        assert all(torch.equal(a, b) for a, b in zip(*got))


def test_means_of_nothing():
    for one_pass in (True, False):
        x = torch.empty(0, 50, device=DEV, requires_grad=True)
        loss = _loss(x, torch.empty(0, 3), torch.empty(0, 3, dtype=torch.int64),
                     one_pass=one_pass)
        assert loss.shape == () and bool(torch.isnan(loss))
        assert torch.autograd.grad(loss, x)[0].shape == (0, 50)


@pytest.mark.parametrize("tail", [False, True])
def test_long_lists_of_few_ids(tail):
    """1024 entries of one id, of two in turn, and each of 512 twice."""
    g = torch.Generator().manual_seed(19)
    x = torch.randn(3, 2000, generator=g)
    t = torch.randn(3, 1024, generator=g)
    j = torch.arange(1024)
    ids = torch.stack([torch.full((1024,), 1999), j % 2 * 7, j % 512])
    _check(x, t, ids, torch.logsumexp(t.double(), 1).float() + 0.25 if tail else None)


def test_the_same_bits_at_every_run():
    g = torch.Generator().manual_seed(14)
    x, t, ids, norm = _inputs(20, 60000, 100, BF, g)
    ids[5:, 50:60] = ids[5:, 10:20]  # ids that come again
    d = x.to(DEV).requires_grad_(True)
    for reduction in ("mean", "none"):
        runs = []
        for _ in range(4):
            loss = _loss(d, t, ids, norm, reduction=reduction)
            runs.append((loss.detach(), torch.autograd.grad(loss.sum(), d)[0]))
        assert all(torch.equal(a, b) for r in runs[1:] for a, b in zip(r, runs[0]))


def test_rows_past_32_bit_offsets():
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB of device memory")
    n, v = 34000, 128256
    x = torch.zeros(n, v, dtype=BF, device=DEV, requires_grad=True)
    ids = torch.full((n, 2), -1, dtype=torch.int64, device=DEV)
    ids[-1] = torch.tensor([5, 128000])
    t = torch.zeros(n, 2, device=DEV)
    for reduction in ("none", "mean"):
        loss = _loss(x, t, ids, reduction=reduction)
        up = 1.0 if reduction == "none" else 1.0 / n
        assert abs(float(loss.detach().sum()) / up - math.log(v / 2)) <= 1e-5 * math.log(v / 2)
        grad, = torch.autograd.grad(loss.sum(), x)
        assert not bool(grad[:-1].any())
        row = grad[-1].double() / up
        assert abs(float(row[5]) + 0.5) < 4e-3 and abs(float(row[128000]) + 0.5) < 4e-3
        assert abs(float(row[7]) * v - 1.0) < 1e-2
        del grad, row, loss
