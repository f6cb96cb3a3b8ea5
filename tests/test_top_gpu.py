"""The top logits against a stable sort on the CPU: values and ids must be equal.

The log-normaliser against 64 bits. Its terms exp2((x - m) c) have arguments off by three
roundings, 3 2^-24 |x - m| / T each, which weigh in by their share p: 3 2^-24 D with D =
sum p (m - x) / T; a thread's sum of up to V / 4096 + 2 vectors adds a rounding a vector
besides three of the tree and the exponential's (one step and a half), and the result is
rounded to fp32: half a step."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32
INF, NAN = float("inf"), float("nan")


def _run(x, k, temperature=1.0):
    import nmce
    return nmce.vocab_parallel_top_logits(x.to(DEV), k, 0, x.shape[-1],
                                          nmce.ParallelContext.single(), temperature=temperature)


def _norm(x, t):
    """(log-normaliser in 64 bits, what its computation may be off by)."""
    z = x.double()
    m = z.amax(-1, keepdim=True)
    z = torch.where(torch.isfinite(m), z - m, torch.where(z == m, 0.0, -INF)) / t
    e = torch.exp(z)
    norm = m[..., 0] / t + torch.log(e.sum(-1))
    spread = (e * torch.where(z == -INF, 0.0, -z)).sum(-1) / e.sum(-1)
    steps = x.shape[-1] / 4096 + 8
    return norm, 2.0 ** -24 * (norm.abs() + 3 * spread + steps)


def _check(x, k, temperature=1.0):
    values, ids, norm = (t.cpu() for t in _run(x, k, temperature))
    want = torch.sort(x, dim=-1, descending=True, stable=True)
    assert values.dtype == x.dtype and values.shape == x.shape[:-1] + (k,)
    assert torch.equal(ids, want.indices[..., :k])
    top = want.values[..., :k]
    assert torch.equal(torch.isnan(values), torch.isnan(top))
    assert torch.equal(values[~torch.isnan(top)], top[~torch.isnan(top)])
    exact, slack = _norm(x, temperature)
    odd = ~torch.isfinite(exact)
    assert torch.equal(torch.isnan(norm), torch.isnan(exact))
    assert torch.equal(norm[odd & ~torch.isnan(exact)].double(),
                       exact[odd & ~torch.isnan(exact)])
    assert bool(((norm.double() - exact).abs()[~odd] <= slack[~odd]).all()), \
        ((norm.double() - exact).abs() / slack)[~odd].max()


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("n,v,k", [
    (1, 1, 1), (3, 2, 2), (5, 7, 3), (4, 64, 64), (7, 513, 512), (300, 1000, 20), (2, 4096, 1),
    (2, 4097, 33), (3, 8191, 500), (3, 8192, 512), (2, 16385, 64), (2, 32769, 512),
    (1, 50257, 20), (9, 50257, 5), (64, 50304, 64), (3, 128256, 512), (700, 20000, 50),
    (1, 300001, 100), (2, 1000003, 17), (33, 100277, 500)])
def test_against_a_stable_sort(n, v, k, dtype):
    g = torch.Generator().manual_seed(n + v + k)
    x = (torch.randn(n, v, generator=g) * 3).to(dtype)
    _check(x, k)
    _check(x, k, 0.6)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("v,k", [(100, 7), (20000, 64), (70000, 512), (140001, 300)])
def test_equal_logits(v, k, dtype):
    """Rows of one value, of few values, and masked but for a few: the lowest ids win."""
    g = torch.Generator().manual_seed(v)
    x = torch.zeros(8, v)
    x[1] = -5.0
    x[2] = torch.randint(0, 3, (v,), generator=g).float()
    x[3] = -INF
    x[4] = -INF
    x[4, torch.randint(0, v, (5,), generator=g)] = torch.randn(5, generator=g)
    x[5] = torch.finfo(dtype).min
    x[5, v // 2] = 1.0
    x[6] = torch.where(torch.arange(v) < v // 3, 1.0, 2.0)
    x[7] = torch.where(torch.arange(v) % 2 == 0, 0.0, -0.0)
    _check(x.to(dtype), k)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("v,k", [(300, 40), (40000, 100), (100000, 512)])
def test_orders(v, k, dtype):
    """Rising, falling, the largest in one thread's places, and in the last columns."""
    g = torch.Generator().manual_seed(k)
    x = torch.randn(6, v, generator=g)
    x[0] = torch.arange(v) / 7.0
    x[1] = -torch.arange(v) / 7.0
    x[2, ::4096 // 2] += 50.0
    x[3, :k] += 40.0
    x[4, -k:] += 40.0 + torch.arange(k) / 100.0
    x[5] = torch.sort(x[5]).values
    _check(x.to(dtype), k)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("v", [50, 9000, 90000])
def test_infinities_and_nan(v, dtype):
    g = torch.Generator().manual_seed(v)
    x = (torch.randn(7, v, generator=g) * 2).to(dtype)
    x[0, 3] = NAN
    x[1, v - 1] = INF
    x[2, 5], x[2, 7] = INF, NAN
    x[3, torch.randperm(v, generator=g)[:40]] = NAN
    x[4, 10:30] = INF
    x[5] = NAN
    x[6, 1:] = -INF
    _check(x, 20)
    _check(x, 45)


def test_values_far_apart_and_extreme_temperatures():
    g = torch.Generator().manual_seed(3)
    x = torch.randn(4, 5000, generator=g)
    x[0] *= 1e30
    x[1] *= 1e-30
    x[2] *= torch.exp(torch.randn(5000, generator=g) * 20)
    _check(x, 50)
    _check(x[1:2], 50, 100.0)
    _check(x[3:], 50, 0.01)
    _check(x[:1], 50, 1e30)
    _check(x[1:2], 50, 1e-30)
    _check(x, 50, 1e30)
    y = torch.full((1, 600), -INF)
    y[0, 7:9] = 3e38  # (over the highest temperature 3e8)
    _check(y, 5, 1e30)
    _check(torch.zeros(1, 600), 5, 1e-30)


def test_shapes_strides_and_empty():
    import nmce
    ctx = nmce.ParallelContext.single()
    g = torch.Generator().manual_seed(4)
    x = torch.randn(3, 5, 1001, generator=g).to(BF)
    _check(x, 10)
    _check(x[0, 0], 10)
    want = [t.cpu() for t in _run(x, 10)]

    def same(y):
        got = nmce.vocab_parallel_top_logits(y, 10, 0, 1001, ctx)
        assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want))

    big = torch.zeros(3, 5, 1024, dtype=BF, device=DEV)
    big[..., 3:1004] = x.to(DEV)
    same(big[..., 3:1004])
    same(x.to(DEV).transpose(0, 1).contiguous().transpose(0, 1))
    same(x.to(DEV).transpose(1, 2).contiguous().transpose(1, 2))
    one = nmce.vocab_parallel_top_logits(x[0, :1].to(DEV).expand(4, 1001), 10, 0, 1001, ctx)
    assert all(torch.equal(t, t[:1].expand_as(t)) for t in one)
    for lead in ((0,), (2, 0), (0, 3)):
        got = nmce.vocab_parallel_top_logits(torch.empty(lead + (1001,), device=DEV), 10, 0, 1001,
                                             ctx)
        assert [t.shape for t in got] == [lead + (10,), lead + (10,), lead]


def test_the_same_bits_at_every_run():
    g = torch.Generator().manual_seed(5)
    for n, v, k, dtype in ((40, 60000, 300, F32), (3, 128256, 64, BF)):
        x = torch.randn(n, v, generator=g).to(dtype).to(DEV)
        first = _run(x, k)
        for _ in range(5):
            assert all(torch.equal(a, b) for a, b in zip(_run(x, k), first))


def test_rows_past_32_bit_offsets():
    """The last row starts past 2^32 elements."""
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB of device memory")
    n, v = 34000, 128256
    x = torch.zeros(n, v, dtype=BF, device=DEV)
    x[n - 1, 128000] = 3.0
    x[n - 1, 5] = 2.0
    values, ids, norm = _run(x, 3)
    assert ids[-1].tolist() == [128000, 5, 0] and values[-1].tolist() == [3.0, 2.0, 0.0]
    assert torch.equal(ids[:-1], torch.arange(3, device=DEV).expand(n - 1, 3))


def test_another_stream():
    g = torch.Generator().manual_seed(6)
    x = torch.randn(6, 30000, generator=g)
    side = torch.cuda.Stream()
    d = x.to(DEV)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _run(d, 30)
    side.synchronize()
    assert torch.equal(got[1].cpu(), torch.sort(x, dim=-1, descending=True, stable=True)
                       .indices[:, :30])


def test_captured_and_replayed():
    import nmce
    ctx = nmce.ParallelContext.single()
    g = torch.Generator().manual_seed(7)
    x = torch.randn(4, 40000, generator=g).to(BF).to(DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        nmce.vocab_parallel_top_logits(x, 40, 0, 40000, ctx)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = nmce.vocab_parallel_top_logits(x, 40, 0, 40000, ctx)
    for _ in range(3):
        x.copy_(torch.randn(4, 40000, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        eager = nmce.vocab_parallel_top_logits(x, 40, 0, 40000, ctx)
        assert all(torch.equal(a, b) for a, b in zip(out, eager))
        assert torch.equal(out[1].cpu(), torch.sort(x.cpu(), dim=-1, descending=True, stable=True)
                           .indices[:, :40])


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("tp,per,k", [(2, 5, 9), (3, 1001, 40), (4, 20000, 512), (14, 600, 512),
                                      (15, 600, 512), (20, 3, 50), (72, 40, 100), (8, 9, 1)])
def test_shards_merged(tp, per, k, dtype):
    """Each shard's list and their merge, as the ranks exchange them."""
    from nmce import _lib as L
    lib = L.load()
    g = torch.Generator().manual_seed(per)
    n, v = 5, tp * per
    x = (torch.randn(n, v, generator=g) * 3).to(dtype)
    x[1] = 0.0
    code = L.dtype_code(dtype)
    parts = torch.zeros(tp, n, k + 1, dtype=torch.int64, device=DEV)
    stream = L.stream_handle(torch.device(DEV))
    for r in range(tp):
        mine = x[:, r * per:(r + 1) * per].contiguous().to(DEV)
        ws = torch.empty(lib.nmce_top_workspace_bytes(n, per, k), dtype=torch.uint8, device=DEV)
        L.check(lib.nmce_top_logits(mine.data_ptr(), code, n, per, per, r * per, k, 1.0,
                                    parts[r].data_ptr(), None, None, None, ws.data_ptr(),
                                    ws.numel(), stream), "top")
    values = torch.empty(n, k, dtype=dtype, device=DEV)
    ids = torch.empty(n, k, dtype=torch.int64, device=DEV)
    norm = torch.empty(n, device=DEV)
    L.check(lib.nmce_top_merge(parts.data_ptr(), tp, code, n, k, 1.0, values.data_ptr(),
                               ids.data_ptr(), norm.data_ptr(), stream), "merge")
    whole = _run(x, k)
    assert torch.equal(values, whole[0]) and torch.equal(ids, whole[1])
    exact, slack = _norm(x, 1.0)
    assert bool(((norm.cpu().double() - exact).abs() <= slack).all())


def test_refusals_on_the_device():
    import nmce
    ctx = nmce.ParallelContext.single()
    x = torch.randn(2, 50, device=DEV)
    with pytest.raises(RuntimeError, match="requires grad"):
        nmce.vocab_parallel_top_logits(x.clone().requires_grad_(True), 3, 0, 50, ctx)
    for k in (0, -1, 51, 513):
        with pytest.raises(ValueError, match="k must be"):
            nmce.vocab_parallel_top_logits(x, k, 0, 50, ctx)
