"""The embedding lookup and its gradient against 64-bit sums.

Bounds. The forward multiplies once in fp32 (2^-24 relative) and rounds to the
output type (half a step: 2^-8 for bf16, 2^-24 for fp32). A gradient element is
a sum of m fp32 terms in some order (at most m roundings of partial sums that no
sum of magnitudes exceeds: m 2^-24 sum|dY|), one fp32 product with the scale and
one rounding to the weight's type. Values here stay far from the subnormals.
"""

from __future__ import annotations

import types

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
BF, F32 = torch.bfloat16, torch.float32


def _reference(tokens, weight, grad, start, scale):
    """(out, dW, sum|dY| * |scale|, terms per row) in 64 bits on the CPU."""
    t = tokens.reshape(-1).cpu()
    v, h = weight.shape
    inside = (t >= start) & (t < start + v)
    local = torch.where(inside, t - start, torch.zeros_like(t))
    w = weight.detach().double().cpu()
    out = torch.where(inside[:, None], w[local] * scale, torch.zeros((), dtype=torch.float64))
    g = grad.double().cpu().reshape(-1, h)[inside]
    dw = torch.zeros(v, h, dtype=torch.float64).index_add_(0, local[inside], g)
    mag = torch.zeros(v, h, dtype=torch.float64).index_add_(0, local[inside], g.abs())
    terms = torch.bincount(local[inside], minlength=v).double()[:, None]
    return out, dw * scale, mag * abs(scale), terms


def _check(out, dw, tokens, weight, grad, start, scale):
    ref, rdw, mag, terms = _reference(tokens, weight, grad, start, scale)
    got = out.detach().double().cpu().reshape(ref.shape)
    err = (got - ref).abs()
    assert bool((err <= ref.abs() * (HALF_STEP[out.dtype] + 2.0 ** -23)).all())
    got = dw.double().cpu()
    bound = mag * (terms + 1) * 2.0 ** -24 * 1.01
    bound = bound + (rdw.abs() + bound) * HALF_STEP[dw.dtype]
    err = (got - rdw).abs()
    assert bool((err <= bound).all()), (err - bound).max()


def _ids(kind, n, v, start, g):
    if kind == "same":
        return torch.full((n,), start + v // 2, dtype=torch.int64)
    if kind == "two":
        return start + torch.randint(0, 2, (n,), generator=g) * (v - 1)
    if kind == "outside":
        return torch.tensor([start - 1, start + v, -1, 1 << 62, -(1 << 63), (1 << 63) - 1])[
            torch.arange(n) % 6]
    if kind == "wide":  # half of them other shards'
        return start + torch.randint(-v, v, (n,), generator=g)
    if kind == "text":
        u = torch.rand(n, generator=g, dtype=torch.float64)
        return start + (torch.exp(u * torch.log(torch.tensor(v + 1.0))) - 1).long().clamp_(0, v - 1)
    return start + torch.randint(0, v, (n,), generator=g)


CASES = [
    # n, h, v, start, weight, output, ids
    (1, 1, 1, 0, F32, F32, "any"),
    (1, 8, 5, 0, BF, BF, "any"),
    (3, 7, 2, 9, F32, BF, "any"),
    (64, 512, 100, 0, BF, BF, "same"),
    (65, 513, 100, 100, F32, F32, "two"),
    (100, 520, 1000, 0, BF, F32, "any"),
    (777, 1601, 300, 300, F32, F32, "wide"),
    (500, 768, 50304, 0, F32, BF, "text"),
    (600, 64, 40, 7, BF, BF, "outside"),
    (4096, 136, 511, 0, F32, F32, "any"),      # one whole tile, one digit
    (4097, 40, 512, 0, BF, BF, "text"),        # a key more than nine bits, a tile and one
    (16384, 72, 128256, 0, BF, BF, "text"),
    (14336, 64, 32000, 0, BF, BF, "same"),
    (14337, 64, 32000, 5, BF, BF, "wide"),
    (16385, 40, 50257, 0, BF, F32, "text"),    # one more than one workgroup sorts
    (20011, 24, 262143, 0, F32, F32, "any"),   # 18 bits of key
    (20011, 24, 262144, 0, F32, F32, "text"),  # 19: three passes
    (131072, 16, 97, 0, BF, F32, "any"),       # hundreds of chunks an id
    (300000, 8, 1000, 0, F32, BF, "two"),      # tiles larger than the smallest
    (70001, 9, 500, 0, F32, BF, "any"),        # eight rows a wave: an odd width,
    (70003, 12, 300, 300, F32, F32, "wide"),   # and whole vectors with a rest
]


@pytest.mark.parametrize("n,h,v,start,wd,od,kind", CASES)
def test_embedding_and_gradient(n, h, v, start, wd, od, kind):
    import nmce
    g = torch.Generator().manual_seed(n + h)
    tokens = _ids(kind, n, v, start, g).to(DEV)
    weight = (torch.randn(v, h, generator=g) * 0.02).to(wd).to(DEV).requires_grad_(True)
    grad = torch.randn(n, h, generator=g).to(od).to(DEV)
    scale = 1.0 if h == 1 else h ** 0.5
    out = nmce.vocab_parallel_embedding(tokens, weight, start, start + v,
                                        nmce.ParallelContext.single(), scale=scale, out_dtype=od,
                                        validate=False)
    assert out.shape == (n, h) and out.dtype == od
    dw, = torch.autograd.grad(out, weight, grad, retain_graph=True)
    assert dw.dtype == wd
    _check(out, dw, tokens, weight, grad, start, scale)
    again, = torch.autograd.grad(out, weight, grad)
    assert torch.equal(dw, again)  # the order of the sums is fixed


def test_no_tokens():
    import nmce
    weight = torch.randn(10, 6, device=DEV, requires_grad=True)
    tokens = torch.zeros(2, 0, dtype=torch.int64, device=DEV)
    out = nmce.vocab_parallel_embedding(tokens, weight, 0, 10, nmce.ParallelContext.single())
    assert out.shape == (2, 0, 6)
    dw, = torch.autograd.grad(out, weight, torch.zeros_like(out))
    assert dw.shape == weight.shape and not dw.any()


@pytest.mark.parametrize("wd", [F32, BF])
def test_strides(wd):
    """Ids transposed, a weight of wider rows that starts off the 16-byte grid,
    a weight whose columns are strided, a transposed and an expanded gradient."""
    import nmce
    ctx = nmce.ParallelContext.single()
    g = torch.Generator().manual_seed(3)
    v, h = 50, 72
    tokens = torch.randint(0, v, (9, 5), generator=g).to(DEV).t()
    wide = torch.randn(v, h + 9, generator=g).to(wd).to(DEV)
    for weight in (wide[:, 1:h + 1], wide[:, :h], wide.t().contiguous()[:h].t(),
                   wide[:1, :h].expand(v, h)):
        leaf = weight.detach().requires_grad_(True)
        assert leaf.stride() == weight.stride()
        out = nmce.vocab_parallel_embedding(tokens, leaf, 0, v, ctx, scale=-0.5)
        assert out.shape == (5, 9, h) and out.is_contiguous()
        for grad in (torch.randn(9, 5, h, generator=g).to(wd).to(DEV).transpose(0, 1),
                     torch.randn(5, 9, h + 3, generator=g).to(wd).to(DEV)[..., 3:],
                     torch.ones((), dtype=wd, device=DEV).expand(5, 9, h),
                     torch.randn(1, 1, h, generator=g).to(wd).to(DEV).expand(5, 9, h)):
            dw, = torch.autograd.grad(out, leaf, grad, retain_graph=True)
            _check(out, dw, tokens, leaf, grad, 0, -0.5)


def test_nan_and_infinity_stay_in_their_rows():
    import nmce
    weight = torch.randn(20, 64, device=DEV)
    weight[3, 5], weight[4, 6] = float("nan"), float("inf")
    weight.requires_grad_(True)
    tokens = torch.tensor([2, 3, 4, 30, 5], device=DEV)
    out = nmce.vocab_parallel_embedding(tokens, weight, 0, 20, nmce.ParallelContext.single(),
                                        validate=False)
    bad = ~torch.isfinite(out)
    assert bad.nonzero().tolist() == [[1, 5], [2, 6]]
    grad = torch.randn(5, 64, device=DEV)
    grad[3] = float("nan")  # another shard's id
    grad[0, 9] = float("inf")
    dw, = torch.autograd.grad(out, weight, grad)
    assert (~torch.isfinite(dw)).nonzero().tolist() == [[2, 9]]


def test_ids_outside_the_vocabulary_are_refused():
    import nmce
    ctx = nmce.ParallelContext.single()
    weight = torch.randn(20, 64, device=DEV)
    for bad in (-1, 20, 1 << 40):
        tokens = torch.tensor([2, bad, 5], device=DEV)
        with pytest.raises(ValueError, match="outside the model vocabulary"):
            nmce.vocab_parallel_embedding(tokens, weight, 0, 20, ctx)
    with pytest.raises(ValueError, match=r"must be \[batch, seq\]"):
        nmce.vocab_parallel_embedding(torch.zeros(4, dtype=torch.int64, device=DEV), weight, 0, 20,
                                      ctx, sequence_parallel=True)
    two = nmce.ParallelContext(rank=0, world_size=2, tp_size=2, tp_rank=0, pp_size=1, pp_rank=0,
                               dp_size=1, dp_rank=0)
    with pytest.raises(ValueError, match="outside the model vocabulary"):
        nmce.vocab_parallel_embedding(torch.tensor([40], device=DEV), weight, 0, 20, two)


def test_workspace_and_output_bounds():
    """The backward through the C ABI with guard bytes around dW and the workspace."""
    from nmce import _lib as L
    lib = L.load()
    g = torch.Generator().manual_seed(8)
    for n, h, v in ((1, 1, 1), (100, 9, 33), (5000, 520, 700), (4500, 3, 2)):
        tokens = torch.randint(0, v, (n,), generator=g).to(DEV)
        dy = torch.randn(n, h, generator=g).to(DEV)
        need = lib.nmce_embedding_bwd_workspace_bytes(n, v, h)
        ws = torch.full((need + 512,), 0x5A, dtype=torch.uint8, device=DEV)
        dw = torch.full((v * h + 64,), 7.0, device=DEV)
        L.check(lib.nmce_embedding_bwd(tokens.data_ptr(), n, dy.data_ptr(), L.NMCE_F32, h, v, h, 0,
                                       1.0, dw.data_ptr() + 64, L.NMCE_F32, ws.data_ptr() + 256,
                                       need, L.stream_handle(torch.device(DEV))), "bwd")
        torch.cuda.synchronize()
        assert bool((ws[:256] == 0x5A).all()) and bool((ws[256 + need:] == 0x5A).all())
        assert bool((dw[:16] == 7.0).all()) and bool((dw[16 + v * h:] == 7.0).all())


def test_other_stream_and_repeated_calls():
    """Two backward passes in flight on two streams give what each gives alone."""
    import nmce
    ctx = nmce.ParallelContext.single()
    g = torch.Generator().manual_seed(5)
    weight = torch.randn(3000, 256, generator=g).to(BF).to(DEV).requires_grad_(True)
    jobs = []
    for i in range(2):
        tokens = torch.randint(0, 3000, (6000 + i,), generator=g).to(DEV)
        grad = torch.randn(6000 + i, 256, generator=g).to(BF).to(DEV)
        out = nmce.vocab_parallel_embedding(tokens, weight, 0, 3000, ctx)
        jobs.append((tokens, grad, torch.autograd.grad(out, weight, grad)[0]))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    got = []
    for (tokens, grad, _), stream in zip(jobs, streams):
        with torch.cuda.stream(stream):
            out = nmce.vocab_parallel_embedding(tokens, weight, 0, 3000, ctx, validate=False)
            got.append(torch.autograd.grad(out, weight, grad)[0])
    torch.cuda.synchronize()
    for (_, _, want), dw in zip(jobs, got):
        assert torch.equal(want, dw)


def test_graph_replays():
    """Forward and backward captured in one graph, replayed on new ids with
    eager work in between."""
    import nmce
    ctx = nmce.ParallelContext.single()
    g = torch.Generator().manual_seed(6)
    n, h, v = 5000, 200, 700
    tokens = torch.zeros(n, dtype=torch.int64, device=DEV)
    grad = torch.zeros(n, h, device=DEV)
    weight = torch.randn(v, h, generator=g).to(DEV).requires_grad_(True)

    def step():
        out = nmce.vocab_parallel_embedding(tokens, weight, 0, v, ctx, validate=False)
        return out.detach(), torch.autograd.grad(out, weight, grad)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, dw = step()
    for _ in range(3):
        tokens.copy_(torch.randint(0, v, (n,), generator=g))
        grad.copy_(torch.randn(n, h, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone(), dw.clone()
        want = step()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_offsets_past_32_bits():
    """A weight and an output of more than 2^31 elements each, and dW of more than
    2^32 bytes: rows at both ends."""
    import nmce
    ctx = nmce.ParallelContext.single()
    v, h, n = 66000, 33000, 66000
    weight = torch.zeros(v, h, dtype=BF, device=DEV)
    weight[0], weight[v // 2], weight[v - 1] = 1.0, 2.0, 3.0
    weight.requires_grad_(True)
    tokens = torch.full((n,), -1, dtype=torch.int64, device=DEV)
    tokens[0], tokens[1], tokens[n - 2], tokens[n - 1] = v - 1, 0, v // 2, v - 1
    out = nmce.vocab_parallel_embedding(tokens, weight, 0, v, ctx, validate=False)
    rows = out.detach()[[0, 1, 2, n - 2, n - 1]]
    assert torch.equal(rows, torch.tensor([3.0, 1, 0, 2, 3], device=DEV).to(BF)[:, None].expand(5, h))
    assert not out.detach()[n // 2].any()
    grad = torch.zeros(n, h, dtype=BF, device=DEV)
    grad[0], grad[1], grad[n - 2], grad[n - 1] = 1.0, 4.0, 8.0, 2.0
    dw, = torch.autograd.grad(out, weight, grad)
    sums = dw.sum(dim=1, dtype=torch.float64)
    want = torch.zeros(v, dtype=torch.float64, device=DEV)
    want[0], want[v // 2], want[v - 1] = 4.0 * h, 8.0 * h, 3.0 * h
    assert torch.equal(sums, want)


def test_second_derivatives():
    """The weight's gradient is linear in the output's: its derivative is the
    lookup of the second gradient, and that one's the scatter again."""
    import nmce
    ctx = nmce.ParallelContext.single()
    g = torch.Generator().manual_seed(11)
    weight = torch.randn(30, 16, generator=g).to(DEV).requires_grad_(True)
    tokens = torch.randint(-5, 35, (4, 9), generator=g).to(DEV)
    dy = torch.randn(4, 9, 16, generator=g).to(DEV).requires_grad_(True)
    out = nmce.vocab_parallel_embedding(tokens, weight, 0, 30, ctx, scale=3.0, validate=False)
    dw, = torch.autograd.grad(out, weight, dy, create_graph=True)
    _check(out, dw.detach(), tokens, weight, dy.detach(), 0, 3.0)
    second = torch.randn(30, 16, generator=g).to(DEV).requires_grad_(True)
    ddy, = torch.autograd.grad(dw, dy, second, create_graph=True)
    back, = torch.autograd.grad(ddy, second, dy.detach())
    _check(ddy, back, tokens, second, dy.detach(), 0, 3.0)


def test_gradient_by_differences():
    """(f(W + e D) - f(W - e D)) / 2 e = <dW, D> for f = <out, dY>: f is linear, so
    the difference is exact up to fp32's rounding of the sums (2^-24 of their
    magnitudes, divided by e)."""
    import nmce
    ctx = nmce.ParallelContext.single()
    g = torch.Generator().manual_seed(12)
    tokens = torch.randint(0, 40, (200,), generator=g).to(DEV)
    w0, d = (torch.randn(40, 24, generator=g).to(DEV) for _ in range(2))
    dy = torch.randn(200, 24, generator=g).to(DEV)
    w = w0.clone().requires_grad_(True)
    out = nmce.vocab_parallel_embedding(tokens, w, 0, 40, ctx, scale=2.0)
    dw, = torch.autograd.grad(out, w, dy)
    step = 2.0 ** -3
    f = [nmce.vocab_parallel_embedding(tokens, w0 + s * step * d, 0, 40, ctx, scale=2.0).double()
         for s in (1, -1)]
    got = ((f[0] - f[1]) * dy.double()).sum() / (2 * step)
    want = (dw.double() * d.double()).sum()
    slack = ((f[0].abs() + f[1].abs()) * dy.double().abs()).sum() * 2.0 ** -23 / step
    assert abs(float(got - want)) <= float(slack)


def test_tied_with_the_fused_head():
    """One training step through both ends of a tied weight: the embedding's
    rows go straight into the fused head + loss. The gradient is the sum of
    both uses', each as it is alone."""
    import nmce
    ctx = nmce.ParallelContext.single()
    cfg = types.SimpleNamespace(vocab_size=1000, n_embd=128, sequence_parallel=False)
    torch.manual_seed(0)
    emb = nmce.VocabParallelEmbedding(cfg, ctx, scale=8.0).to(DEV)
    head = nmce.FusedParallelLMHead(cfg, ctx)
    head.weight = emb.weight
    g = torch.Generator().manual_seed(1)
    tokens = torch.randint(0, 1000, (2, 65), generator=g).to(DEV)
    x = emb(tokens[:, :-1], out_dtype=BF)
    with torch.autocast("cuda", dtype=BF):
        loss = head(x, tokens[:, 1:])
    loss.backward()
    # Each use on its own.
    w = emb.weight.detach().clone().requires_grad_(True)
    xin = x.detach().requires_grad_(True)
    with torch.autocast("cuda", dtype=BF):
        nmce.lmhead_vocab_parallel_cross_entropy(xin, w, tokens[:, 1:], 0, 1000, ctx).backward()
    _, rdw, mag, terms = _reference(tokens[:, :-1], w, xin.grad, 0, 8.0)
    want = rdw + w.grad.double().cpu()
    bound = mag * (terms + 1) * 2.0 ** -24 * 1.01 + (want.abs() + rdw.abs()) * 2.0 ** -23
    assert bool(((emb.weight.grad.double().cpu() - want).abs() <= bound).all())


def _with_hooks(unpack):
    return torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack)


def test_saved_ids_through_hooks():
    """Ids that saved-tensor hooks keep elsewhere (save_on_cpu) or hand back in other
    strides give the same gradients, the second ones too."""
    import nmce
    ctx = nmce.ParallelContext.single()
    g = torch.Generator().manual_seed(13)
    weight = torch.randn(300, 40, generator=g).to(DEV).requires_grad_(True)
    tokens = torch.randint(-5, 305, (9, 50), generator=g).to(DEV)
    dy = torch.randn(9, 50, 40, generator=g).to(DEV).requires_grad_(True)
    second = torch.randn(300, 40, generator=g).to(DEV)

    def step():
        out = nmce.vocab_parallel_embedding(tokens, weight, 0, 300, ctx, scale=2.0, validate=False)
        dw, = torch.autograd.grad(out, weight, dy, create_graph=True)
        return dw.detach(), torch.autograd.grad(dw, dy, second)[0]

    want = step()
    for hooks in (torch.autograd.graph.save_on_cpu(),
                  _with_hooks(lambda t: t.t().contiguous().t())):
        with hooks:
            got = step()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("what", ["device", "type", "fewer", "more", "shape"])
def test_other_ids_from_hooks_are_refused(what):
    """Hooks that hand back something else than the ids that were saved: nothing is
    launched on it, by the gradient and by the gradient's own backward."""
    import nmce
    ctx = nmce.ParallelContext.single()
    weight = torch.randn(30, 16, device=DEV, requires_grad=True)
    tokens = torch.arange(12, device=DEV).view(3, 4)
    unpack = {"device": lambda t: t.cpu(), "type": lambda t: t.int(), "fewer": lambda t: t[:2],
              "more": lambda t: torch.cat([t, t]), "shape": lambda t: t.view(4, 3)}[what]
    with _with_hooks(unpack):
        out = nmce.vocab_parallel_embedding(tokens, weight, 0, 30, ctx)
    with pytest.raises(RuntimeError, match="nmce: saved-tensor hooks"):
        out.sum().backward()
    dy = torch.randn(3, 4, 16, device=DEV, requires_grad=True)
    out = nmce.vocab_parallel_embedding(tokens, weight, 0, 30, ctx)
    with _with_hooks(unpack):
        dw, = torch.autograd.grad(out, weight, dy, create_graph=True)
    with pytest.raises(RuntimeError, match="nmce: saved-tensor hooks"):
        dw.sum().backward()


def test_a_weight_with_a_tangent_is_refused():
    """Forward-mode derivatives: refused, not dropped."""
    from torch.autograd import forward_ad
    import nmce
    weight, tokens = torch.randn(30, 16, device=DEV), torch.arange(12, device=DEV)
    with forward_ad.dual_level():
        for leaf in (weight, weight.clone().requires_grad_(True)):
            for mode in (torch.enable_grad, torch.no_grad):
                with mode(), pytest.raises((RuntimeError, NotImplementedError)):
                    nmce.vocab_parallel_embedding(
                        tokens, forward_ad.make_dual(leaf, torch.ones_like(weight)), 0, 30,
                        nmce.ParallelContext.single())


@pytest.mark.parametrize("n,h", [(530001, 8), (1100003, 8), (1100003, 9)])
@pytest.mark.parametrize("kind", ["lengths", "two", "any", "few"])
def test_long_chunks(n, h, kind):
    """Lists long enough that a wave adds 128 or 256 positions, 64 keys at a time, all
    of the shard: runs of equal ids that end on both sides of every 64th place and of
    the chunks' ends. Gradients are small integers, so every sum is exact."""
    import nmce
    g = torch.Generator().manual_seed(n + h)
    v = {"lengths": 20000, "two": 2, "any": 50257, "few": 700}[kind]
    if kind == "lengths":
        runs = torch.tensor([63, 1, 64, 65, 127, 128, 129, 191, 193, 255, 256, 257, 1, 2, 511, 513])
        ids = torch.arange(v).repeat_interleave(runs[torch.arange(v) % len(runs)])[:n]
        ids = ids[torch.randperm(n, generator=g)]
    else:
        ids = torch.randint(0, v, (n,), generator=g)
    grad = torch.randint(-3, 4, (n, h), generator=g)
    weight = torch.zeros(v, h, device=DEV, requires_grad=True)
    out = nmce.vocab_parallel_embedding(ids.to(DEV), weight, 0, v, nmce.ParallelContext.single(),
                                        scale=0.5, validate=False)
    dw, = torch.autograd.grad(out, weight, grad.float().to(DEV))
    want = torch.zeros(v, h, dtype=torch.int64).index_add_(0, ids, grad)
    assert torch.equal(dw.double().cpu() * 2.0, want.double())
