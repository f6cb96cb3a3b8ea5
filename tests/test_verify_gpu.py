"""Verification of drafted tokens against the definition in 64 bits, sequence by
sequence on the CPU. The tokens and counts must be equal: both sides carry 64
bits, so only a number within about 1e-13 of a border could tell them apart.
The log-probabilities are fp32 roundings of 64-bit values (half a step, plus
1e-7 for values near 0, where log p loses what p's own rounding, 2^-52, leaves).
"""

from __future__ import annotations

import math
import types

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32
INF, NAN = float("inf"), float("nan")


def _distribution(row, t):
    """softmax(row / t) in 64 bits, or None where there is none."""
    z = row.double()
    if bool(torch.isnan(z).any()) or bool((z == INF).any()) or bool((z == -INF).all()):
        return None
    # a masked logit weighs nothing at any temperature (-inf / inf would be NaN)
    e = torch.where(z == -INF, 0.0, torch.exp((z - z.max()) / t))
    return e / e.sum()


def _draw(w, u):
    mass = torch.cumsum(w, 0)
    i = int(torch.searchsorted(mass, u * mass[-1].item(), right=True))
    return min(i, int(torch.nonzero(w)[-1]))


def _clamped(u):
    return min(max(u, 0.0), 1.0 - 2.0 ** -53) if u == u else 0.0


def _reference(x, tokens, y, au, su, temperature):
    x, tokens = x.cpu(), tokens.cpu()
    y = None if y is None else y.cpu()
    b, rows, v = x.shape
    k = rows - 1
    heat = temperature.tolist() if isinstance(temperature, torch.Tensor) else [temperature] * b
    out = torch.full((b, k + 1), -1, dtype=torch.int64)
    logp = torch.zeros((b, k + 1), dtype=torch.float64)
    count = torch.zeros((b,), dtype=torch.int64)
    for s in range(b):
        t, j = heat[s], 0
        greedy = not t > 0
        while True:
            p = _distribution(x[s, j], 1.0 if greedy else t)
            d = int(tokens[s, j]) if j < k else -1
            drafted = 0 <= d < v
            if p is None:
                nxt = -1
                break
            if greedy:
                nxt = int((x[s, j] == x[s, j].max()).nonzero()[0])
                if not (drafted and nxt == d):
                    break
            else:
                u = _clamped(float(su[s]))
                q = None
                if drafted and y is None:
                    q = torch.zeros(v, dtype=torch.float64)
                    q[d] = 1.0
                elif drafted:
                    q = _distribution(y[s, j], t)
                if q is None:
                    nxt = _draw(p, u)
                    break
                if not _clamped(float(au[s, j])) * float(q[d]) < float(p[d]):
                    rest = (p - q).clamp(min=0.0)
                    nxt = _draw(rest if float(rest.sum()) > 0 else p, u)
                    break
            out[s, j], logp[s, j] = d, math.log(float(p[d]))
            j += 1
        count[s], out[s, j] = j, nxt
        if nxt >= 0:
            logp[s, j] = math.log(float(p[nxt])) if float(p[nxt]) > 0 else -INF
    return out, count, logp


def _run(x, tokens, y, au, su, temperature=1.0):
    import nmce
    t = temperature.to(DEV) if isinstance(temperature, torch.Tensor) else temperature
    return nmce.vocab_parallel_verify_drafts(
        x.to(DEV), tokens.to(DEV), None if y is None else y.to(DEV), au.to(DEV), su.to(DEV), 0,
        x.shape[-1], nmce.ParallelContext.single(), temperature=t)


def _check(x, tokens, y, au, su, temperature=1.0):
    got = _run(x, tokens, y, au, su, temperature)
    want = _reference(x, tokens, y, au, su, temperature)
    assert torch.equal(got[1].cpu(), want[1])
    assert torch.equal(got[0].cpu(), want[0])
    err = (got[2].double().cpu() - want[2]).abs()
    assert bool((err <= want[2].abs() * 2.0 ** -24 + 1e-7).all())
    return want


def _inputs(b, k, v, dtype, g, spread=2.0):
    x = torch.randn(b, k + 1, v, generator=g) * spread
    y = x[:, :k] + torch.randn(b, k, v, generator=g) * 0.5
    x, y = x.to(dtype), y.to(dtype)
    noise = torch.empty(b, k, v).exponential_(generator=g)
    tokens = (torch.softmax(y.float(), -1) / noise).argmax(-1) if k else torch.zeros(
        b, 0, dtype=torch.int64)
    return x, tokens, y, torch.rand(b, k, generator=g), torch.rand(b, generator=g)


@pytest.mark.parametrize("drafts", ["model", "copied"])
@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("b,k,v", [(1, 0, 1), (1, 1, 1), (3, 2, 2), (40, 3, 7), (5, 0, 1000),
                                   (9, 4, 1001), (4, 2, 8191), (4, 2, 8192), (4, 2, 8193),
                                   (3, 16, 300), (3, 15, 300), (2, 40, 50), (6, 5, 50257),
                                   (2, 3, 128256), (1, 1, 300001)])
def test_against_the_definition(b, k, v, dtype, drafts):
    g = torch.Generator().manual_seed(b + 10 * k + v)
    x, tokens, y, au, su = _inputs(b, k, v, dtype, g)
    if drafts == "copied":
        y = None
    heat = torch.tensor([0.0, 0.3, 1.0, 4.0])[torch.arange(b) % 4]
    for temperature in (1.0, 0.0, 0.7, heat):
        _check(x, tokens, y, au, su, temperature)


def test_long_drafts_that_all_stand():
    """More positions than are decided at once; equal models accept everything,
    greedy too."""
    g = torch.Generator().manual_seed(1)
    x, _, _, au, su = _inputs(3, 40, 100, F32, g)
    y = x[:, :40].clone()
    tokens = y.argmax(-1)
    for t in (1.0, 0.0):
        want = _check(x, tokens, y, au, su, t)
        assert want[1].tolist() == [40, 40, 40]
    tokens[1, 33] = (tokens[1, 33] + 1) % 100
    tokens[2, 16] = -1
    want = _check(x, tokens, y, au, su, 0.0)
    assert want[1].tolist() == [40, 33, 16]


def test_first_token_has_the_targets_distribution():
    """What verification is for: whatever the draft model, the first token out is
    distributed as p. 65536 sequences of one row pair; each id's count within 6
    standard deviations of a binomial's."""
    g = torch.Generator().manual_seed(2)
    n, v = 65536, 6
    x = torch.randn(1, 2, v, generator=g).expand(n, 2, v)
    y = torch.randn(1, 1, v, generator=g).expand(n, 1, v)
    for t in (1.0, 0.5):
        p = torch.softmax(x[0, 0].double() / t, -1)
        q = torch.softmax(y[0, 0].double() / t, -1)
        tokens = torch.multinomial(q, n, replacement=True, generator=g)[:, None]
        out, _, _ = _run(x, tokens, y, torch.rand(n, 1, generator=g), torch.rand(n, generator=g),
                         t)
        counts = torch.bincount(out[:, 0].cpu(), minlength=v).double()
        assert bool(((counts - n * p).abs() <= 6 * (n * p * (1 - p)).sqrt()).all())


def test_padded_drafts_and_ids_outside():
    g = torch.Generator().manual_seed(3)
    x, tokens, y, au, su = _inputs(8, 3, 500, BF, g)
    tokens[0, 0], tokens[1, 1], tokens[2, 2] = -1, -1, -1
    tokens[3, 0], tokens[4, 1], tokens[5, 0] = 500, 1 << 40, -(1 << 63)
    au[:] = 0.0
    for draft in (y, None):
        for t in (1.0, 0.0):
            _check(x, tokens, draft, au, su, t)
    assert _run(x, tokens, y, au, su)[1].tolist() == [0, 1, 2, 0, 1, 0, 3, 3]


@pytest.mark.parametrize("dtype", [F32, BF])
def test_masked_empty_and_broken_rows(dtype):
    """Logits of -inf, of the type's lowest value, rows of nothing but -inf,
    infinities and NaN, in the target's and in the draft's rows."""
    g = torch.Generator().manual_seed(4)
    v = 9000
    x, tokens, y, au, su = _inputs(24, 2, v, dtype, g)
    au[:] = 0.25
    low = torch.finfo(dtype).min
    for t in (x, y):
        t[0, 0, ::2] = -INF
        t[1, :, 100:] = -INF          # a whole slab masked
        t[2, :, :8500] = -INF         # and the other
        t[3, 0] = -INF
        t[3, 0, 8999] = 3.0           # one left
        t[4, 0] = low                 # all equal
        t[5, 0, 1:] = low
    x[6, 0], x[7, 1] = -INF, -INF
    x[8, 0, 17], x[9, 0, 8998] = INF, NAN
    x[10, 0], x[11, 2] = NAN, -INF
    y[12, 0], y[13, 1] = -INF, NAN
    y[14, 0, 5], y[15, 0, 8999] = INF, NAN
    x[16, 0, int(tokens[16, 0])] = -INF      # the target rules the draft out
    x[17, 0, int(tokens[17, 0])] = low
    y[18, 0, int(tokens[18, 0])] = -INF      # not the draft's own, yet the target's
    for s in (19, 20):                       # neither's: p = q without it
        x[s, 0, int(tokens[s, 0])] = -INF
        y[s, 0] = x[s, 0]
    x[21, 0, 0] = torch.finfo(dtype).max     # exp of everything else is 0
    x[22, 0] = torch.finfo(dtype).max
    heat = torch.tensor([1.0, 0.5])[torch.arange(24) % 2]
    odd = torch.tensor([NAN, -1.0, INF, 2.0 ** -149])[torch.arange(24) % 4]
    for draft in (y, None):
        for t in (1.0, 0.0, heat, 1e-30, INF, odd):
            _check(x, tokens, draft, au, su, t)


def test_ties_go_to_the_lowest_id():
    x = torch.zeros(3, 2, 20000)
    x[0, 0, [19999, 9000, 8192]] = 5.0
    x[1, 0, [300, 299, 8191]] = 5.0
    x[2, 0, 0], x[2, 0, 1] = 0.0, -0.0
    tokens = torch.tensor([[8192], [300], [0]])
    u = torch.zeros(3, 1), torch.zeros(3)
    out, n, _ = _run(x, tokens, None, *u, 0.0)
    assert n.tolist() == [1, 0, 1]
    assert out.tolist() == [[8192, 0], [299, -1], [0, 0]]


def test_uniform_numbers_at_the_ends():
    g = torch.Generator().manual_seed(5)
    ends = torch.tensor([0.0, 1.0 - 2.0 ** -24, 1.0, 2.0, -1.0, NAN, INF, 2.0 ** -149])
    x, tokens, y, au, _ = _inputs(8, 2, 10000, F32, g)
    x[:, :, :3], x[:, :, 9990:] = -INF, -INF   # the first and the last id are masked
    for draft in (y, None):
        _check(x, tokens, draft, ends[:, None].expand(8, 2).contiguous(), ends)
        _check(x, tokens, draft, au, ends.flip(0))
    # u = 0 is the first id with any weight, the largest u the last
    out, _, _ = _run(x[:, :1], tokens[:, :0], None, au[:, :0], ends)
    assert out[0, 0] == 3 and out[2, 0] == 9989 and out[5, 0] == 3


@pytest.mark.parametrize("dtype", [F32, BF])
def test_strides(dtype):
    """Rows that start anywhere, transposed and expanded batches, ids and numbers
    that are not contiguous, a vocabulary that is not (copied)."""
    g = torch.Generator().manual_seed(6)
    b, k, v = 4, 3, 1003
    x, tokens, y, au, su = _inputs(b, k, v, dtype, g)
    want = _reference(x, tokens, y, au, su, 1.0)
    wide = torch.zeros(b, k + 3, v + 5, dtype=dtype, device=DEV)
    wide[:, 1:k + 2, 3:v + 3] = x.to(DEV)
    turned = y.transpose(0, 1).contiguous().to(DEV).transpose(0, 1)
    import nmce

    def run(x, y, tokens=tokens.to(DEV), au=au.to(DEV), su=su.to(DEV)):
        return nmce.vocab_parallel_verify_drafts(x, tokens, y, au, su, 0, v,
                                                 nmce.ParallelContext.single())[0].cpu()

    views = [wide[:, 1:k + 2, 3:v + 3], x.transpose(1, 2).contiguous().to(DEV).transpose(1, 2)]
    for xv in views:
        assert torch.equal(run(xv, turned), want[0])
    pair = torch.stack([tokens, tokens], -1).to(DEV)[..., 0]
    au2, su2 = au.t().contiguous().to(DEV).t(), torch.stack([su, su], -1).to(DEV)[:, 0]
    assert torch.equal(run(views[0], turned, pair, au2, su2), want[0])
    one = x[:1].to(DEV).expand(b, k + 1, v)
    ref = _reference(x[:1].expand(b, k + 1, v), tokens, y, au, su, 1.0)
    assert torch.equal(run(one, turned), ref[0])


def test_rows_past_32_bits():
    """Two sequences 2^31 elements apart."""
    import nmce
    g = torch.Generator().manual_seed(7)
    v = 5000
    x, tokens, _, au, su = _inputs(2, 1, v, BF, g)
    buf = torch.empty((1 << 31) + 2 * v + 1, dtype=BF, device=DEV)
    far = buf.as_strided((2, 2, v), ((1 << 31) + 1, v, 1))
    far.copy_(x)
    got = nmce.vocab_parallel_verify_drafts(far, tokens.to(DEV), None, au.to(DEV), su.to(DEV), 0,
                                            v, nmce.ParallelContext.single())
    want = _reference(x, tokens, None, au, su, 1.0)
    assert torch.equal(got[0].cpu(), want[0])


def test_guard_bytes():
    from nmce import _lib as L
    import ctypes
    lib = L.load()
    g = torch.Generator().manual_seed(8)
    for b, k, v in ((1, 0, 1), (3, 2, 9000), (5, 17, 40)):
        x, tokens, y, au, su = (t.to(DEV) for t in _inputs(b, k, v, F32, g))
        n, slabs = b * (2 * k + 1), lib.nmce_verify_slabs(v)

        def guarded(count, dtype):
            t = torch.full((count + 64,), 77, dtype=dtype, device=DEV)
            return t, t[32:].data_ptr()

        st, st_p = guarded(n * slabs * 4, torch.float64)
        ma, ma_p = guarded(b * slabs * 2, torch.float64)
        tk, tk_p = guarded(b * (k + 1), torch.int64)
        ac, ac_p = guarded(b, torch.int64)
        lp, lp_p = guarded(b * (k + 1), torch.float32)
        need = lib.nmce_verify_workspace_bytes(b)
        ws, ws_p = guarded(need, torch.uint8)
        batch = L.VerifyBatch(x.data_ptr(), y.data_ptr() if k else None, tokens.data_ptr(),
                              au.data_ptr(), su.data_ptr(), None, x.stride(0), x.stride(1),
                              y.stride(0), y.stride(1), b, k, v, 0, v, 1.0, L.NMCE_F32)
        s = L.stream_handle(torch.device(DEV))
        p = ctypes.addressof(batch)
        L.check(lib.nmce_verify_stats(p, st_p, s), "stats")
        L.check(lib.nmce_verify_masses(p, st_p, 1, ma_p, tk_p, ac_p, lp_p, ws_p, need, s), "masses")
        L.check(lib.nmce_verify_pick(p, ma_p, 1, 0, ws_p, need, tk_p, lp_p, None, s), "pick")
        torch.cuda.synchronize()
        for t in (st, ma, tk, ac, lp, ws):
            assert bool((t[:32] == 77).all()) and bool((t[-32:] == 77).all())
        want = _reference(x, tokens, y if k else None, au, su, 1.0)
        assert torch.equal(tk[32:-32].cpu().view(b, k + 1), want[0])


def test_no_sequences_and_streams():
    import nmce
    ctx = nmce.ParallelContext.single()
    e = torch.zeros(0, 3, 10, device=DEV)
    out, n, lp = nmce.vocab_parallel_verify_drafts(
        e, torch.zeros(0, 2, dtype=torch.int64, device=DEV), None, torch.zeros(0, 2, device=DEV),
        torch.zeros(0, device=DEV), 0, 10, ctx)
    assert out.shape == (0, 3) and n.shape == (0,) and lp.shape == (0, 3)
    g = torch.Generator().manual_seed(9)
    jobs = [tuple(t.to(DEV) for t in _inputs(6, 3, 9001, BF, g)) for _ in range(2)]
    want = [_run(*j) for j in jobs]
    torch.cuda.synchronize()
    got = []
    for job in jobs:
        with torch.cuda.stream(torch.cuda.Stream()):
            got.append(_run(*job))
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_graph_replays():
    g = torch.Generator().manual_seed(10)
    x, tokens, y, au, su = (t.to(DEV) for t in _inputs(5, 3, 9001, BF, g))
    heat = torch.ones(5, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _run(x, tokens, y, au, su, heat)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _run(x, tokens, y, au, su, heat)
    for rep in range(3):
        for dst, src in zip((x, tokens, y, au, su), _inputs(5, 3, 9001, BF, g)):
            dst.copy_(src)
        heat[rep] = 0.0
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        want = _run(x, tokens, y, au, su, heat)
        assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_verify_refusals():
    import nmce
    ctx = nmce.ParallelContext.single()
    g = torch.Generator().manual_seed(11)
    x, tokens, y, au, su = (t.to(DEV) for t in _inputs(2, 3, 50, F32, g))

    def call(x=x, tokens=tokens, y=y, au=au, su=su, start=0, end=50, t=1.0):
        return nmce.vocab_parallel_verify_drafts(x, tokens, y, au, su, start, end, ctx,
                                                 temperature=t)

    call()
    for kwargs, error in ((dict(x=x.half()), TypeError), (dict(y=y.to(BF)), TypeError),
                          (dict(tokens=tokens.int()), TypeError), (dict(au=au.double()), TypeError),
                          (dict(su=su.to(BF)), TypeError), (dict(x=x[0]), ValueError),
                          (dict(x=x[:, :0]), ValueError), (dict(x=x[..., :0], end=0), ValueError),
                          (dict(x=x[:, :3]), ValueError), (dict(y=y[..., :49]), ValueError),
                          (dict(tokens=tokens[:1]), ValueError), (dict(su=su[:1]), ValueError),
                          (dict(end=51), ValueError), (dict(start=50, end=100), ValueError),
                          (dict(start=-50, end=0), ValueError), (dict(t=-0.5), ValueError),
                          (dict(t=NAN), ValueError),
                          (dict(t=torch.ones(3, device=DEV)), ValueError),
                          (dict(t=torch.ones(2, dtype=torch.float64, device=DEV)), TypeError),
                          (dict(t=torch.ones(2)), RuntimeError), (dict(su=su.cpu()), RuntimeError),
                          (dict(y=y.cpu()), RuntimeError),
                          (dict(x=x.clone().requires_grad_(True)), RuntimeError),
                          (dict(y=y.clone().requires_grad_(True)), RuntimeError)):
        with pytest.raises(error, match="nmce|unsupported"):
            call(**kwargs)


@pytest.mark.parametrize("v", [1000, 50257])
def test_a_serving_step(v):
    """The operators as a decoding step uses them: ids to rows, rows to logits with
    the 8-bit head, logits to tokens; greedy verification of the head's own
    choices accepts all of them, and the step can run on its own output."""
    import nmce
    ctx = nmce.ParallelContext.single()
    cfg = types.SimpleNamespace(vocab_size=v, n_embd=96, sequence_parallel=False)
    torch.manual_seed(0)
    emb = nmce.VocabParallelEmbedding(cfg, ctx, scale=96 ** 0.5).to(DEV)
    head = nmce.FusedParallelLMHead(cfg, ctx).to(DEV).quantized()
    g = torch.Generator().manual_seed(1)
    last = torch.randint(0, v, (5, 1), generator=g).to(DEV)
    with torch.no_grad():
        drafts = []
        for _ in range(3):  # a draft "model" that is the model itself
            drafts.append(head(emb((drafts or [last])[-1], out_dtype=BF)).argmax(-1))
        tokens = torch.cat(drafts, 1)
        logits = head(emb(torch.cat([last, tokens], 1), out_dtype=BF))
        u = torch.rand(5, 3, generator=g).to(DEV), torch.rand(5, generator=g).to(DEV)
        out, n, _ = nmce.vocab_parallel_verify_drafts(logits, tokens, None, *u, 0, v, ctx,
                                                      temperature=0.0)
        assert n.tolist() == [3] * 5 and torch.equal(out[:, :3], tokens)
        assert torch.equal(out[:, 3], logits[:, 3].argmax(-1))
        out, n, lp = nmce.vocab_parallel_verify_drafts(logits, tokens, None, *u, 0, v, ctx)
    want = _reference(logits, tokens, None, u[0], u[1], 1.0)
    assert torch.equal(out.cpu(), want[0]) and torch.equal(n.cpu(), want[1])


def test_tensors_that_want_a_derivative_are_refused():
    """The log-probabilities have none, in either mode: none is dropped in silence."""
    from torch.autograd import forward_ad
    g = torch.Generator().manual_seed(14)
    x, tokens, y, au, su = (t.to(DEV) for t in _inputs(2, 3, 50, F32, g))
    heat = torch.ones(2, device=DEV)
    for i, name in enumerate(("target_logits", "draft_logits", "temperature")):
        args = [x, y, heat]
        args[i] = args[i].clone().requires_grad_(True)
        with pytest.raises(RuntimeError, match=f"nmce: {name} requires grad"):
            _run(args[0], tokens, args[1], au, su, args[2])
        with forward_ad.dual_level(), torch.no_grad():
            args[i] = forward_ad.make_dual(args[i].detach(), torch.ones_like(args[i]))
            with pytest.raises(RuntimeError, match=f"nmce: {name} has a forward-mode tangent"):
                _run(args[0], tokens, args[1], au, su, args[2])


def test_a_number_as_temperature_keeps_its_bits():
    """A Python number's temperature is 64 bits wide like the rest: uniform numbers
    that lie between a border of p at 0.7 and the same border at fp32's 0.7, where the
    two give neighbouring ids (each at least 1e-11 from both, 100 times what the
    sums' rounding moves a border)."""
    import nmce
    g = torch.Generator().manual_seed(15)
    v = 20000
    x = torch.randn(v, generator=g) * 2.0
    t = 0.7
    near = torch.tensor(t, dtype=F32).double().item()
    a, b = (torch.cumsum(torch.softmax(x.double() / s, -1), 0) for s in (t, near))
    lo, hi = torch.minimum(a, b), torch.maximum(a, b)
    u = ((lo + hi) / 2).float()
    inside = (u.double() > lo + 1e-11) & (u.double() < hi - 1e-11)
    u = u[inside]
    assert u.numel() > 200
    want, other = (torch.searchsorted(c, u.double(), right=True) for c in (a, b))
    assert bool((want != other).all())
    n = u.numel()

    def draw(temperature):
        return nmce.vocab_parallel_verify_drafts(
            x.to(DEV).expand(n, 1, v), torch.zeros(n, 0, dtype=torch.int64, device=DEV), None,
            torch.zeros(n, 0, device=DEV), u.to(DEV), 0, v, nmce.ParallelContext.single(),
            temperature=temperature)[0][:, 0].cpu()

    assert torch.equal(draw(t), want)
    assert torch.equal(draw(torch.full((n,), t, device=DEV)), other)  # fp32 as given


def test_temperatures_outside_of_fp32():
    """Numbers that fp32 would take for 0 or infinity: above 0 is not greedy (equal
    largest logits share), and the largest only levels."""
    g = torch.Generator().manual_seed(16)
    x, tokens, y, au, su = _inputs(6, 2, 9000, F32, g)
    x[0, 0, [3, 8999]] = 40.0
    x[1, :, 7] = x[1, :, 8500] = 50.0
    x[2, 0, 1:] = -INF
    for draft in (y, None):
        for t in (5e-324, 1e-300, 1e-60, 1e39, 1e300):
            _check(x, tokens, draft, au, su, t)


def _stops(b, k, v, g):
    """Drafts that stand up to a place of each sequence's own: any of the ends of the
    rounds in which positions are decided (16 or 64 at a time), or all of them."""
    x = torch.randn(b, k + 1, v, generator=g) * 2.0
    y = x[:, :k].clone()
    tokens = y.argmax(-1)
    su = torch.rand(b, generator=g)
    places = [p for p in (0, 1, 14, 15, 16, 17, 31, 32, 33, 62, 63, 64, 65, 127, 128, 129, k - 1, k)
              if p <= k]
    at = torch.tensor(places)[torch.randint(0, len(places), (b,), generator=g)]
    for s in range(min(b, len(places))):
        at[s] = places[s]
    return x, tokens, y, su, at


@pytest.mark.parametrize("b,k", [(30, 63), (30, 64), (30, 65), (20, 130), (18, 200),   # 1024 threads
                                 (300, 15), (300, 16), (300, 17), (300, 33), (260, 70)])  # 256
def test_decisions_in_several_rounds(b, k):
    """More drafts than positions are decided at once, in workgroups of 1024 threads
    (64 of them) and, from 257 workgroups on, of 256 (16): stops at the ends of the
    rounds and on both sides, refused by their number, by greedy choice, or padding."""
    v = 60
    g = torch.Generator().manual_seed(b + k)
    x, tokens, y, su, at = _stops(b, k, v, g)
    every = torch.arange(b)
    stop = at < k
    au = torch.zeros(b, k)
    # Copied drafts: u = 0 stands, and the largest number below 1 is not below p.
    refused = au.clone()
    refused[every[stop], at[stop]] = 1.0 - 2.0 ** -24
    assert _check(x, tokens, None, refused, su)[1].tolist() == at.tolist()
    padded = tokens.clone()
    padded[every[stop], at[stop]] = -1
    for draft in (y, None):
        assert _check(x, padded, draft, au, su)[1].tolist() == at.tolist()
        assert _check(x, padded, draft, au, su, 0.0)[1].tolist() == at.tolist()
    other = tokens.clone()
    other[every[stop], at[stop]] = (other[every[stop], at[stop]] + 1) % v
    assert _check(x, other, y, au, su, 0.0)[1].tolist() == at.tolist()
    ruled = x.clone()  # the target rules the draft out; the draft model is sure of it
    ruled[every[stop], at[stop], tokens[every[stop], at[stop]]] = -INF
    assert _check(ruled, tokens, y, au, su)[1].tolist() == at.tolist()


@pytest.mark.parametrize("drafts", ["model", "copied"])
@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("b,k,v", [(32, 2, 65536), (33, 2, 65536),   # 256 and 264 slabs' masses
                                   (40, 5, 60001), (257, 0, 9000),
                                   (256, 1, 9001), (257, 1, 9001)])  # sequences that draw
def test_both_workgroup_sizes(b, k, v, dtype, drafts):
    """Both sides of the change from 1024 threads a workgroup to 256, in the masses
    and in the draw, over several slabs: whole tokens, counts and log-probabilities."""
    g = torch.Generator().manual_seed(b + k + v)
    x, tokens, y, au, su = _inputs(b, k, v, dtype, g)
    heat = torch.tensor([0.0, 0.3, 1.0, 4.0])[torch.arange(b) % 4]
    for temperature in (heat, 1.0):
        _check(x, tokens, None if drafts == "copied" else y, au, su, temperature)
