"""Penalties, biases and masks on logits against the definition in 64 bits, on the CPU.

An element that nothing touches comes back bit for bit, a masked one as -inf. A touched
one is the rounding of a 64-bit value (half a step of its type), whose own error is a
few 2^-53 of the largest value on the way to it (2^-50 of it is allowed)."""

from __future__ import annotations

import math
import types

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32
INF, NAN = float("inf"), float("nan")


def _each(value, s):
    return float(value[s]) if isinstance(value, torch.Tensor) else float(value)


def _reference(x, start=0, total=None, prompt=None, output=None, drafts=None, r=1.0, f=0.0, p=0.0,
               bias_ids=None, bias=None, allowed=None):
    """(value in 64 bits, largest value on the way to it, whether it is touched)."""
    b, rows, v = x.shape
    total = v if total is None else total
    z, most, touched = x.double().clone(), x.double().abs(), torch.zeros(x.shape, dtype=torch.bool)

    def local(ids):
        return [int(j) - start for j in ids.tolist() if start <= j < min(start + v, total)]

    for s in range(b):
        rr, ff, pp = _each(r, s), _each(f, s), _each(p, s)
        if not (rr > 0 and rr < INF):
            rr = 1.0
        seen = local(prompt[s]) if prompt is not None else []
        for i in range(rows):
            made = (local(output[s]) if output is not None else []) + \
                (local(drafts[s, :i]) if drafts is not None else [])
            times = {}
            for j in made:
                times[j] = times.get(j, 0) + 1
            row = z[s, i]

            def change(j, value):
                row[j] = value
                touched[s, i, j] = True
                if abs(value) < INF:
                    most[s, i, j] = max(float(most[s, i, j]), abs(value))

            if rr != 1.0:
                for j in set(seen) | set(times):
                    old = float(row[j])
                    change(j, old / rr if old > 0 else old * rr)
            if ff != 0.0 or pp != 0.0:
                for j, n in times.items():
                    most[s, i, j] = max(float(most[s, i, j]), abs(ff * n) + abs(pp))
                    change(j, float(row[j]) - ff * n - pp)
            if bias_ids is not None:
                for j, value in zip(bias_ids[s].tolist(), bias[s].tolist()):
                    if start <= j < min(start + v, total):
                        change(j - start, float(row[j - start]) + value)
            if allowed is not None:
                g = torch.arange(start, start + v)
                keep = (allowed[s, i].long()[g // 32] >> (g % 32)) & 1
                row[keep == 0] = -INF
                touched[s, i][keep == 0] = True
    return z, most, touched


NAMES = {"prompt": "prompt_tokens", "output": "output_tokens", "drafts": "draft_tokens",
         "r": "repetition_penalty", "f": "frequency_penalty", "p": "presence_penalty",
         "bias_ids": "bias_ids", "bias": "bias_values", "allowed": "allowed"}


def _run(x, inplace=False, start=0, total=None, ctx=None, **kw):
    import nmce
    if ctx is None:
        ctx = nmce.ParallelContext.single()
    args = {NAMES[k]: t.to(DEV) if isinstance(t, torch.Tensor) else t for k, t in kw.items()}
    return nmce.vocab_parallel_adjust_logits(x, start, start + x.shape[-1], ctx, inplace=inplace,
                                             **args)


def _compare(got, x, want):
    z, most, touched = want
    got = got.cpu()
    same = ~touched
    assert torch.equal(got[same].view(torch.int32 if x.dtype == F32 else torch.int16),
                       x[same].view(torch.int32 if x.dtype == F32 else torch.int16))
    y, z, most = got[touched].double(), z[touched], most[touched]
    # Half a step past the type's largest value and beyond rounds to infinity: 1.5 times
    # the lowest one, for instance.
    info = torch.finfo(x.dtype)
    z = torch.where(z.abs() >= info.max * (1 + info.eps / 4), torch.copysign(
        torch.tensor(INF, dtype=torch.float64), z), z)
    odd = ~torch.isfinite(z)
    assert torch.equal(torch.isnan(y), torch.isnan(z))
    assert torch.equal(y[odd & ~torch.isnan(z)], z[odd & ~torch.isnan(z)])
    y, z, most = y[~odd], z[~odd], most[~odd]
    bound = info.eps / 2 * z.abs() + 2.0 ** -50 * most + info.smallest_normal * info.eps
    assert bool(((y - z).abs() <= bound).all()), float(((y - z).abs() - bound).max())


def _check(x, **kw):
    want = _reference(x, **kw)
    d = x.to(DEV)
    got = _run(d, **kw)
    assert got.data_ptr() != d.data_ptr() and torch.equal(
        d.cpu().view(torch.uint8), x.view(torch.uint8))
    _compare(got, x, want)
    assert _run(d, inplace=True, **kw) is d
    assert torch.equal(d.view(torch.uint8), got.view(torch.uint8))
    return want


def _ids(b, n, v, g, padded=True):
    ids = (torch.exp(torch.rand(b, n, generator=g) * math.log(v + 1)) - 1).long().clamp(0, v - 1)
    if padded and n > 1:
        ids[torch.rand(b, n, generator=g) < 0.1] = -1
    return ids


def _inputs(b, k, v, dtype, g, prompt=50, output=20, bias=0, mask=False):
    kw = dict(prompt=_ids(b, prompt, v, g), output=_ids(b, output, v, g),
              r=1.0 + torch.rand(b, generator=g), f=torch.rand(b, generator=g) - 0.3,
              p=torch.rand(b, generator=g) - 0.3)
    if k:
        kw["drafts"] = _ids(b, k, v, g)
    if bias:
        kw["bias_ids"], kw["bias"] = _ids(b, bias, v, g), torch.randn(b, bias, generator=g) * 4
    if mask:
        kw["allowed"] = torch.randint(-2 ** 31, 2 ** 31, (b, k + 1, -(-v // 32)), generator=g,
                                      dtype=torch.int64).to(torch.int32)
    return (torch.randn(b, k + 1, v, generator=g) * 4).to(dtype), kw


@pytest.mark.parametrize("mask", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("b,k,v,prompt,output,bias", [
    (1, 0, 1, 1, 1, 1), (2, 1, 2, 3, 3, 2), (3, 0, 31, 40, 0, 5), (3, 2, 33, 0, 40, 0),
    (5, 3, 1000, 100, 50, 9), (2, 0, 8191, 300, 100, 20), (2, 1, 8192, 300, 100, 20),
    (2, 2, 8193, 300, 100, 20), (40, 0, 50257, 30, 10, 4), (2, 8, 50257, 2000, 700, 64),
    (1, 0, 128256, 20000, 3000, 300), (2, 0, 256001, 100, 100, 3)])
def test_against_the_definition(b, k, v, prompt, output, bias, dtype, mask):
    g = torch.Generator().manual_seed(v + 7 * b + k)
    x, kw = _inputs(b, k, v, dtype, g, prompt, output, bias, mask)
    _check(x, **kw)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("inplace", [False, True])
def test_long_lists_of_several_rows(dtype, inplace):
    """Lists longer than a slab: a workgroup takes several rows, whose counts grow, with
    fewer and with more places than are listed, and biases on counted ids."""
    g = torch.Generator().manual_seed(20)
    b, k, v = 16, 5, 50257
    x, kw = _inputs(b, k, v, dtype, g, 9000, 400, 30, True)
    kw["bias_ids"][:, :10] = kw["prompt"][:, :10]
    kw["bias_ids"][:, 10:13] = kw["drafts"][:, :3]
    kw["prompt"][3:] %= 300  # few ids, often
    kw["prompt"][1] = torch.randperm(v, generator=g)[:9000]
    kw["drafts"][:, 1] = torch.arange(b) * 3100 + 11
    kw["drafts"][:, 3] = kw["drafts"][:, 1]
    want = _reference(x, **kw)
    _compare(_run(x.to(DEV), inplace, **kw), x, want)


@pytest.mark.parametrize("times", [16381, 16382, 16383, 16384, 70000])
def test_an_id_thousands_of_times(times):
    """At both sides of what a count of 16 bits holds, beside a neighbour that has none."""
    x = torch.randn(2, 2, 500)
    output = torch.full((2, times), 41)
    output[1, ::2] = 40
    kw = dict(prompt=torch.tensor([[41, 43], [42, 40]]), output=output, r=1.5, f=0.25, p=-0.5,
              drafts=torch.tensor([[41], [40]]), bias_ids=torch.tensor([[41, 42], [39, 40]]),
              bias=torch.randn(2, 2))
    _check(x, **kw)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_every_part_alone_and_numbers_for_tensors(dtype):
    g = torch.Generator().manual_seed(5)
    x, kw = _inputs(4, 2, 9001, dtype, g, 200, 90, 10, True)
    lists = {n: kw[n] for n in ("prompt", "output", "drafts")}
    _check(x, **lists)
    _check(x, **lists, r=1.3)
    _check(x, **lists, r=0.5)
    _check(x, **lists, f=0.25)
    _check(x, **lists, f=-2.0, p=1e-3)
    _check(x, drafts=kw["drafts"], p=-1.5)
    _check(x, drafts=kw["drafts"], prompt=kw["prompt"], r=2.0)
    _check(x, drafts=kw["drafts"], bias_ids=kw["bias_ids"], bias=kw["bias"])
    _check(x, drafts=kw["drafts"], allowed=kw["allowed"])
    _check(x[:, :1].contiguous(), allowed=kw["allowed"][:, :1])


@pytest.mark.parametrize("dtype", [F32, BF])
def test_an_id_that_comes_again(dtype):
    """In a list, in several lists, and several times with a bias."""
    g = torch.Generator().manual_seed(6)
    x = (torch.randn(2, 4, 500, generator=g) * 3).to(dtype)
    prompt = torch.tensor([[7, 7, 7, 499], [0, 0, 1, -1]])
    output = torch.tensor([[7, 8, 8, 8, 8], [499, 499, 0, 0, 0]])
    drafts = torch.tensor([[8, 8, 7], [3, 3, 3]])
    ids = torch.tensor([[7, 9, 7, 7, 9, -1], [0, 0, 0, 0, 0, 0]])
    bias = torch.tensor([[1e8, 2.0, -1e8, 1.0, 0.5, 9.0], [1.0, -2.0, 3.0, 0.1, 0.2, 0.3]])
    lists = dict(prompt=prompt, output=output, drafts=drafts, r=1.7, f=0.3, p=0.6)
    _check(x, **lists)
    _check(x, **lists, bias_ids=ids, bias=bias)
    # every id of a slab, many times each
    many = torch.arange(500).repeat(1, 40).expand(2, -1)
    _check(x, drafts=drafts, output=many, f=0.01, p=-1.0, r=1.1)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_rows_that_a_mask_empties_and_odd_values(dtype):
    g = torch.Generator().manual_seed(8)
    v = 8200
    x = (torch.randn(3, 2, v, generator=g) * 3).to(dtype)
    for j, value in ((0, NAN), (1, INF), (2, -INF), (3, 0.0), (4, -0.0),
                     (5, torch.finfo(dtype).min), (8199, NAN), (8198, INF)):
        x[:, :, j] = value
    words = -(-v // 32)
    allowed = torch.full((3, 2, words), -1, dtype=torch.int32)
    allowed[0] = 0  # nothing left
    allowed[1, 0] = 0
    allowed[1, 0, 100] = 1 << 5  # one id
    allowed[1, 1, ::2] = 0x0F0F00FF
    ids = torch.tensor([[0, 1, 2, 3, 4, 5, 8198, 8199, 3205]] * 3)
    drafts = torch.tensor([[3205], [-1], [8200]])
    bias = torch.tensor([[1.0, 2.0, INF, -INF, 0.5, -1.0, NAN, 1.0, -0.5]] * 3)
    _check(x, drafts=drafts, allowed=allowed)
    _check(x, drafts=drafts, allowed=allowed, prompt=ids, output=ids[:, :5], r=1.5, f=0.5, p=0.5)
    # (-inf + inf is NaN, as everywhere.)
    _check(x, drafts=drafts, allowed=allowed, bias_ids=ids, bias=bias)
    got = _run(x.to(DEV), drafts=drafts, allowed=allowed)
    assert bool((got[0] == -INF).all()) and int((got[1, 0] != -INF).sum()) == 1


def test_a_halfway_value_is_rounded_once():
    """1 + 2^-8 is halfway between two bf16 values; a little above it rounds up, which
    a rounding to fp32 on the way would hide."""
    x = torch.ones(1, 1, 64, dtype=BF)
    bias = torch.tensor([[2.0 ** -8 + 2.0 ** -40, 2.0 ** -8, 2.0 ** -8 - 2.0 ** -40,
                          3 * 2.0 ** -8, -(2.0 ** -9) - 2.0 ** -40]], dtype=torch.float32)
    # fp32 keeps 2^-8 + 2^-32 at most, so build the excess from two biases
    ids = torch.tensor([[0, 1, 2, 3, 4, 0, 2]])
    values = torch.tensor([[2.0 ** -8, 2.0 ** -8, 2.0 ** -8, 3 * 2.0 ** -8, -(2.0 ** -9),
                            2.0 ** -40, -(2.0 ** -40)]])
    del bias
    got = _run(x.to(DEV), bias_ids=ids, bias=values).cpu()[0, 0, :6].float().tolist()
    up = 1.0 + 2.0 ** -7
    assert got == [up, 1.0, 1.0, 1.0 + 4 * 2.0 ** -8, 1.0, 1.0]


@pytest.mark.parametrize("dtype", [F32, BF])
def test_penalties_that_are_no_penalties(dtype):
    g = torch.Generator().manual_seed(9)
    x, kw = _inputs(5, 1, 777, dtype, g)
    kw["r"] = torch.tensor([0.0, -1.0, INF, NAN, 2.0])
    _check(x, **kw)
    kw.update(r=torch.ones(5), f=torch.zeros(5), p=torch.zeros(5))
    _check(x, **kw)


def test_strides_and_padding():
    """Logits, lists and masks as parts of larger tensors, expanded, and transposed."""
    import nmce
    g = torch.Generator().manual_seed(10)
    b, k, v = 3, 2, 1003
    x, kw = _inputs(b, k, v, BF, g, 40, 20, 6, True)
    want = _reference(x, **kw)
    ctx = nmce.ParallelContext.single()

    def wide(t, more):
        big = torch.full(t.shape[:-1] + (t.shape[-1] + more,), 1, dtype=t.dtype)
        big[..., :t.shape[-1]] = t
        return big.to(DEV)[..., :t.shape[-1]]

    def call(logits, **other):
        args = {NAMES[n]: t.to(DEV) for n, t in kw.items()}
        args.update(other)
        return nmce.vocab_parallel_adjust_logits(logits, 0, v, ctx, **args)

    _compare(call(wide(x, 5)), x, want)
    _compare(call(wide(x, 13), prompt_tokens=wide(kw["prompt"], 9),
                  output_tokens=wide(kw["output"], 1), draft_tokens=wide(kw["drafts"], 3),
                  bias_ids=wide(kw["bias_ids"], 2), bias_values=wide(kw["bias"], 4),
                  allowed=wide(kw["allowed"], 3)), x, want)
    back = x.to(DEV).transpose(0, 1).contiguous().transpose(0, 1)
    _compare(call(back), x, want)
    _compare(call(x.to(DEV).transpose(1, 2).contiguous().transpose(1, 2)), x, want)
    _compare(call(x.to(DEV), prompt_tokens=kw["prompt"].to(DEV).t().contiguous().t()), x, want)
    # in place, the elements between the rows stay
    big = torch.full((b, k + 1, v + 5), 7.0, dtype=BF, device=DEV)
    big[..., :v] = x.to(DEV)
    args = {NAMES[n]: t.to(DEV) for n, t in kw.items()}
    before = big._version
    nmce.vocab_parallel_adjust_logits(big[..., :v], 0, v, ctx, inplace=True, **args)
    _compare(big[..., :v], x, want)
    assert bool((big[..., v:] == 7.0).all()) and big._version > before
    # one mask for every row
    kw["allowed"] = kw["allowed"][:, :1].expand(-1, k + 1, -1)
    want = _reference(x, **kw)
    _compare(call(x.to(DEV), allowed=kw["allowed"][:, :1].to(DEV).expand(-1, k + 1, -1)), x, want)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("tp,per", [(2, 1001), (3, 33), (4, 8000)])
def test_shards_are_columns_of_the_whole(tp, per, dtype):
    import nmce
    g = torch.Generator().manual_seed(tp)
    x, kw = _inputs(3, 2, tp * per, dtype, g, 300, 60, 20, True)
    whole = _run(x.to(DEV), **kw)
    _compare(whole, x, _reference(x, **kw))
    for rank in range(tp):
        ctx = types.SimpleNamespace(tp_size=tp, tp_rank=rank, tp_group=None)
        mine = slice(rank * per, (rank + 1) * per)
        for inplace in (False, True):
            got = _run(x[..., mine].contiguous().to(DEV), inplace, rank * per, ctx=ctx, **kw)
            assert torch.equal(got, whole[..., mine])


def test_ids_outside_and_empty_batches():
    g = torch.Generator().manual_seed(12)
    x = torch.randn(2, 2, 100, generator=g)
    odd = torch.tensor([[-1, 100, 2 ** 62, -2 ** 62, 2 ** 32 + 5, 50],
                        [2 ** 31, -2 ** 31, 99, 0, -7, 100]])
    _check(x, prompt=odd, output=odd, drafts=odd[:, 1:2], r=1.5, f=0.5, p=0.25, bias_ids=odd,
           bias=torch.ones(2, 6))
    empty = _run(torch.empty(0, 3, 100, device=DEV), drafts=torch.empty(0, 2, dtype=torch.int64))
    assert empty.shape == (0, 3, 100)
    _check(x[:, :1].contiguous(), prompt=torch.empty(2, 0, dtype=torch.int64),
           output=torch.empty(2, 0, dtype=torch.int64), drafts=torch.empty(2, 0, dtype=torch.int64),
           bias_ids=torch.empty(2, 0, dtype=torch.int64), bias=torch.empty(2, 0), r=2.0)


def test_as_many_biases_as_are_taken():
    g = torch.Generator().manual_seed(13)
    n = 8192
    x = torch.randn(1, 1, 20000, generator=g)
    ids = torch.randperm(20000, generator=g)[None, :n].clone()
    _check(x, bias_ids=ids, bias=torch.randn(1, n, generator=g))
    ids[0, ::2] = 17  # half of them one id's
    _check(x, bias_ids=ids, bias=torch.randn(1, n, generator=g))


def test_another_stream_and_inference_mode():
    g = torch.Generator().manual_seed(14)
    x, kw = _inputs(4, 1, 30000, BF, g, mask=True)
    want = _reference(x, **kw)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = _run(x.to(DEV), **kw)
    side.synchronize()
    _compare(got, x, want)
    with torch.inference_mode():
        d = x.to(DEV)
        _compare(_run(d, **kw), x, want)
        _compare(_run(d, inplace=True, **kw), x, want)


def test_captured_and_replayed():
    """A decoding step's call in a graph, replayed with other logits and lists."""
    import nmce
    g = torch.Generator().manual_seed(15)
    ctx = nmce.ParallelContext.single()
    v = 20000
    x, kw = _inputs(3, 1, v, F32, g, 64, 32, 4, True)
    logits = x.to(DEV)
    args = {NAMES[n]: t.to(DEV) for n, t in kw.items()}
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        nmce.vocab_parallel_adjust_logits(logits, 0, v, ctx, **args)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = nmce.vocab_parallel_adjust_logits(logits, 0, v, ctx, **args)
    for _ in range(3):
        x, kw = _inputs(3, 1, v, F32, g, 64, 32, 4, True)
        logits.copy_(x)
        for n, t in kw.items():
            args[NAMES[n]].copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        _compare(out, x, _reference(x, **kw))
        assert torch.equal(nmce.vocab_parallel_adjust_logits(logits, 0, v, ctx, **args), out)


def test_refusals_on_the_device():
    import nmce
    ctx = nmce.ParallelContext.single()
    x = torch.randn(2, 1, 50, device=DEV)
    ids = torch.zeros(2, 3, dtype=torch.int64, device=DEV)

    def call(logits=x, **kw):
        return nmce.vocab_parallel_adjust_logits(logits, 0, 50, ctx, **kw)

    with pytest.raises(RuntimeError, match="requires grad"):
        call(x.clone().requires_grad_(True))
    with pytest.raises(RuntimeError, match="requires grad"):
        call(bias_ids=ids, bias_values=torch.zeros(2, 3, device=DEV, requires_grad=True))
    with pytest.raises(RuntimeError, match="requires grad"):
        call(presence_penalty=torch.zeros(2, device=DEV, requires_grad=True))
    with torch.no_grad():
        call(x.clone().requires_grad_(True))
    with pytest.raises(ValueError, match="overlap"):
        call(x[:1].expand(2, 1, 50), inplace=True)
    with pytest.raises(ValueError, match="overlap"):
        call(torch.as_strided(x, (2, 1, 50), (20, 50, 1)), inplace=True)
    with pytest.raises(ValueError, match="contiguous vocabulary"):
        call(torch.as_strided(x, (2, 1, 50), (50, 50, 2), 0) if x.numel() > 150 else
             torch.randn(2, 50, 2, device=DEV)[..., 0].unsqueeze(1), inplace=True)
    with pytest.raises(RuntimeError, match="prompt_tokens on"):
        call(prompt_tokens=ids.cpu())
