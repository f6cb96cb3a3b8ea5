"""8-bit rows and their product against 64-bit arithmetic.

The integers are exact: q must equal the 64-bit quotient's rounding (halves to
even), and the integer sums have no error. The product then rounds four times in
fp32 (the sum's conversion, the token's scale, two products) and once to the output:
(4 2^-24 + half a step of the output) relative, the fp32 scale of q by half a step.
"""

from __future__ import annotations

import types

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32
HALF_STEP = {F32: 2.0 ** -24, BF: 2.0 ** -8}


def _quotients(x):
    """(q int64, scale) in 64 bits on the CPU; rows are finite."""
    wide = x.double().cpu()
    top = wide.abs().amax(-1, keepdim=True)
    q = torch.round(127.0 * wide / torch.where(top > 0, top, torch.ones_like(top)))
    return q.long(), top.squeeze(-1) / 127.0


def _rows(n, k, dtype, g, how):
    x = torch.randn(n, k, generator=g)
    if how == "halves":  # multiples of a 254th of the largest: every odd one is a half
        x = torch.randint(-254, 255, (n, k), generator=g).float()
        x[:, 0] = 254.0
        x = x * 2.0 ** torch.randint(-20, 20, (n, 1), generator=g).float()
    elif how == "ends":  # around half of the largest, neighbours of it
        x = torch.full((n, k), 0.5) + torch.randint(-3, 4, (n, k), generator=g) * 2.0 ** -24
        x[:, -1] = -1.0
    elif how == "tiny":  # the reciprocal of the largest is not finite
        x = x * 1e-39
    elif how == "huge":
        x = x * 1e37
    elif how == "zeros":
        x[::2] = 0.0
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("n,k", [(1, 1), (3, 7), (5, 16), (33, 100), (4, 4096), (2, 8192),
                                 (2, 8200), (7, 10007), (300, 520), (3, 40000), (2047, 130),
                                 (2048, 1), (2050, 17), (2049, 127), (2051, 128), (2048, 129),
                                 (2048, 255), (2049, 256), (2050, 257), (2048, 512),
                                 (2053, 511), (2048, 513), (2055, 1000), (2048, 1024),
                                 (2049, 1025), (2500, 1600), (2048, 2048), (2048, 2049)])
@pytest.mark.parametrize("how", ["normal", "halves", "ends", "tiny", "huge", "zeros"])
def test_quantize_rows(n, k, dtype, how):
    import nmce
    g = torch.Generator().manual_seed(n * k)
    x = _rows(n, k, dtype, g, how)
    q, s = nmce.quantize_rows(x.to(DEV))
    assert q.shape == (n, k) and q.dtype == torch.int8 and s.shape == (n,)
    assert n == 1 or q.stride(0) == -(-k // 16) * 16
    want, scale = _quotients(x)
    assert torch.equal(q.cpu().long(), want)
    # half a step, or half of the smallest number where the scale is that small
    assert bool(((s.double().cpu() - scale).abs() <= scale * 2.0 ** -24 + 2.0 ** -150).all())


def test_quantize_rows_that_are_not_finite():
    import nmce
    x = torch.randn(5, 40, device=DEV)
    x[1, 3], x[3, 39], x[4, 0] = float("nan"), float("inf"), float("-inf")
    for t in (x, x.to(BF)):
        q, s = nmce.quantize_rows(t)
        assert torch.isnan(s).tolist() == [False, True, False, True, True]
        assert not q[[1, 3, 4]].any() and bool(q[[0, 2]].any(dim=1).all())


def test_quantize_strides_and_padding():
    """Transposed, sliced, expanded rows; the bytes between padded rows are zero."""
    import nmce
    g = torch.Generator().manual_seed(2)
    base = torch.randn(6, 5, 50, generator=g).to(DEV)
    for x in (base.transpose(0, 1), base[..., 3:], base[:, ::2, 1:34], base[:1, :1].expand(4, 3, 50),
              base.permute(2, 0, 1), base[0, 0], base[:0]):
        q, s = nmce.quantize_rows(x)
        want, scale = _quotients(x.reshape(-1, x.shape[-1]))
        assert q.shape == x.shape and s.shape == x.shape[:-1]
        assert torch.equal(q.cpu().long().reshape(want.shape), want)
        k = x.shape[-1]
        whole = q.as_strided((max(1, want.shape[0]), -(-k // 16) * 16),
                             (-(-k // 16) * 16, 1)) if want.shape[0] else q
        assert not whole[..., k:].any()


def _product(x, wq, ws):
    q, s = _quotients(x)
    y = q.double() @ wq.cpu().double().t()
    return y * s[:, None] * ws.cpu().double()[None, :]


def _check(y, x, wq, ws):
    want = _product(x, wq, ws)
    err = (y.double().cpu() - want).abs()
    bound = want.abs() * (4 * 2.0 ** -24 + HALF_STEP[y.dtype]) * 1.01
    assert bool((err <= bound).all()), (err - bound).max()


SIZES = [  # n, k, v
    (1, 1, 1), (1, 16, 5), (2, 15, 17), (1, 4096, 1000), (3, 130, 257), (8, 64, 333),
    (15, 1600, 50257), (16, 128, 64), (17, 127, 65), (31, 257, 1001), (32, 768, 512),
    (33, 2000, 300), (48, 96, 50), (63, 1024, 77), (64, 640, 4100), (65, 640, 257),
    (100, 48, 31), (128, 300, 700), (129, 512, 2048), (255, 1, 3), (256, 256, 256),
    (257, 8192, 129), (700, 72, 513), (1000, 1000, 1000), (4, 131072, 33), (300, 131072, 20),
]


@pytest.mark.parametrize("dtype,od", [(BF, BF), (F32, F32), (BF, F32)])
@pytest.mark.parametrize("n,k,v", SIZES)
def test_int8_linear(n, k, v, dtype, od):
    import nmce
    g = torch.Generator().manual_seed(n + k + v)
    x = torch.randn(n, k, generator=g).to(dtype).to(DEV)
    w = torch.randn(v, k, generator=g) * 2.0 ** torch.randint(-9, 3, (v, 1), generator=g)
    wq, ws = nmce.quantize_rows(w.to(DEV))
    y = nmce.int8_linear(x, wq, ws, out_dtype=od)
    assert y.shape == (n, v) and y.dtype == od
    _check(y, x, wq, ws)


@pytest.mark.parametrize("n", [1, 40, 300])
def test_largest_sums(n):
    """Every product 127 x 127 of one sign over the most columns: the sum is
    2114060416, just inside 32 bits."""
    import nmce
    k = 131072
    x = torch.ones(n, k, dtype=BF, device=DEV)
    wq = torch.full((3, k), 127, dtype=torch.int8, device=DEV)
    wq[1] = -127
    wq[2] = -128  # not what quantize_rows makes, but a weight may hold it: -2130706432
    y = nmce.int8_linear(x, wq, torch.full((3,), 127.0, device=DEV), out_dtype=F32)
    want = torch.tensor([127.0 * k, -127.0 * k, -128.0 * k], dtype=torch.float64) * 127.0
    err = (y.double().cpu() - want).abs()
    assert bool((err <= want.abs() * 5 * 2.0 ** -24).all())


def test_weight_layouts_agree():
    """Rows the kernel takes as they lie, and others, which are copied: the
    same bits. Bytes behind a row's end change nothing."""
    import nmce
    g = torch.Generator().manual_seed(4)
    for n in (2, 40, 70, 300):
        for k in (33, 160):
            x = torch.randn(n, k, generator=g).to(DEV)
            wq, ws = nmce.quantize_rows(torch.randn(130, k, generator=g).to(DEV))
            y = nmce.int8_linear(x, wq, ws)
            other = [wq.contiguous(), wq.t().contiguous().t(), wq.clone()]
            wide = torch.randint(-128, 128, (130, 256), generator=g, dtype=torch.int8).to(DEV)
            wide[:, 16:16 + k] = wq
            other += [wide[:, 16:16 + k], wide.clone()[:, 15:15 + k].copy_(wq)]
            tight = torch.empty(129 * 48 * 4 + k, dtype=torch.int8, device=DEV)
            last = tight.as_strided((130, k), (48 * 4, 1))  # ends with its last element
            last.copy_(wq)
            other.append(last)
            for w in other:
                assert torch.equal(w, wq)
                assert torch.equal(nmce.int8_linear(x, w, ws), y)
            s2 = torch.stack([ws, ws], dim=1)[:, 0]  # a strided scale
            assert torch.equal(nmce.int8_linear(x, wq, s2), y)


def test_x_strides_shapes_and_empty():
    import nmce
    g = torch.Generator().manual_seed(5)
    wq, ws = nmce.quantize_rows(torch.randn(70, 40, generator=g).to(DEV))
    base = torch.randn(3, 5, 48, generator=g).to(BF).to(DEV)
    for x in (base[..., 1:41], base.transpose(0, 1)[..., :40], base[:1, :1, 8:].expand(3, 4, 40),
              base[0, 0, :40]):
        y = nmce.int8_linear(x, wq, ws)
        assert y.shape == x.shape[:-1] + (70,)
        _check(y.reshape(-1, 70), x.reshape(-1, 40), wq, ws)
    assert nmce.int8_linear(base[:0, :, :40], wq, ws).shape == (0, 5, 70)


@pytest.mark.parametrize("n", [3, 70, 300])
def test_rows_that_are_not_finite(n):
    """A token with a NaN or an infinity gives NaN, its neighbours are untouched;
    a token of zeros gives zeros; a weight row's NaN scale stays in its column."""
    import nmce
    g = torch.Generator().manual_seed(6)
    x = torch.randn(n, 100, generator=g).to(DEV)
    wq, ws = nmce.quantize_rows(torch.randn(80, 100, generator=g).to(DEV))
    clean = nmce.int8_linear(x, wq, ws)
    x[0, 99], x[1] = float("inf"), 0.0
    ws[7] = float("nan")
    y = nmce.int8_linear(x, wq, ws)
    assert bool(torch.isnan(y[0]).all()) and bool(torch.isnan(y[:, 7]).all())
    keep = torch.arange(80, device=DEV) != 7
    assert not y[1, keep].any() and torch.equal(y[2:, keep], clean[2:, keep])


@pytest.mark.parametrize("n,v,k", [(8300, 260000, 16), (40, 1100000, 4096), (300, 1100000, 4096)])
def test_offsets_past_32_bits(n, v, k):
    """Logits of more than 2^31 elements; a weight of more than 2^32 bytes, by both
    kernels: rows and columns at the ends and in the middle."""
    import nmce
    g = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randn(n, k, device=DEV, generator=g).to(BF)
    wq = torch.randint(-127, 128, (v, k), device=DEV, generator=g, dtype=torch.int8)
    ws = torch.rand(v, device=DEV, generator=g)
    y = nmce.int8_linear(x, wq, ws)
    for rows, cols in ((slice(0, 3), slice(0, 5)), (slice(n - 3, n), slice(v - 5, v)),
                       (slice(n - 3, n), slice(0, 5)), (slice(n // 2, n // 2 + 3),
                                                        slice(v // 2, v // 2 + 5))):
        _check(y[rows, cols], x[rows], wq[cols], ws[cols])


def test_int8_refusals():
    import nmce
    x = torch.randn(4, 32, device=DEV)
    wq, ws = nmce.quantize_rows(torch.randn(10, 32, device=DEV))
    with pytest.raises(RuntimeError, match="no backward"):
        nmce.int8_linear(x.clone().requires_grad_(True), wq, ws)
    with pytest.raises(RuntimeError, match="no backward"):
        nmce.quantize_rows(x.clone().requires_grad_(True))
    with torch.no_grad():
        nmce.int8_linear(x.clone().requires_grad_(True), wq, ws)
    for bad, error in (((x.half(), wq, ws), TypeError), ((x, wq.int(), ws), TypeError),
                       ((x, wq, ws.double()), TypeError), ((x[:, :31], wq, ws), ValueError),
                       ((x, wq, ws[:9]), ValueError), ((x, wq[:0], ws[:0]), ValueError),
                       ((x[:, :0], wq[:, :0], ws), ValueError),
                       ((x, wq.cpu(), ws), RuntimeError), ((x, wq, ws.cpu()), RuntimeError)):
        with pytest.raises(error, match="nmce|unsupported"):
            nmce.int8_linear(*bad)
    with pytest.raises(TypeError, match="unsupported"):
        nmce.int8_linear(x, wq, ws, out_dtype=torch.float16)
    big = torch.zeros(1, 131073, device=DEV)
    with pytest.raises(ValueError, match="at most 131072"):
        nmce.int8_linear(big, *nmce.quantize_rows(big))


def test_guard_bytes():
    """Through the C ABI: nothing outside the output's rows and the workspace
    is written."""
    from nmce import _lib as L
    import nmce
    lib = L.load()
    g = torch.Generator().manual_seed(7)
    for n, k, v, od in ((1, 33, 70, F32), (20, 100, 301, BF), (64, 16, 63, F32),
                        (130, 48, 259, BF), (300, 129, 257, F32)):
        x = torch.randn(n, k, generator=g).to(DEV)
        wq, ws = nmce.quantize_rows(torch.randn(v, k, generator=g).to(DEV))
        ldo = v + 5
        out = torch.full((n + 2, ldo), 7.0, dtype=od, device=DEV)
        need = lib.nmce_int8_linear_workspace_bytes(n, k)
        buf = torch.full((need + 512,), 0x5A, dtype=torch.uint8, device=DEV)
        L.check(lib.nmce_int8_linear(x.data_ptr(), L.NMCE_F32, n, k, k, wq.data_ptr(), v,
                                     wq.stride(0), ws.data_ptr(), out[1].data_ptr(),
                                     L.dtype_code(od), ldo, buf.data_ptr() + 256, need,
                                     L.stream_handle(torch.device(DEV))), "int8_linear")
        torch.cuda.synchronize()
        assert bool((buf[:256] == 0x5A).all()) and bool((buf[256 + need:] == 0x5A).all())
        assert bool((out[0] == 7.0).all()) and bool((out[n + 1] == 7.0).all())
        assert bool((out[:, v:] == 7.0).all())
        _check(out[1:n + 1, :v], x, wq, ws)


def test_graph_replays():
    import nmce
    g = torch.Generator().manual_seed(9)
    wq, ws = nmce.quantize_rows(torch.randn(1000, 200, generator=g).to(DEV))
    for n in (1, 33, 300):
        x = torch.zeros(n, 200, dtype=BF, device=DEV)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            nmce.int8_linear(x, wq, ws)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = nmce.int8_linear(x, wq, ws)
        for _ in range(3):
            x.copy_(torch.randn(n, 200, generator=g))
            graph.replay()
            torch.cuda.synchronize()
            got = y.clone()
            assert torch.equal(got, nmce.int8_linear(x, wq, ws))


def test_head_of_a_trained_head():
    """FusedParallelLMHead.quantized(): its logits are the 8-bit product of its
    weight, close to the head's own; a checkpoint carries them over."""
    import nmce
    ctx = nmce.ParallelContext.single()
    for width in (128, 100):
        cfg = types.SimpleNamespace(vocab_size=500, n_embd=width, sequence_parallel=False)
        torch.manual_seed(1)
        head = nmce.FusedParallelLMHead(cfg, ctx).to(DEV)
        serving = head.quantized()
        x = torch.randn(2, 3, width, device=DEV)
        with torch.no_grad():
            y, own = serving(x), head(x)
        wq, ws = nmce.quantize_rows(head.weight.detach())
        _check(y.reshape(-1, 500), x.reshape(-1, width), wq, ws)
        # each operand is off by at most half a step of 1 / 127 of its row's largest
        a, b = x.abs(), head.weight.detach().abs()
        step_a, step_b = a.amax(-1, keepdim=True) / 254, b.amax(-1, keepdim=True) / 254
        bound = step_a * b.sum(-1) + a.sum(-1, keepdim=True) * step_b.t() \
            + width * step_a * step_b.t()
        assert bool(((y - own).abs() <= bound + 1e-5).all())
        other = nmce.Int8ParallelLMHead(cfg, ctx).to(DEV)
        other.load_state_dict(serving.state_dict())
        with torch.no_grad():
            assert torch.equal(other(x), y)
        with pytest.raises(ValueError, match="is not this head's"):
            other.load_weight(head.weight[:, 1:])


def test_head_of_a_model_that_is_cast():
    """The serving head in a model cast to bf16 (and back) gives the logits it gave,
    to the bit."""
    import nmce
    cfg = types.SimpleNamespace(vocab_size=300, n_embd=72, sequence_parallel=False)
    torch.manual_seed(2)
    head = nmce.FusedParallelLMHead(cfg, nmce.ParallelContext.single()).to(DEV).quantized()
    x = torch.randn(2, 3, 72, device=DEV).to(BF)
    want = head(x)
    model = torch.nn.Sequential(head)
    for dtype in (BF, torch.float16, F32):
        assert torch.equal(model.to(dtype)(x), want)


def test_tangents_and_scales_that_require_grad_are_refused():
    """There is no derivative in either mode: none is dropped in silence."""
    from torch.autograd import forward_ad
    import nmce
    x = torch.randn(4, 32, device=DEV)
    wq, ws = nmce.quantize_rows(torch.randn(10, 32, device=DEV))
    with pytest.raises(RuntimeError, match="nmce: weight_scale requires grad"):
        nmce.int8_linear(x, wq, ws.clone().requires_grad_(True))
    with forward_ad.dual_level(), torch.no_grad():
        nmce.int8_linear(x, *nmce.quantize_rows(x))
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(RuntimeError, match="nmce: x has a forward-mode tangent"):
            nmce.quantize_rows(dual)
        with pytest.raises(RuntimeError, match="nmce: x has a forward-mode tangent"):
            nmce.int8_linear(dual, wq, ws)
        with pytest.raises(RuntimeError, match="nmce: weight_scale has a forward-mode tangent"):
            nmce.int8_linear(x, wq, forward_ad.make_dual(ws, torch.ones_like(ws)))


@pytest.mark.parametrize("copies", [1, 17])
def test_every_bf16_quotient(copies):
    """Every bf16 mantissa as the largest magnitude against every bf16 number from
    2^-10 up to it: quotients as near to a half as they come (129 x 2^-15 under 1 gives
    16383 / 32768), few rows and many."""
    import nmce
    top = 1.0 + torch.arange(128).float() / 128
    steps = torch.arange(2 ** 7, 2 ** 8).float() / 2 ** 7
    x = torch.cat([steps * 2.0 ** e for e in range(-10, 1)])
    rows = torch.where(x[None] <= top[:, None], x[None], 0.0)
    rows[:, ::3] *= -1.0
    rows = torch.cat([rows, top[:, None]], 1).repeat(copies, 1)
    assert torch.equal(rows.to(BF).float(), rows)
    q, s = nmce.quantize_rows(rows.to(BF).to(DEV))
    want, scale = _quotients(rows)
    assert torch.equal(q.cpu().long(), want)
    assert bool(((s.double().cpu() - scale).abs() <= scale * 2.0 ** -24).all())


@pytest.mark.parametrize("n", [40, 2100])
def test_fp32_neighbours_of_halves(n):
    """fp32 numbers next to (k + 1/2) top / 127 for every k: up to three steps off on
    both sides, under random largest magnitudes of any exponent."""
    import nmce
    g = torch.Generator().manual_seed(17)
    top = (1.0 + torch.rand(n, 1, generator=g)) * 2.0 ** torch.randint(-70, 70, (n, 1),
                                                                       generator=g).float()
    half = (torch.arange(127).double() + 0.5)[None] * top.double() / 127.0
    bits = half.float().view(torch.int32)[:, :, None] + torch.arange(-3, 4, dtype=torch.int32)
    x = torch.cat([bits.view(torch.float32).reshape(n, -1), top], 1)
    x[:, ::2] *= -1.0
    q, _ = nmce.quantize_rows(x.to(DEV))
    want, _ = _quotients(x)
    assert torch.equal(q.cpu().long(), want)


def test_fp32_logits_of_vast_vocabularies():
    """Rows of more than 2^21 fp32 logits, whose tiles leave element by element: the
    bits that the same tokens give a hundred at a time, and the definition's."""
    import nmce
    n, v, k = 300, (1 << 21) + 5, 16
    g = torch.Generator(device=DEV).manual_seed(18)
    x = torch.randn(n, k, device=DEV, generator=g)
    wq = torch.randint(-127, 128, (v, k), device=DEV, generator=g, dtype=torch.int8)
    ws = torch.rand(v, device=DEV, generator=g)
    y = nmce.int8_linear(x, wq, ws)
    for r in range(0, n, 100):
        assert torch.equal(y[r:r + 100], nmce.int8_linear(x[r:r + 100], wq, ws))
    for cols in (slice(0, 9), slice(v // 2, v // 2 + 300), slice(v - 300, v)):
        _check(y[:, cols], x, wq[cols], ws[cols])
