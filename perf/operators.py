"""The operators at the vocabulary's two ends, in the calls that a training or a
serving loop makes of them, with their plain forms.

* ``embed``: token ids to hidden rows over a vocabulary shard of the (tied)
  weight, scaled, and the weight's dense gradient; ``lookup`` is its forward
  alone, as a decoding step makes it.
* ``int8``: hidden rows to logits with an 8-bit weight: each token quantised to
  8 bits by its largest magnitude, an integer product, one scale per token and
  per vocabulary row. ``quantize`` makes such a weight.
* ``verify``: drafted tokens against the target model's probabilities, from
  given uniform numbers: the accepted ones and the token that follows, how many
  were accepted, and the log-probability of each.
"""

import math
import pathlib
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # One decoding step of a small batch: a few rows fetched; latency.
        _lookup("lookup_decode", "bf16", 17, 4096, 128256),
        # A fine-tuning step of a small model on one short sequence: fp32 master
        # weights, bf16 activations.
        _embed("embed_small", "f32", "bf16", 512, 768, 50304),
        # Odd everywhere: an odd width and the unpadded vocabulary, one rank of
        # a pair (half of the ids are the other rank's).
        _embed("embed_shard", "f32", "f32", 2103, 1601, 25129, start=25129),
        # The ordinary pretraining micro-batch of a large model.
        _embed("embed_large", "bf16", "bf16", 16384, 4096, 128256),
        # A long batch over a small vocabulary: the common ids come thousands
        # of times each.
        _embed("embed_long", "bf16", "bf16", 131072, 1024, 32000),
        # One token's logits: the weight is read once.
        _int8("int8_token", "bf16", 1, 4096, 128256),
        # A decoding batch on the unpadded vocabulary, fp32 logits.
        _int8("int8_batch", "f32", 48, 1600, 50257),
        # Prompt scoring: every token's logits, a product that fills the chip.
        _int8("int8_prompt", "bf16", 2048, 4096, 128256),
        # Making the 8-bit weight from a bf16 checkpoint's.
        dict(name="quantize_weight", kind="quantize", dtype="bf16", n=50257, h=1600),
        # One user's decoding step, four drafted tokens, fp32 logits.
        _verify("verify_one", "f32", 1, 4, 50257, "model"),
        # A serving batch with a draft model.
        _verify("verify_batch", "bf16", 64, 5, 128256, "model"),
        # Drafts copied from the prompt: no draft probabilities.
        _verify("verify_copied", "bf16", 24, 8, 151936, "none"),
    ]


def _lookup(name, dtype, n, h, v):
    return dict(name=name, kind="lookup", wdtype=dtype, odtype=dtype, n=n, h=h, v=v, start=0)


def _embed(name, wdtype, odtype, n, h, v, start=0):
    return dict(name=name, kind="embed", wdtype=wdtype, odtype=odtype, n=n, h=h, v=v, start=start)


def _int8(name, dtype, n, h, v):
    return dict(name=name, kind="int8", dtype=dtype, n=n, h=h, v=v)


def _verify(name, dtype, b, k, v, drafts):
    return dict(name=name, kind="verify", dtype=dtype, b=b, k=k, v=v, drafts=drafts)


_VOCABS = (32000, 50257, 50304, 64128, 100277, 128256, 151936, 256000)


def draw(rng):
    """A case of the listed ones' ranges: sizes spread over their logarithm, a
    known vocabulary half of the time, any width."""
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))

    kind = rng.choice(("lookup", "embed", "embed", "embed", "int8", "int8", "int8", "quantize",
                       "verify", "verify", "verify"))
    v = rng.choice(_VOCABS) if rng.random() < 0.5 else spread(4096, 256000)
    dtype = rng.choice(("bf16", "bf16", "f32"))
    if kind in ("lookup", "embed"):
        es = 2 if dtype == "bf16" else 4
        h = spread(64, min(8192, (3 << 28) // (v * es)))
        h = h if rng.random() < 0.3 else max(64, h // 64 * 64)
        n = spread(1, 1024) if kind == "lookup" else spread(1, min(131072, (1 << 27) * 2 // (h * es)))
        start = rng.choice((0, 0, v))
        odtype = rng.choice(("bf16", dtype))
        return dict(kind=kind, wdtype=dtype, odtype=odtype, n=n, h=h, v=v, start=start)
    if kind == "quantize":
        h = spread(64, 8192)
        return dict(kind=kind, dtype=dtype, n=spread(1, (1 << 27) // h), h=h)
    if kind == "int8":
        h = spread(64, 8192)
        h = h if rng.random() < 0.3 else max(64, h // 64 * 64)
        v = min(v, (1 << 29) // h)
        most = 2048 * 128256  # int8_prompt's logits; three quarters of its products
        n = spread(1, min(4096, most // v, most * 4096 * 3 // (4 * h * v)))
        return dict(kind=kind, dtype=dtype, n=n, h=h, v=v)
    k = rng.randint(0, 8)
    b = spread(1, min(128, 64 * 11 * 128256 // ((2 * k + 1) * v)))
    return dict(kind=kind, dtype=dtype, b=b, k=k, v=v, drafts=rng.choice(("model", "model", "none")))


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _ids(shape, total, g):
    # Token ids as text has them, many small and few large: log-uniform.
    u = torch.rand(shape, device="cuda", generator=g, dtype=torch.float64)
    return (torch.exp(u * math.log(total + 1.0)) - 1.0).long().clamp_(0, total - 1)


def prepare(case, seed):
    """Inputs and the weights that a program keeps. The tensors are the same
    with ``own`` on and off; with it the 8-bit weight is made by the framework."""
    g = _generator(seed)
    st = dict(case)
    kind = case["kind"]
    if own:
        sys.path.insert(0, str(pathlib.Path(__file__).resolve().parent.parent /
                               "nano-megatron_amd"))
        import nmce
        st["nmce"] = nmce
        st["ctx"] = nmce.ParallelContext.single()
    if kind in ("lookup", "embed"):
        n, h, v = case["n"], case["h"], case["v"]
        # A shard that does not start at 0 is the upper half of the ids, and
        # spread ids keep both halves in use.
        if case["start"]:
            st["tokens"] = torch.randint(0, 2 * v, (n,), device="cuda", generator=g)
        else:
            st["tokens"] = _ids((n,), v, g)
        st["weight"] = _normal((v, h), 0.02, case["wdtype"], g)
        st["scale"] = math.sqrt(h)
        if kind == "embed":
            st["grad"] = _normal((n, h), 1e-3, case["odtype"], g)
            if own:
                st["weight"].requires_grad_(True)
    elif kind == "quantize":
        st["x"] = _normal((case["n"], case["h"]), 0.02, case["dtype"], g)
    elif kind == "int8":
        st["x"] = _hidden(case, g)
        w = _normal((case["v"], case["h"]), 0.02, "bf16", g)
        st["wq"], st["ws"] = st["nmce"].quantize_rows(w) if own else _quantize(w)
    else:
        st.update(_drafted(case, g))
    return st


def _normal(shape, std, dtype, g):
    x = torch.empty(shape, device="cuda", dtype=_DTYPES[dtype])
    rows = max(1, (1 << 28) // max(1, shape[1]))
    for r in range(0, shape[0], rows):
        part = x[r:r + rows]
        part.copy_(torch.randn(part.shape, device="cuda", generator=g).mul_(std))
    return x


def _hidden(case, g):
    # Normalised hidden rows with a few channels much larger than the others.
    x = torch.randn((case["n"], case["h"]), device="cuda", generator=g)
    big = torch.rand((case["h"],), device="cuda", generator=g) < 0.005
    return torch.where(big, x * 12.0, x).to(_DTYPES[case["dtype"]])


def _drafted(case, g):
    # The draft model sees nearly the target's logits, and its tokens are drawn
    # from its own distribution (or copied from a prompt: likely ones).
    b, k, v = case["b"], case["k"], case["v"]
    dt = _DTYPES[case["dtype"]]
    x = torch.randn((b, k + 1, v), device="cuda", generator=g).mul_(2.0)
    up = torch.randint(0, v, (b, k + 1, 4), device="cuda", generator=g)
    x.scatter_add_(2, up, torch.rand(up.shape, device="cuda", generator=g).mul_(12.0))
    y = x[:, :k] + torch.randn((b, k, v), device="cuda", generator=g).mul_(0.5)
    x, y = x.to(dt), y.to(dt)
    temperature = 0.5 + torch.rand((b,), device="cuda", generator=g)
    temperature[3::4] = 0.0  # a user in four decodes greedily
    t = torch.where(temperature > 0, temperature, 0.2).view(b, 1, 1)
    noise = torch.empty((b, k, v), device="cuda").exponential_(generator=g)
    tokens = (torch.softmax(y.float() / t, dim=-1) / noise).argmax(-1) if k else \
        torch.zeros((b, 0), dtype=torch.int64, device="cuda")
    if k > 1 and b > 1:
        tokens[1::3, -1] = -1  # some have one draft fewer
    return dict(target=x, draft=y if case["drafts"] == "model" else None, tokens=tokens,
                temperature=temperature,
                accept_u=torch.rand((b, k), device="cuda", generator=g),
                sample_u=torch.rand((b,), device="cuda", generator=g))


def run(st):
    return _run_own(st) if own else _run_plain(st)


def _run_own(st):
    nmce, kind = st["nmce"], st["kind"]
    if kind in ("lookup", "embed"):
        out = nmce.vocab_parallel_embedding(
            st["tokens"], st["weight"], st["start"], st["start"] + st["v"], st["ctx"],
            scale=st["scale"], out_dtype=_DTYPES[st["odtype"]], validate=False)
        if kind == "lookup":
            return out
        return out.detach(), torch.autograd.grad(out, st["weight"], st["grad"])[0]
    if kind == "quantize":
        return nmce.quantize_rows(st["x"])
    if kind == "int8":
        return nmce.int8_linear(st["x"], st["wq"], st["ws"])
    return nmce.vocab_parallel_verify_drafts(
        st["target"], st["tokens"], st["draft"], st["accept_u"], st["sample_u"], 0, st["v"],
        st["ctx"], temperature=st["temperature"])


def _run_plain(st):
    kind = st["kind"]
    if kind in ("lookup", "embed"):
        local = st["tokens"] - st["start"]
        inside = (local >= 0) & (local < st["v"])
        at = torch.where(inside, local, 0)
        rows = st["weight"][at].float() * st["scale"]
        out = torch.where(inside[:, None], rows, 0.0).to(_DTYPES[st["odtype"]])
        if kind == "lookup":
            return out
        dw = torch.zeros((st["v"], st["h"]), dtype=torch.float32, device="cuda")
        part = torch.where(inside[:, None], st["grad"].float() * st["scale"], 0.0)
        dw.index_add_(0, at, part)
        return out, dw.to(_DTYPES[st["wdtype"]])
    if kind == "quantize":
        return _quantize(st["x"])
    if kind == "int8":
        q, s = _quantize(st["x"])
        y = q.float() @ st["wq"].float().t()
        return (y * s[:, None] * st["ws"][None, :]).to(_DTYPES[st["dtype"]])
    return _verify_plain(st)


def _quantize(x):
    """8-bit rows and their scales. The quotient is taken in 64 bits: halves
    (an element of half the largest magnitude) go to the even neighbour."""
    q = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    s = torch.empty(x.shape[:1], dtype=torch.float32, device=x.device)
    rows = max(1, (1 << 27) // x.shape[1])
    for r in range(0, x.shape[0], rows):
        part = x[r:r + rows].double()
        top = part.abs().amax(dim=1, keepdim=True)
        q[r:r + rows] = torch.round(part * 127.0 / torch.where(top > 0, top, 1.0)).to(torch.int8)
        s[r:r + rows] = (top[:, 0] / 127.0).float()
    return q, s


def _verify_plain(st):
    # In 64 bits: a token lies next to the border of its interval as soon as
    # the vocabulary is large.
    x, tokens, temperature = st["target"], st["tokens"], st["temperature"]
    b, k, v = st["b"], st["k"], st["v"]
    greedy = temperature == 0
    t = torch.where(greedy, 1.0, temperature.double()).view(b, 1, 1)
    p = _probabilities(x, t)
    best = _first_max(x)
    drafted = tokens >= 0
    at = torch.where(drafted, tokens, 0).unsqueeze(2)
    p_d = p[:, :k].gather(2, at).squeeze(2)
    if st["draft"] is not None:
        q = _probabilities(st["draft"], t)
        q_d = q.gather(2, at).squeeze(2)
    else:
        q = None
        q_d = torch.ones_like(p_d)
    ok = torch.where(greedy[:, None], tokens == best[:, :k], st["accept_u"].double() * q_d < p_d)
    ok = ok & drafted
    accepted = torch.cumprod(ok.long(), dim=1).sum(dim=1)
    every = torch.arange(b, device="cuda")
    row = p[every, accepted]
    # Stopped at a draft: what the target has above the draft's distribution.
    last = accepted.clamp(max=max(k - 1, 0))
    if k:
        refused = (accepted < k) & drafted[every, last]
        if q is not None:
            rest = (row - q[every, last]).clamp_(min=0.0)
        else:
            rest = row.scatter(1, at[every, last], 0.0)
        refused = refused & (rest.sum(dim=1) > 0)
        row = torch.where(refused[:, None], rest, row)
    mass = torch.cumsum(row, dim=1)
    level = st["sample_u"].double() * mass[:, -1]
    pick = (mass <= level[:, None]).sum(dim=1).clamp_(max=v - 1)
    pick = torch.where(greedy, best[every, accepted], pick)
    places = torch.arange(k + 1, device="cuda")[None, :]
    out = torch.full((b, k + 1), -1, dtype=torch.int64, device="cuda")
    out[:, :k] = tokens
    out = torch.where(places < accepted[:, None], out, -1)
    out = torch.where(places == accepted[:, None], pick[:, None], out)
    given = p.gather(2, out.clamp(min=0).unsqueeze(2)).squeeze(2)
    logp = torch.where(out >= 0, torch.log(torch.where(out >= 0, given, 1.0)), 0.0).float()
    return out, accepted, logp


def _probabilities(x, t):
    z = x.double()
    e = torch.exp((z - z.amax(dim=-1, keepdim=True)) / t)
    return e / e.sum(dim=-1, keepdim=True)


def _first_max(x):
    # The lowest id of the largest logit.
    ids = torch.arange(x.shape[-1], device=x.device)
    top = x.amax(dim=-1, keepdim=True)
    return torch.where(x == top, ids, x.shape[-1]).amin(dim=-1)


def work(case):
    kind = case["kind"]
    if kind in ("lookup", "embed"):
        n, h, v = case["n"], case["h"], case["v"]
        w, o = (2 if case[d] == "bf16" else 4 for d in ("wdtype", "odtype"))
        share = 0.5 if case["start"] else 1.0  # ids that are this shard's
        rows = min(n * share, v)
        bytes_, flops = 8 * n + rows * h * w + n * h * o, n * share * h
        if kind == "embed":
            bytes_ += 8 * n + n * share * h * o + v * h * w
            flops += 2 * n * share * h
        return {"bytes": bytes_, "flops": flops}
    if kind == "quantize":
        n, h = case["n"], case["h"]
        return {"bytes": n * h * ((2 if case["dtype"] == "bf16" else 4) + 1) + 4 * n,
                "flops": 3 * n * h}
    es = 2 if case["dtype"] == "bf16" else 4
    if kind == "int8":
        n, h, v = case["n"], case["h"], case["v"]
        return {"bytes": n * h * es + v * h + 4 * v + n * v * es, "flops": 2 * n * h * v}
    b, k, v = case["b"], case["k"], case["v"]
    rows = b * (2 * k + 1) if case["drafts"] == "model" else b * (k + 1)
    return {"bytes": rows * v * es + b * (24 * k + 28), "flops": 4 * rows * v}


def exact(case, seed):
    """The definitions in 64 bits, row by row where that is quick."""
    st = prepare(case, seed)
    kind = case["kind"]
    if kind in ("lookup", "embed"):
        n, h, v = case["n"], case["h"], case["v"]
        scale = math.sqrt(h)
        padded = torch.cat([torch.zeros((1, h), dtype=torch.float64, device="cuda"),
                            st["weight"].detach().double()])
        slot = st["tokens"] - case["start"] + 1
        slot = torch.where((slot < 1) | (slot > v), torch.zeros_like(slot), slot)
        out = padded.index_select(0, slot).mul_(scale)
        if kind == "lookup":
            return out
        del padded
        order = torch.argsort(slot, stable=True)
        ids, counts = torch.unique_consecutive(slot[order], return_counts=True)
        dw = torch.zeros((v + 1, h), dtype=torch.float64, device="cuda")
        ends = torch.cumsum(counts, 0).tolist()
        first = 0
        # Segments by their length: the long ones each summed as a block, the
        # short ones in one padded gather of each power of two.
        groups = {}
        for i, end in enumerate(ends):
            size = end - first
            groups.setdefault(1 << (size - 1).bit_length(), []).append((i, first, size))
            first = end
        grad = torch.cat([st["grad"].double(),
                          torch.zeros((1, h), dtype=torch.float64, device="cuda")])
        for width, segments in groups.items():
            most = max(1, (1 << 27) // (width * h))
            for lo in range(0, len(segments), most):
                part = segments[lo:lo + most]
                which = torch.tensor([s[0] for s in part], device="cuda")
                begin = torch.tensor([s[1] for s in part], device="cuda")[:, None]
                size = torch.tensor([s[2] for s in part], device="cuda")[:, None]
                j = torch.arange(width, device="cuda")[None, :]
                pos = torch.where(j < size, order[(begin + j).clamp(max=n - 1)], n)
                dw[ids[which]] = grad[pos].sum(dim=1)
        return out, dw[1:].mul_(scale)
    if kind == "quantize":
        return _exact_rows(st["x"])
    if kind == "int8":
        q, s = _exact_rows(st["x"])
        out = torch.empty((case["n"], case["v"]), dtype=torch.float64, device="cuda")
        for lo in range(0, case["v"], 16384):
            w = st["wq"][lo:lo + 16384].double()
            out[:, lo:lo + 16384] = torch.mm(q.double(), w.t().contiguous())
        return out.mul_(s[:, None]).mul_(st["ws"].double()[None, :])
    return _exact_verify(case, st)


def _exact_rows(x):
    q = torch.empty(x.shape, dtype=torch.int8, device="cuda")
    scales = []
    for part, out in zip(x.split(16384), q.split(16384)):
        wide = part.to(torch.float64)
        top = torch.maximum(wide.max(dim=1).values, -wide.min(dim=1).values)
        steps = torch.div(127.0 * wide, torch.where(top == 0, 1.0, top).unsqueeze(1))
        low = torch.floor(steps)
        up = (steps - low > 0.5) | ((steps - low == 0.5) & (torch.remainder(low, 2.0) == 1.0))
        out.copy_((low + up).to(torch.int8))
        scales.append(top / 127.0)
    return q, torch.cat(scales)


def _exact_verify(case, st):
    b, k, v = case["b"], case["k"], case["v"]
    out = torch.full((b, k + 1), -1, dtype=torch.int64)
    logp = torch.zeros((b, k + 1), dtype=torch.float64)
    accepted = torch.zeros((b,), dtype=torch.int64)
    tokens = st["tokens"].tolist()
    heat, au, su = st["temperature"].tolist(), st["accept_u"].tolist(), st["sample_u"].tolist()

    def weights(row, t):
        z = (row.double() - row.double().max()) / t
        e = torch.exp(z)
        return e / e.sum()

    for i in range(b):
        j, t = 0, heat[i]
        while True:
            row = st["target"][i, j]
            more = j < k and tokens[i][j] >= 0
            p = weights(row, t if t > 0 else 1.0)
            if t == 0:
                nxt = int(torch.nonzero(row == row.max())[0])
                if more and nxt == tokens[i][j]:
                    out[i, j], logp[i, j] = nxt, math.log(p[nxt].item())
                    j += 1
                    continue
                break
            if not more:
                nxt = _draw_exact(p, su[i])
                break
            d = tokens[i][j]
            if st["draft"] is None:
                q = torch.zeros_like(p)
                q[d] = 1.0
            else:
                q = weights(st["draft"][i, j], t)
            if au[i][j] * q[d].item() < p[d].item():
                out[i, j], logp[i, j] = d, math.log(p[d].item())
                j += 1
                continue
            rest = torch.relu(p - q)
            nxt = _draw_exact(rest if rest.sum().item() > 0 else p, su[i])
            break
        accepted[i] = j
        out[i, j], logp[i, j] = nxt, math.log(p[nxt].item())
    return out.cuda(), accepted.cuda(), logp.cuda()


def _draw_exact(weight, u):
    mass = torch.cumsum(weight, 0)
    return min(int(torch.searchsorted(mass, u * mass[-1].item(), right=True)), len(weight) - 1)
