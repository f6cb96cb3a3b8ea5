"""What stands between a row of logits and those who use it, in the calls that a
serving or a distilling loop makes, with the plain forms.

* ``adjust``: penalties for tokens that a sequence holds already, biases of
  single ids and a bit mask of allowed ids, on the logits of each sequence's
  next token and of the tokens after its drafts.
* ``top``: the largest logits of each row with their ids (the lowest id first
  of equal ones) and the row's log-normaliser: what a server returns as top
  log-probabilities and what a teacher hands to a student.
* ``distill``: the Kullback-Leibler divergence from a teacher's top logits to
  the student's distribution over the whole vocabulary, and its gradient. With
  the teacher's log-normaliser the rest of the vocabulary is one class more;
  without, the teacher's distribution is over its top logits alone.
"""

import math
import pathlib
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # One user's decoding step a few tokens into the answer: latency.
        _adjust("adjust_one", "f32", 1, 0, 50257, prompt=37, output=5, bias=3, mask=False),
        # A serving batch, half of it under a grammar.
        _adjust("adjust_batch", "bf16", 64, 0, 128256, prompt=2048, output=512, bias=16, mask=True),
        # The positions of eight drafted tokens, each counting those before it.
        _adjust("adjust_drafts", "bf16", 24, 8, 151936, prompt=1000, output=250, bias=0, mask=True),
        # Long documents and their long answers, many biased ids.
        _adjust("adjust_long", "f32", 8, 0, 100277, prompt=131072, output=8192, bias=300,
                mask=False),
        # One user's top log-probabilities.
        _top("top_one", "f32", 1, 20, 50257),
        # The same for a serving batch.
        _top("top_batch", "bf16", 64, 20, 128256),
        # A teacher's logits of a micro-batch, what distillation keeps of them.
        _top("top_teacher", "bf16", 4096, 64, 128256),
        # An odd number of rows of an unpadded vocabulary, many kept.
        _top("top_wide", "f32", 777, 500, 100277),
        # A short sequence, the teacher's top logits alone.
        _distill("distill_small", "f32", 256, 20, 50257, False, 1.0, "mean"),
        # Odd rows and an unpadded vocabulary, softened.
        _distill("distill_odd", "bf16", 2047, 50, 50257, True, 2.0, "mean"),
        # A pretraining micro-batch.
        _distill("distill_large", "bf16", 8192, 64, 128256, True, 1.0, "mean"),
        # Losses by token, which the caller weights, over a wide vocabulary.
        _distill("distill_tokens", "bf16", 4096, 128, 151936, True, 1.0, "none"),
    ]


def _adjust(name, dtype, b, k, v, prompt, output, bias, mask):
    return dict(name=name, kind="adjust", dtype=dtype, b=b, k=k, v=v, prompt=prompt,
                output=output, bias=bias, mask=mask)


def _top(name, dtype, n, k, v):
    return dict(name=name, kind="top", dtype=dtype, n=n, k=k, v=v)


def _distill(name, dtype, n, k, v, tail, temperature, reduction):
    return dict(name=name, kind="distill", dtype=dtype, n=n, k=k, v=v, tail=tail,
                temperature=temperature, reduction=reduction)


_VOCABS = (32000, 50257, 50304, 64128, 100277, 128256, 151936, 256000)


def draw(rng):
    """A case of the listed ones' ranges: sizes spread over their logarithm, a
    known vocabulary half of the time, any width."""
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))

    kind = rng.choice(("adjust", "top", "distill"))
    v = rng.choice(_VOCABS) if rng.random() < 0.5 else spread(4096, 256000)
    dtype = rng.choice(("bf16", "bf16", "f32"))
    es = 2 if dtype == "bf16" else 4
    if kind == "adjust":
        k = rng.choice((0, 0, 1, 3, 5, 8))
        b = spread(1, min(64, 24 * 9 * 151936 * 2 // ((k + 1) * v * es)))
        return dict(kind=kind, dtype=dtype, b=b, k=k, v=v,
                    prompt=spread(1, min(131072, (1 << 20) // b)),
                    output=rng.choice((0, spread(1, min(8192, (1 << 16) // b)))),
                    bias=rng.choice((0, spread(1, 300))), mask=rng.random() < 0.5)
    if kind == "top":
        k = spread(1, 512)
        return dict(kind=kind, dtype=dtype, n=spread(1, min(4096, 4096 * 128256 * 2 // (v * es))),
                    k=k, v=v)
    return dict(kind=kind, dtype=dtype, n=spread(64, min(8192, 8192 * 128256 * 2 // (v * es))),
                k=spread(4, 256), v=v, tail=rng.random() < 0.6,
                temperature=rng.choice((1.0, 1.0, 2.0, 0.7)),
                reduction=rng.choice(("mean", "mean", "none")))


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _ids(shape, total, g):
    # Token ids as text has them, many small and few large: log-uniform.
    u = torch.rand(shape, device="cuda", generator=g, dtype=torch.float64)
    return (torch.exp(u * math.log(total + 1.0)) - 1.0).long().clamp_(0, total - 1)


def _logits(shape, dtype, g):
    """Rows with a body of small logits and a few that stand out."""
    x = torch.randn(shape, device="cuda", generator=g).mul_(2.0)
    up = torch.randint(0, shape[-1], shape[:-1] + (8,), device="cuda", generator=g)
    x.scatter_add_(-1, up, torch.rand(up.shape, device="cuda", generator=g).mul_(10.0))
    return x.to(_DTYPES[dtype])


def _padded(shape, total, g):
    """Lists of ids of several lengths, padded with -1."""
    ids = _ids(shape, total, g)
    if shape[1] == 0:
        return ids
    length = shape[1] - (torch.rand((shape[0], 1), device="cuda", generator=g)
                         * (shape[1] / 2)).long()
    return torch.where(torch.arange(shape[1], device="cuda") < length, ids, -1)


def prepare(case, seed):
    """Inputs, the same with ``own`` on and off."""
    g = _generator(seed)
    st = dict(case)
    if own:
        sys.path.insert(0, str(pathlib.Path(__file__).resolve().parent.parent /
                               "nano-megatron_amd"))
        import nmce
        st["nmce"] = nmce
        st["ctx"] = nmce.ParallelContext.single()
    if case["kind"] == "adjust":
        st.update(_adjust_inputs(case, g))
    elif case["kind"] == "top":
        st["logits"] = _logits((case["n"], case["v"]), case["dtype"], g)
    else:
        st.update(_distill_inputs(case, g))
    return st


def _adjust_inputs(case, g):
    b, k, v = case["b"], case["k"], case["v"]

    def rand(*shape):
        return torch.rand(shape, device="cuda", generator=g)

    r, f, p = 1.0 + 0.5 * rand(b), rand(b) - 0.25, rand(b) - 0.25
    if b > 2:  # a user in three has no penalties
        for t, neutral in ((r, 1.0), (f, 0.0), (p, 0.0)):
            t[2::3] = neutral
    st = dict(logits=_logits((b, k + 1, v), case["dtype"], g),
              prompt_tokens=_padded((b, case["prompt"]), v, g),
              output_tokens=_padded((b, case["output"]), v, g) if case["output"] else None,
              draft_tokens=_padded((b, k), v, g) if k else None,
              repetition=r, frequency=f, presence=p, bias_ids=None, bias_values=None,
              allowed=None)
    if case["bias"]:
        st["bias_ids"] = _padded((b, case["bias"]), v, g)
        st["bias_values"] = 8.0 * rand(b, case["bias"]) - 4.0
    if case["mask"]:
        words = (v + 31) // 32
        # Under a grammar: a row in two, of which a third allow few ids, a third
        # half of them, a third nearly all; other rows allow every id.
        kind = torch.randint(0, 6, (b, k + 1, 1), device="cuda", generator=g)

        def bits():
            return torch.randint(-(1 << 31), 1 << 31, (b, k + 1, words), device="cuda",
                                 generator=g)

        a, c = bits(), bits()
        few = a & c & bits() & bits() & bits() & bits()
        most = a | c | bits() | bits() | bits() | bits()
        st["allowed"] = torch.where(kind > 2, -1, torch.where(
            kind == 0, few, torch.where(kind == 1, a, most))).to(torch.int32)
    return st


def _distill_inputs(case, g):
    n, k, v = case["n"], case["k"], case["v"]
    x = _logits((n, v), case["dtype"], g)
    values = torch.empty((n, k), device="cuda")
    ids = torch.empty((n, k), dtype=torch.int64, device="cuda")
    norm = torch.empty((n,), device="cuda")
    for lo in range(0, n, 1024):  # a teacher that sees nearly the same logits
        part = x[lo:lo + 1024].float()
        part = part + torch.randn(part.shape, device="cuda", generator=g).mul_(0.7)
        values[lo:lo + 1024], ids[lo:lo + 1024] = torch.topk(part, k, dim=1)
        norm[lo:lo + 1024] = torch.logsumexp(part / case["temperature"], dim=1)
    # The first tokens are the prompt's and have no teacher; some lists are shorter.
    ids[:n // 8] = -1
    ids[n // 8::5, (k + 1) // 2:] = -1
    st = dict(logits=x.requires_grad_(True), teacher_logits=values, teacher_ids=ids,
              normalizer=norm if case["tail"] else None)
    if case["reduction"] == "none":
        st["weights"] = torch.rand((n,), device="cuda", generator=g) / n
    return st


def run(st):
    return _run_own(st) if own else _run_plain(st)


def _run_own(st):
    nmce = st["nmce"]
    v = st["v"]
    if st["kind"] == "adjust":
        return nmce.vocab_parallel_adjust_logits(
            st["logits"], 0, v, st["ctx"], prompt_tokens=st["prompt_tokens"],
            output_tokens=st["output_tokens"], draft_tokens=st["draft_tokens"],
            repetition_penalty=st["repetition"], frequency_penalty=st["frequency"],
            presence_penalty=st["presence"], bias_ids=st["bias_ids"],
            bias_values=st["bias_values"], allowed=st["allowed"])
    if st["kind"] == "top":
        return nmce.vocab_parallel_top_logits(st["logits"], st["k"], 0, v, st["ctx"])
    loss = nmce.vocab_parallel_distillation_loss(
        st["logits"], st["teacher_logits"], st["teacher_ids"], 0, v, st["ctx"],
        teacher_log_normalizer=st["normalizer"], temperature=st["temperature"],
        reduction=st["reduction"])
    return loss.detach(), torch.autograd.grad(loss, st["logits"], st.get("weights"))[0]


def _run_plain(st):
    if st["kind"] == "adjust":
        return _adjust_plain(st)
    if st["kind"] == "top":
        return _top_plain(st)
    return _distill_plain(st)


def _counts(lists, v):
    """How often each id occurs in each list, [B, V]."""
    b = lists[0].shape[0]
    out = torch.zeros((b, v + 1), device="cuda")
    for ids in lists:
        inside = (ids >= 0) & (ids < v)
        out.scatter_add_(1, torch.where(inside, ids, v), inside.float())
    return out[:, :v]


def _adjust_plain(st):
    x, v, k = st["logits"], st["v"], st["k"]
    out = torch.empty_like(x)
    r, f, p = (st[name][:, None] for name in ("repetition", "frequency", "presence"))
    prompt = _counts([st["prompt_tokens"]], v) > 0
    held = [st["output_tokens"]] if st["output_tokens"] is not None else []
    bias = None
    if st["bias_ids"] is not None:
        inside = st["bias_ids"] >= 0
        bias = torch.zeros((st["b"], v + 1), device="cuda")
        bias.scatter_add_(1, torch.where(inside, st["bias_ids"], v),
                          torch.where(inside, st["bias_values"], 0.0))
        bias = bias[:, :v]
    for i in range(k + 1):
        lists = held + ([st["draft_tokens"][:, :i]] if i else [])
        count = _counts(lists, v) if lists else torch.zeros_like(prompt, dtype=torch.float32)
        z = x[:, i].float()
        z = torch.where(prompt | (count > 0), torch.where(z > 0, z / r, z * r), z)
        z = z - f * count - p * (count > 0)
        if bias is not None:
            z = z + bias
        if st["allowed"] is not None:
            z = torch.where(_unpacked(st["allowed"][:, i], v), z, -math.inf)
        out[:, i] = z.to(x.dtype)
    return out


def _unpacked(words, v):
    bits = torch.arange(32, device="cuda", dtype=torch.int32)
    return ((words[..., None] >> bits) & 1).bool().flatten(-2)[..., :v]


def _top_plain(st):
    x, k = st["logits"], st["k"]
    n = x.shape[0]
    values = torch.empty((n, k), dtype=x.dtype, device="cuda")
    ids = torch.empty((n, k), dtype=torch.int64, device="cuda")
    norm = torch.empty((n,), device="cuda")
    for lo in range(0, n, 1024):
        part = x[lo:lo + 1024]
        # Stable: of equal logits the lowest id comes first.
        order = torch.sort(part, dim=1, descending=True, stable=True)
        values[lo:lo + 1024] = order.values[:, :k]
        ids[lo:lo + 1024] = order.indices[:, :k]
        top = order.values[:, :1].float()
        norm[lo:lo + 1024] = top[:, 0] + torch.log(torch.exp(part.float() - top).sum(dim=1))
    return values, ids, norm


def _distill_plain(st):
    x, t = st["logits"].detach(), st["temperature"]
    n, v = x.shape
    scale = st["weights"] if st["reduction"] == "none" else \
        torch.full((n,), 1.0 / n, device="cuda")
    grad = torch.empty_like(x)
    loss = torch.empty((n,), dtype=torch.float64, device="cuda")
    for lo in range(0, n, 2048):
        part = slice(lo, lo + 2048)
        ids = st["teacher_ids"][part]
        held = (ids >= 0) & (ids < v)
        at = torch.where(held, ids, v)
        # The teacher's side in 64 bits: few values, and 1 less their sum.
        teacher = torch.where(held, st["teacher_logits"][part].double() / t, -math.inf)
        some = held.any(dim=1)
        if st["normalizer"] is not None:
            p = torch.exp(teacher - st["normalizer"][part].double()[:, None])
            rest = torch.where(some, (1.0 - p.sum(dim=1)).clamp(min=0.0), 0.0)
        else:
            top = torch.where(some, teacher.amax(dim=1), 0.0)
            p = torch.exp(teacher - top[:, None])
            p = p / torch.where(some, p.sum(dim=1), 1.0)[:, None]
            rest = torch.zeros_like(top)
        whole = p.sum(dim=1) + rest
        z = x[part].float() / t
        top = z.amax(dim=1, keepdim=True)
        e = torch.exp(z - top)
        total = e.sum(dim=1)
        inside = torch.zeros((z.shape[0], v + 1), dtype=torch.bool, device="cuda")
        inside.scatter_(1, at, held)
        inside = inside[:, :v]
        outside = torch.where(inside, 0.0, e).sum(dim=1)
        log_total = torch.log(total.double())
        log_q = torch.where(held, (z - top).gather(1, at.clamp(max=v - 1)), 0.0).double() \
            - log_total[:, None]
        log_p = torch.log(torch.where(p > 0, p, 1.0))
        one = (p * (log_p - log_q)).sum(dim=1)
        more = rest > 0
        log_rest = torch.log(torch.where(more, rest, 1.0))
        log_outside = torch.log(torch.where(more, outside.double(), 1.0)) - log_total
        one = one + torch.where(more, rest * (log_rest - log_outside), 0.0)
        loss[part] = torch.where(some, one, 0.0)
        share = torch.where(more, rest.float() / outside, 0.0)
        dz = e * (whole.float() / total)[:, None]
        dz = dz - torch.where(inside, 0.0, e * share[:, None])
        full = torch.zeros((z.shape[0], v + 1), device="cuda")
        full.scatter_add_(1, at, p.float())
        dz = torch.where(some[:, None], dz - full[:, :v], 0.0)
        grad[part] = (dz * (scale[part] / t)[:, None]).to(x.dtype)
    if st["reduction"] == "none":
        return loss.float(), grad
    return loss.mean().float(), grad


def work(case):
    es = 2 if case["dtype"] == "bf16" else 4
    v, k = case["v"], case["k"]
    if case["kind"] == "adjust":
        b = case["b"]
        rows = b * (k + 1)
        ids = case["prompt"] + case["output"] + k
        return {"bytes": 2 * rows * v * es + b * (8 * ids + 12 * case["bias"] + 12)
                + (rows * 4 * ((v + 31) // 32) if case["mask"] else 0),
                "flops": rows * v + b * ids}
    n = case["n"]
    if case["kind"] == "top":
        return {"bytes": n * v * es + n * (k * (es + 8) + 4), "flops": 4 * n * v}
    return {"bytes": 2 * n * v * es + n * (12 * k + 8), "flops": 8 * n * v}


def exact(case, seed):
    """The definitions in 64 bits, a row at a time or over blocks of rows."""
    st = prepare(case, seed)
    if case["kind"] == "adjust":
        return _adjust_exact(case, st)
    if case["kind"] == "top":
        return _top_exact(case, st)
    return _distill_exact(case, st)


def _adjust_exact(case, st):
    b, k, v = case["b"], case["k"], case["v"]
    out = st["logits"].double()
    lists = {}
    for name in ("prompt_tokens", "output_tokens", "draft_tokens", "bias_ids", "bias_values"):
        lists[name] = st[name].cpu() if st[name] is not None else \
            torch.zeros((b, 0), dtype=torch.int64)
    for s in range(b):
        r, f, p = (float(st[name][s]) for name in ("repetition", "frequency", "presence"))
        prompt = lists["prompt_tokens"][s]
        prompt = torch.unique(prompt[prompt >= 0])
        for i in range(k + 1):
            mine = torch.cat([lists["output_tokens"][s], lists["draft_tokens"][s, :i]])
            ids, times = torch.unique(mine[mine >= 0], return_counts=True)
            row = out[s, i].cpu()
            seen = torch.unique(torch.cat([prompt, ids]))
            old = row[seen]
            row[seen] = torch.where(old > 0, old / r, old * r)
            row[ids] -= f * times.double() + p
            for j, value in zip(lists["bias_ids"][s].tolist(), lists["bias_values"][s].tolist()):
                if j >= 0:
                    row[j] += value
            if st["allowed"] is not None:
                words = st["allowed"][s, i].cpu().numpy().view("uint8")
                keep = torch.tensor([(byte >> j) & 1 for byte in range(256) for j in range(8)],
                                    dtype=torch.bool).view(256, 8)[torch.from_numpy(words).long()]
                row[~keep.flatten()[:v]] = -math.inf
            out[s, i] = row.cuda()
    return out


def _top_exact(case, st):
    n, k = case["n"], case["k"]
    values, ids, norm = [], [], []
    for lo in range(0, n, 1024):
        z = st["logits"][lo:lo + 1024].double()
        low = torch.kthvalue(-z, k, dim=1).values.neg()[:, None]  # the k-th largest
        above = z > low
        need = k - above.sum(dim=1, keepdim=True)
        ties = z == low
        keep = above | (ties & (torch.cumsum(ties, dim=1) <= need))
        which = torch.nonzero(keep)[:, 1].view(-1, k)  # by id
        got = z.gather(1, which)
        order = torch.argsort(got, dim=1, descending=True, stable=True)
        values.append(got.gather(1, order))
        ids.append(which.gather(1, order))
        norm.append(torch.logsumexp(z, dim=1))
    return torch.cat(values), torch.cat(ids), torch.cat(norm)


def _distill_exact(case, st):
    n, v, t = case["n"], case["v"], case["temperature"]
    x = st["logits"].detach()
    grad = torch.empty((n, v), dtype=torch.float64, device="cuda")
    losses = []
    for lo in range(0, n, 512):
        z = x[lo:lo + 512].double() / t
        ids = st["teacher_ids"][lo:lo + 512]
        rows = torch.arange(z.shape[0], device="cuda")[:, None].expand_as(ids)
        on = ids >= 0
        # Dense in the classes: -inf where the teacher has no logit.
        dense = torch.full_like(z, -math.inf)
        dense[rows[on], ids[on]] = st["teacher_logits"][lo:lo + 512].double()[on] / t
        listed_ = dense > -math.inf
        taught = listed_.any(dim=1)
        norm = torch.logsumexp(dense, dim=1) if st["normalizer"] is None else \
            st["normalizer"][lo:lo + 512].double()
        log_p = torch.where(taught[:, None], dense - norm[:, None], -math.inf)
        p = torch.exp(log_p)
        left = 1.0 - p.sum(dim=1)
        if st["normalizer"] is None:
            left = torch.zeros_like(left)
        left = torch.where(taught, torch.relu(left), 0.0)
        log_q = torch.log_softmax(z, dim=1)
        terms = torch.where(listed_, p * (torch.where(listed_, log_p, 0.0) - log_q), 0.0)
        log_s = torch.logsumexp(torch.where(listed_, -math.inf, log_q), dim=1)
        loss = terms.sum(dim=1) + torch.special.xlogy(left, left) - left * log_s
        others = torch.exp(log_q - log_s[:, None])  # within the rest
        mass = (p.sum(dim=1) + left)[:, None]
        d = mass * torch.exp(log_q) - torch.where(listed_, p, left[:, None] * others)
        up = st["weights"][lo:lo + 512].double() if case["reduction"] == "none" else \
            torch.full((z.shape[0],), 1.0 / n, dtype=torch.float64, device="cuda")
        grad[lo:lo + 512] = torch.where(taught[:, None], d * (up / t)[:, None], 0.0)
        losses.append(torch.where(taught, loss, 0.0))
    loss = torch.cat(losses)
    return (loss if case["reduction"] == "none" else loss.mean()), grad
