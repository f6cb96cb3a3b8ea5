"""The operators together, as a server and a distilling training step use them, and under
tensor parallelism (ranks share cuda:0 and talk over gloo, with host copies)."""

from __future__ import annotations

import os
import socket
import types

import numpy as np
import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
B, K, H, V = 3, 2, 96, 4 * 1500


def _inputs():
    g = torch.Generator().manual_seed(31)
    weight = torch.randn(V, H, generator=g) * 0.2
    teacher = weight + 0.05 * torch.randn(V, H, generator=g)
    x = torch.randn(B, K + 1, H, generator=g)
    prompt = torch.randint(0, V, (B, 40), generator=g)
    output = torch.randint(0, V, (B, 12), generator=g)
    drafts = torch.randint(0, V, (B, K), generator=g)
    drafts[1, 1] = -1
    allowed = torch.randint(-2 ** 31, 2 ** 31, (B, K + 1, -(-V // 32)), generator=g,
                            dtype=torch.int64).to(torch.int32)
    u = torch.rand(B, K, generator=g), torch.rand(B, generator=g)
    targets = torch.randint(0, V, (B, K + 1), generator=g)
    return weight, teacher, x, prompt, output, drafts, allowed, u, targets


def _results(rank, ctx, dev):
    """A serving step and a distilling step on this rank's shard."""
    import nmce
    weight, teacher, x, prompt, output, drafts, allowed, u, targets = _inputs()
    per = V // ctx.tp_size
    lo, hi = rank * per, (rank + 1) * per
    cfg = types.SimpleNamespace(vocab_size=V, n_embd=H, sequence_parallel=False)
    res = {}

    def head(w):
        module = nmce.FusedParallelLMHead(cfg, ctx)
        module.weight = torch.nn.Parameter(w[lo:hi].to(dev))
        return module

    # Serving: 8-bit logits, adjusted, their top log-probabilities, the drafts verified.
    with torch.no_grad():
        logits = head(weight).quantized()(x.to(dev))
        adjusted = nmce.vocab_parallel_adjust_logits(
            logits, lo, hi, ctx, prompt_tokens=prompt.to(dev), output_tokens=output.to(dev),
            draft_tokens=drafts.to(dev), repetition_penalty=1.2, frequency_penalty=0.3,
            presence_penalty=0.1, bias_ids=prompt[:, :4].to(dev),
            bias_values=torch.full((B, 4), 2.0, device=dev), allowed=allowed.to(dev))
        top = nmce.vocab_parallel_top_logits(adjusted, 10, lo, hi, ctx)
        tokens, accepted, logprobs = nmce.vocab_parallel_verify_drafts(
            adjusted, drafts.to(dev), None, u[0].to(dev), u[1].to(dev), lo, hi, ctx)
    res.update(logits=logits, adjusted=adjusted, top_values=top[0], top_ids=top[1],
               top_norm=top[2], tokens=tokens, accepted=accepted, logprobs=logprobs)
    # Training: the teacher's top logits, the student's two losses, the weight's gradient.
    with torch.no_grad():
        taught = head(teacher)
        t_values, t_ids, t_norm = nmce.vocab_parallel_top_logits(
            taught(x.to(dev)), 20, lo, hi, ctx, temperature=2.0)
    student = head(weight)
    for name, kw in (("mean", {}), ("none", {"reduction": "none"})):
        z = student(x.to(dev))
        distilled = nmce.vocab_parallel_distillation_loss(
            z, t_values, t_ids, lo, hi, ctx, teacher_log_normalizer=t_norm, temperature=2.0, **kw)
        loss = 4.0 * distilled.mean() + nmce.vocab_parallel_cross_entropy(
            z, targets.to(dev), lo, hi, ctx, inplace=False)
        student.weight.grad = None
        loss.backward()
        res[f"loss_{name}"], res[f"dw_{name}"] = distilled.detach(), student.weight.grad
    res.update(t_values=t_values, t_ids=t_ids, t_norm=t_norm)
    torch.cuda.synchronize()
    return {k: v.float().cpu().numpy() if v.dtype == torch.bfloat16 else v.cpu().numpy()
            for k, v in res.items()}


@pytest.fixture(scope="module")
def whole():
    import nmce
    return _results(0, nmce.ParallelContext.single(), torch.device(DEV))


def test_serving_step(whole):
    """What the sampler is given: no masked id comes out, the log-probabilities are those
    of the adjusted logits."""
    adjusted = torch.from_numpy(whole["adjusted"]).double()
    logp = torch.log_softmax(adjusted, -1)
    order = torch.sort(adjusted, dim=-1, descending=True, stable=True)
    assert np.array_equal(whole["top_ids"], order.indices[..., :10].numpy())
    got = whole["top_values"] - whole["top_norm"][..., None]
    want = logp.gather(2, order.indices[..., :10]).numpy()
    assert np.abs(got - want).max() <= 2.0 ** -20 * 20
    for b in range(B):
        n = int(whole["accepted"][b])
        for i in range(n + 1):
            j = int(whole["tokens"][b, i])
            assert j >= 0 and np.isfinite(whole["adjusted"][b, i, j])
            assert abs(whole["logprobs"][b, i] - float(logp[b, i, j])) <= 2.0 ** -20 * 20


def test_two_captured_runs_at_once():
    """A server's and a trainer's calls, captured twice with other inputs and upstream
    values, and replayed on two streams at the same time: no memory is shared."""
    import nmce
    ctx = nmce.ParallelContext.single()
    n, v, k = 24, 20000, 20
    g = torch.Generator().manual_seed(32)
    runs = []
    for i, up in enumerate((1.0, 8.0)):
        logits = (torch.randn(n, 1, v, generator=g) * 3).to(DEV, torch.bfloat16)
        output = torch.randint(0, v, (n, 300), generator=g).to(DEV)
        student = torch.randn(n, v, generator=g).to(DEV, torch.bfloat16).requires_grad_(True)
        runs.append((logits, output, student, torch.tensor(up, device=DEV)))

    def step(logits, output, student, up):
        with torch.no_grad():
            adjusted = nmce.vocab_parallel_adjust_logits(
                logits, 0, v, ctx, output_tokens=output, repetition_penalty=1.3,
                frequency_penalty=0.5, bias_ids=output[:, :7], bias_values=output[:, :7].float())
            values, ids, norm = nmce.vocab_parallel_top_logits(adjusted[:, 0], k, 0, v, ctx)
        loss = nmce.vocab_parallel_distillation_loss(student, values, ids, 0, v, ctx,
                                                     teacher_log_normalizer=norm)
        grad, = torch.autograd.grad(loss, student, up)
        return adjusted, values, ids, norm, loss.detach(), grad

    want = [tuple(t.clone() for t in step(*r)) for r in runs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for r in runs:
            step(*r)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for r in runs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(*r))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for turn in range(4):
        for o in outs:
            for t in o:
                t.fill_(-1)
        torch.cuda.synchronize()
        for _ in range(5):
            for graph, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for o, w, r in zip(outs, want, runs):
            assert all(torch.equal(a, b) for a, b in zip(o[:5], w[:5]))
            # (Written for the assumed upstream value or again: a bf16 step of rounding.)
            a, b = o[5].float(), w[5].float()
            assert bool(((a - b).abs() <= 2.0 ** -7 * b.abs() + float(r[3]) / n * 2.0 ** -24).all())
        step(*runs[turn % 2])  # eager work between


def test_distilling_step(whole):
    """The step's loss and weight gradient against the same in 64 bits. The logits are
    fp32 products of 96 terms (sums off by 96 2^-24 of their terms' sizes, about 2^-24
    96 * 20 = 1e-4), the gradient's sums of B (K + 1) = 9 terms smaller still."""
    weight, teacher, x, *_, targets = _inputs()
    w = weight.double().requires_grad_(True)
    z = x.double().view(-1, H) @ w.t()
    t = (x.double().view(-1, H) @ teacher.double().t()) / 2.0
    ids = torch.from_numpy(whole["t_ids"]).view(-1, 20)
    p_all = torch.softmax(t, 1)
    p = p_all.gather(1, ids)
    q_all = torch.softmax(z / 2.0, 1)
    q = q_all.gather(1, ids)
    r, s = 1.0 - p.sum(1), 1.0 - q.sum(1)
    each = (p * (p.log() - q.log())).sum(1) + r * (r.log() - s.log())
    loss = 4.0 * each.mean() + torch.nn.functional.cross_entropy(z, targets.view(-1))
    loss.backward()
    assert np.abs(whole["loss_none"].ravel() - each.detach().numpy()).max() <= 1e-4
    assert abs(float(whole["loss_mean"]) - float(each.detach().mean())) <= 1e-4
    size = float(w.grad.abs().max())
    for name in ("mean", "none"):
        assert np.abs(whole[f"dw_{name}"] - w.grad.numpy()).max() <= 2e-4 * size


def _worker(rank: int, world: int, port: int, out_dir: str) -> None:
    os.environ["MASTER_ADDR"] = "127.0.0.1"
    os.environ["MASTER_PORT"] = str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        torch.cuda.set_device(0)
        import nmce
        ctx = nmce.ParallelContext(rank=rank, world_size=world, tp_size=world, tp_rank=rank,
                                   pp_size=1, pp_rank=0, dp_size=1, dp_rank=0)
        np.savez(os.path.join(out_dir, f"rank{rank}.npz"),
                 **_results(rank, ctx, torch.device(DEV)))
        print(f"[rank {rank}] done", flush=True)
    finally:
        dist.destroy_process_group()


def _free_port() -> int:
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        return s.getsockname()[1]


@pytest.fixture(scope="module", params=[2, 4], ids=["tp2", "tp4"])
def ranks(request, tmp_path_factory):
    world = request.param
    out = tmp_path_factory.mktemp(f"more_operators_tp{world}")
    mp.start_processes(_worker, args=(world, _free_port(), str(out)), nprocs=world, join=True,
                       start_method="spawn")
    return [dict(np.load(out / f"rank{r}.npz")) for r in range(world)]


def test_ranks_agree_with_one(ranks, whole):
    """Shards exactly (the logits are the same products), tokens and ids exactly; what is
    summed over the vocabulary, in another order over the ranks, within fp32's roundings of
    sums (2^-20 of a log-normaliser near 8, and of the gradient's largest)."""
    per = V // len(ranks)
    for r, res in enumerate(ranks):
        mine = slice(r * per, (r + 1) * per)
        for name in ("logits", "adjusted"):
            assert np.array_equal(res[name], whole[name][..., mine])
        for name in ("top_values", "top_ids", "tokens", "accepted"):
            assert np.array_equal(res[name], whole[name]), name
        assert np.array_equal(res["t_ids"], ranks[0]["t_ids"])
        for name in ("top_norm", "logprobs", "t_norm", "loss_mean", "loss_none", "t_values"):
            assert np.abs(res[name] - whole[name]).max() <= 2.0 ** -20 * 8, name
            assert np.array_equal(res[name], ranks[0][name]), name
        for name in ("dw_mean", "dw_none"):
            size = np.abs(whole[name]).max()
            assert np.abs(res[name] - whole[name][mine]).max() <= 2.0 ** -18 * size, name
