"""The embedding, the 8-bit head and the draft verification under tensor
parallelism: two or four ranks share cuda:0 and talk over gloo (host copies).

Every rank must return what one rank returns on the whole vocabulary: the
embedding's rows exactly (each id is one rank's), its gradient shard exactly
the matching rows (the order of a row's sum depends on its positions in the
sorted list, so compared within the sums' rounding), the logits exactly the
matching columns, and the verification's tokens and counts exactly; its
log-probabilities within one rounding of fp32 (sums over slabs are merged in
another order)."""

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

B, S, H, V, K = 4, 12, 96, 4 * 9000, 3


def _inputs():
    g = torch.Generator().manual_seed(21)
    weight = torch.randn(V, H, generator=g) * 0.1
    tokens = torch.randint(0, V, (B, S), generator=g)
    grad = torch.randn(B, S, H, generator=g)
    x = torch.randn(B, K + 1, H, generator=g)
    target = torch.randn(B, K + 1, V, generator=g) * 2.0
    draft = target[:, :K] + 0.3 * torch.randn(B, K, V, generator=g)
    drafted = draft.argmax(-1)
    drafted[1, 2], drafted[2, 0] = -1, 5
    u = torch.rand(B, K, generator=g), torch.rand(B, generator=g)
    return weight, tokens, grad, x, target, draft, drafted, u


def _temperatures():
    return torch.tensor([1.0, 0.5, 2.0, 0.0])


def _results(rank, ctx, dev):
    """Every operator's outputs on this rank's shard."""
    import nmce
    weight, tokens, grad, x, target, draft, drafted, u = _inputs()
    per = V // ctx.tp_size
    lo, hi = rank * per, (rank + 1) * per
    res = {}
    t = tokens.to(dev)
    for sp in (False, True):
        cfg = types.SimpleNamespace(vocab_size=V, n_embd=H, sequence_parallel=sp)
        emb = nmce.VocabParallelEmbedding(cfg, ctx, scale=3.0)
        emb.weight = torch.nn.Parameter(weight[lo:hi].to(dev))
        out = emb(t)
        part = S // ctx.tp_size
        g = grad[:, rank * part:(rank + 1) * part] if sp else grad
        out.backward(g.to(dev))
        tag = "sp" if sp else "tp"
        res[f"{tag}_out"], res[f"{tag}_dw"] = out.detach(), emb.weight.grad
    cfg = types.SimpleNamespace(vocab_size=V, n_embd=H, sequence_parallel=False)
    head = nmce.FusedParallelLMHead(cfg, ctx)
    head.weight = torch.nn.Parameter(weight[lo:hi].to(dev))
    with torch.no_grad():
        res["logits"] = head.quantized()(x.to(dev))
    for name, y in (("model", draft[..., lo:hi].to(dev)), ("copied", None)):
        out = nmce.vocab_parallel_verify_drafts(
            target[..., lo:hi].to(dev), drafted.to(dev), y, u[0].to(dev), u[1].to(dev), lo, hi,
            ctx, temperature=_temperatures().to(dev))
        for part, value in zip(("tokens", "accepted", "logprobs"), out):
            res[f"{name}_{part}"] = value
    torch.cuda.synchronize()
    return {k: v.cpu().numpy() for k, v in res.items()}


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
                 **_results(rank, ctx, torch.device("cuda:0")))
        print(f"[rank {rank}] done", flush=True)
    finally:
        dist.destroy_process_group()


def _free_port() -> int:
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        return s.getsockname()[1]


@pytest.fixture(scope="module", params=[2, 4], ids=["tp2", "tp4"])
def ranks(request, tmp_path_factory):
    assert torch.cuda.is_available(), "GPU tests need a ROCm device"
    world = request.param
    out = tmp_path_factory.mktemp(f"operators_tp{world}")
    mp.start_processes(_worker, args=(world, _free_port(), str(out)), nprocs=world, join=True,
                       start_method="spawn")
    return [dict(np.load(out / f"rank{r}.npz")) for r in range(world)]


@pytest.fixture(scope="module")
def whole():
    import nmce
    return _results(0, nmce.ParallelContext.single(), torch.device("cuda:0"))


def test_embedding_ranks(ranks, whole):
    world = len(ranks)
    per, part = V // world, S // world
    counts = np.bincount(_inputs()[1].numpy().ravel(), minlength=V)
    for r, res in enumerate(ranks):
        assert np.array_equal(res["tp_out"], whole["tp_out"])
        assert np.array_equal(res["sp_out"], whole["tp_out"][:, r * part:(r + 1) * part])
        for tag in ("tp", "sp"):
            want = whole["tp_dw"][r * per:(r + 1) * per]
            # each id comes a few times: two sums of m terms of size up to 5 * 3
            slack = 2 * counts[r * per:(r + 1) * per, None].astype(float) ** 2 * 15 * 2.0 ** -24
            assert np.all(np.abs(res[f"{tag}_dw"] - want) <= slack)


def test_head_ranks(ranks, whole):
    per = V // len(ranks)
    for r, res in enumerate(ranks):
        assert np.array_equal(res["logits"], whole["logits"][..., r * per:(r + 1) * per])


@pytest.mark.parametrize("drafts", ["model", "copied"])
def test_verification_ranks(ranks, whole, drafts):
    assert whole[f"{drafts}_accepted"].sum() > 0
    for res in ranks:
        for part in ("tokens", "accepted"):
            assert np.array_equal(res[f"{drafts}_{part}"], whole[f"{drafts}_{part}"])
        a, b = res[f"{drafts}_logprobs"], whole[f"{drafts}_logprobs"]
        assert np.all(np.abs(a - b) <= np.abs(b) * 2.0 ** -23 + 1e-12)


def _second(rank, ctx, dev):
    """The embedding's second derivatives on this rank's shard: d<dW, C> / d(dY)."""
    import nmce
    weight, tokens, grad, *_ = _inputs()
    c = torch.randn(V, H, generator=torch.Generator().manual_seed(22))
    per = V // ctx.tp_size
    lo, hi = rank * per, (rank + 1) * per
    res = {}
    for sp in (False, True):
        w = weight[lo:hi].to(dev).requires_grad_(True)
        out = nmce.vocab_parallel_embedding(tokens.to(dev), w, lo, hi, ctx, scale=3.0,
                                            sequence_parallel=sp)
        part = S // ctx.tp_size
        dy = grad[:, rank * part:(rank + 1) * part] if sp else grad
        dy = dy.to(dev).requires_grad_(True)
        dw, = torch.autograd.grad(out, w, dy, create_graph=True)
        ddy, = torch.autograd.grad(dw, dy, c[lo:hi].to(dev))
        res["sp" if sp else "tp"] = ddy.cpu().numpy()
    return res


def _second_worker(rank: int, world: int, port: int, out_dir: str) -> None:
    os.environ["MASTER_ADDR"] = "127.0.0.1"
    os.environ["MASTER_PORT"] = str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        torch.cuda.set_device(0)
        import nmce
        ctx = nmce.ParallelContext(rank=rank, world_size=world, tp_size=world, tp_rank=rank,
                                   pp_size=1, pp_rank=0, dp_size=1, dp_rank=0)
        np.savez(os.path.join(out_dir, f"rank{rank}.npz"),
                 **_second(rank, ctx, torch.device("cuda:0")))
        print(f"[rank {rank}] done", flush=True)
    finally:
        dist.destroy_process_group()


def test_embeddings_second_derivatives_cross_the_ranks(tmp_path):
    import nmce
    world = 2
    mp.start_processes(_second_worker, args=(world, _free_port(), str(tmp_path)), nprocs=world,
                       join=True, start_method="spawn")
    ranks = [dict(np.load(tmp_path / f"rank{r}.npz")) for r in range(world)]
    whole = _second(0, nmce.ParallelContext.single(), torch.device("cuda:0"))
    part = S // world
    for r, res in enumerate(ranks):
        assert np.array_equal(res["tp"], whole["tp"])
        assert np.array_equal(res["sp"], whole["tp"][:, r * part:(r + 1) * part])
