"""The collectives on the embedding's output side over gloo, on CPU tensors: two
ranks, forward values and gradients against the sums they stand for."""

from __future__ import annotations

import os
import socket

import numpy as np
import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp


def _worker(rank: int, world: int, port: int, out_dir: str) -> None:
    os.environ["MASTER_ADDR"] = "127.0.0.1"
    os.environ["MASTER_PORT"] = str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        import nmce
        ctx = nmce.ParallelContext(rank=rank, world_size=world, tp_size=world, tp_rank=rank,
                                   pp_size=1, pp_rank=0, dp_size=1, dp_rank=0)
        g = torch.Generator().manual_seed(100 + rank)
        x = torch.randn(3, 4, 5, generator=g).requires_grad_(True)
        kept = x.detach().clone()
        up = torch.randn(3, 4, 5, generator=torch.Generator().manual_seed(7))
        y = nmce.reduce_from_tensor_parallel_region(x, ctx)
        (y * up).sum().backward()
        res = dict(x=kept.numpy(), y=y.detach().numpy(), dx=x.grad.numpy())
        assert torch.equal(x.detach(), kept)  # the input is left as it was
        x.grad = None
        z = nmce.reduce_scatter_to_sequence_parallel_region(x, ctx)
        (z * up[:, 2 * rank:2 * rank + 2]).sum().backward()
        res.update(z=z.detach().numpy(), dz=x.grad.numpy())
        with pytest.raises(ValueError, match="not divisible"):
            nmce.reduce_scatter_to_sequence_parallel_region(torch.zeros(2, 3, 4), ctx)
        np.savez(os.path.join(out_dir, f"rank{rank}.npz"), up=up.numpy(), **res)
    finally:
        dist.destroy_process_group()


def test_output_side_collectives(tmp_path):
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    mp.start_processes(_worker, args=(2, port, str(tmp_path)), nprocs=2, join=True,
                       start_method="spawn")
    ranks = [dict(np.load(tmp_path / f"rank{r}.npz")) for r in range(2)]
    total = ranks[0]["x"] + ranks[1]["x"]
    for r, res in enumerate(ranks):
        assert np.array_equal(res["y"], total)
        assert np.array_equal(res["dx"], res["up"])
        assert np.array_equal(res["z"], total[:, 2 * r:2 * r + 2])
        assert np.array_equal(res["dz"], res["up"])  # all-gathered back


def test_one_rank_is_the_identity():
    import nmce
    ctx = nmce.ParallelContext.single()
    x = torch.randn(2, 3, 4, requires_grad=True)
    for f in (nmce.reduce_from_tensor_parallel_region,
              nmce.reduce_scatter_to_sequence_parallel_region):
        y = f(x, ctx)
        assert torch.equal(y, x)
        g, = torch.autograd.grad(y, x, torch.ones_like(y))
        assert torch.equal(g, torch.ones_like(x))
    with pytest.raises(ValueError, match="at least 2 dims"):
        nmce.reduce_scatter_to_sequence_parallel_region(torch.zeros(3), ctx)


def _grad_worker(rank: int, world: int, port: int, out_dir: str) -> None:
    os.environ["MASTER_ADDR"] = "127.0.0.1"
    os.environ["MASTER_PORT"] = str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        import nmce
        ctx = nmce.ParallelContext(rank=rank, world_size=world, tp_size=world, tp_rank=rank,
                                   pp_size=1, pp_rank=0, dp_size=1, dp_rank=0)
        x = torch.randn(3, 4, generator=torch.Generator().manual_seed(1)).requires_grad_(True)
        u = torch.zeros(3, 4, requires_grad=True)
        dy = torch.randn(3, 4, generator=torch.Generator().manual_seed(300 + rank))
        kept = dy.clone()
        y = nmce.copy_to_tensor_parallel_region(x, ctx)
        first, = torch.autograd.grad(y, x, dy, retain_graph=True)
        again, = torch.autograd.grad(y, x, dy)
        assert torch.equal(dy, kept) and torch.equal(first, again)
        # a sum hands the same gradient to both of its inputs
        (nmce.copy_to_tensor_parallel_region(x, ctx) + u).backward(dy)
        assert torch.equal(dy, kept)
        np.savez(os.path.join(out_dir, f"rank{rank}.npz"), dy=kept.numpy(), first=first.numpy(),
                 du=u.grad.numpy(), dx=x.grad.numpy())
    finally:
        dist.destroy_process_group()


def test_the_copys_backward_leaves_the_incoming_gradient(tmp_path):
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    mp.start_processes(_grad_worker, args=(2, port, str(tmp_path)), nprocs=2, join=True,
                       start_method="spawn")
    ranks = [dict(np.load(tmp_path / f"rank{r}.npz")) for r in range(2)]
    total = ranks[0]["dy"] + ranks[1]["dy"]
    for res in ranks:
        assert np.array_equal(res["first"], total) and np.array_equal(res["dx"], total)
        assert np.array_equal(res["du"], res["dy"])


def _second_worker(rank: int, world: int, port: int, out_dir: str) -> None:
    os.environ["MASTER_ADDR"] = "127.0.0.1"
    os.environ["MASTER_PORT"] = str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        import nmce
        ctx = nmce.ParallelContext(rank=rank, world_size=world, tp_size=world, tp_rank=rank,
                                   pp_size=1, pp_rank=0, dp_size=1, dp_rank=0)
        own, same = torch.Generator().manual_seed(200 + rank), torch.Generator().manual_seed(9)

        def randn(g, cols):
            return torch.randn(3, cols, 5, generator=g).requires_grad_(True)

        res = {}
        # name: the mapping, columns in and out, whose numbers the input and the output are
        for name, cols, outs, gin, gout in (
                ("reduce_from_tensor_parallel_region", 4, 4, own, same),
                ("copy_to_tensor_parallel_region", 4, 4, same, own),
                ("reduce_scatter_to_sequence_parallel_region", 4, 2, own, own),
                ("gather_from_sequence_parallel_region", 2, 4, own, own)):
            x, dy, c = randn(gin, cols), randn(gout, outs), randn(gin, cols)
            y = getattr(nmce, name)(x, ctx)
            dx, = torch.autograd.grad(y, x, dy, create_graph=True)
            ddy, = torch.autograd.grad(dx, dy, c, create_graph=True)
            e = torch.randn(ddy.shape, generator=gout)
            dc, = torch.autograd.grad(ddy, c, e)  # and the third is the first's form again
            for key, t in (("dy", dy), ("dx", dx), ("c", c), ("ddy", ddy), ("e", e), ("dc", dc)):
                res[f"{name}_{key}"] = t.detach().numpy()
        np.savez(os.path.join(out_dir, f"rank{rank}.npz"), **res)
    finally:
        dist.destroy_process_group()


def test_second_derivatives_cross_the_ranks(tmp_path):
    """Each mapping's backward is its adjoint, and the derivative of that the mapping
    again: sums over the ranks of what they hold of their own, shards of the rest."""
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    mp.start_processes(_second_worker, args=(2, port, str(tmp_path)), nprocs=2, join=True,
                       start_method="spawn")
    ranks = [dict(np.load(tmp_path / f"rank{r}.npz")) for r in range(2)]

    def total(key):
        return ranks[0][key] + ranks[1][key]

    def joined(key):
        return np.concatenate([ranks[0][key], ranks[1][key]], 1)

    for r, res in enumerate(ranks):
        part = slice(2 * r, 2 * r + 2)
        g, f = "reduce_from_tensor_parallel_region_", "copy_to_tensor_parallel_region_"
        rs, ag = "reduce_scatter_to_sequence_parallel_region_", "gather_from_sequence_parallel_region_"
        for name, first, second in ((g, lambda k: res[k], total), (f, total, lambda k: res[k]),
                                    (rs, joined, lambda k: total(k)[:, part]),
                                    (ag, lambda k: total(k)[:, part], joined)):
            assert np.array_equal(res[name + "dx"], first(name + "dy")), name
            assert np.array_equal(res[name + "ddy"], second(name + "c")), name
            assert np.array_equal(res[name + "dc"], first(name + "e")), name
