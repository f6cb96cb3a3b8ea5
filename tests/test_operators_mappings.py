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
