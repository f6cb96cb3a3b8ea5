"""The losses' saved tensors under saved-tensor hooks that hand back something else:
strides are taken as they come, another device, type or shape is refused before a
kernel is given the address."""

from __future__ import annotations

import contextlib

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF = torch.bfloat16
N, V, H = 37, 1000, 128

# node -> how many tensors it saves
NODES = {"one pass": 5, "one pass, in place": 3, "two passes": 3, "two passes, in place": 4,
         "per token": 3, "fused": 7, "fused, per token": 4}


class _Alias(torch.autograd.Function):
    @staticmethod
    def forward(ctx, anchor, buf):
        return buf.view_as(buf)

    @staticmethod
    def backward(ctx, grad):
        return torch.zeros(1, device=grad.device, dtype=grad.dtype), None


def _hooks(which, change):
    """The `which`-th saved tensor (None: every one) comes back as `change` makes it."""
    count = iter(range(99))

    def pack(t):
        return next(count), t

    def unpack(held):
        return change(held[1]) if which in (None, held[0]) else held[1]

    return torch.autograd.graph.saved_tensors_hooks(pack, unpack), count


def _loss(node, hooks):
    """(loss, its inputs, what their gradients leave in) of one node."""
    import nmce
    ctx = nmce.ParallelContext.single()
    g = torch.Generator(device=DEV).manual_seed(1)
    t = torch.randint(0, V, (N,), device=DEV, generator=g)
    hint = torch.ones(1, device=DEV)
    x = torch.randn(N, V, device=DEV, generator=g).to(BF)
    got = []
    if node.startswith("fused"):
        h = torch.randn(N, H, device=DEV, generator=g).to(BF).requires_grad_(True)
        w = (torch.randn(V, H, device=DEV, generator=g) * 0.1).to(BF).requires_grad_(True)
        for leaf in (h, w):
            leaf.register_hook(lambda d: got.append(d.clone()))
        with hooks:
            if node == "fused":
                loss = nmce.lmhead_vocab_parallel_cross_entropy(h, w, t, 0, V, ctx,
                                                                upstream_hint=hint)
            else:
                loss = nmce._LMHeadVocabParallelCrossEntropy.apply(h, w, t, 0, V, None, 1)
    else:
        inplace = node.endswith("in place")
        anchor = torch.zeros(1, device=DEV, dtype=BF, requires_grad=True)
        logits = _Alias.apply(anchor, x) if inplace else x.requires_grad_(True)
        logits.register_hook(lambda d: got.append(d.clone()))
        with hooks:
            if node == "per token":
                loss = nmce._VocabParallelCrossEntropy.apply(logits, t, 0, V, None, 1, False)
            else:
                loss = nmce.vocab_parallel_cross_entropy(
                    logits, t, 0, V, ctx, inplace=inplace, upstream_hint=hint,
                    one_pass=node.startswith("one pass"))
    return loss, got


@pytest.mark.parametrize("node", NODES)
def test_other_strides(node):
    want = _loss(node, contextlib.nullcontext())
    hooks, count = _hooks(None, lambda t: torch.stack([t, t], -1)[..., 0])
    got = _loss(node, hooks)
    for loss, _ in (want, got):
        (loss.sum() * 0.5).backward()
    assert next(count) == NODES[node]
    for a, b in zip(want[1], got[1]):
        assert b.abs().sum() > 0 and torch.equal(a, b)


@pytest.mark.parametrize("how", ["device", "type", "fewer", "more"])
@pytest.mark.parametrize("node,which", [(n, i) for n in NODES for i in range(NODES[n])])
def test_other_tensors_are_refused(node, which, how):
    change = {"device": lambda t: t.cpu(), "type": lambda t: t.to(torch.float64),
              "fewer": lambda t: t[:-1], "more": lambda t: torch.cat([t, t])}[how]
    print(f"[gpu] {node} tensor {which}: {how}", flush=True)
    loss, got = _loss(node, _hooks(which, change)[0])
    with pytest.raises(RuntimeError, match="nmce: saved-tensor hooks"):
        loss.sum().backward()
    assert not got
