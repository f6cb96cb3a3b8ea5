"""Which calls share the upstream value that a one-pass forward assumes."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def test_losses_on_one_line_keep_their_own():
    """Two losses of one line, weighted differently: each call's next forward assumes what its
    own backward received, not the other's."""
    import nmce
    from nmce import cross_entropy
    ctx = nmce.ParallelContext.single()
    n, v = 8, 4000
    g = torch.Generator().manual_seed(1)
    leaf = torch.randn(n, v, generator=g).to(DEV).requires_grad_(True)
    target = torch.randint(0, v, (n,), generator=g).to(DEV)
    values, ids = torch.topk(torch.randn(n, v, generator=g), 16)
    values, ids = values.to(DEV), ids.to(DEV)
    before = set(cross_entropy._upstream_hints)
    for _ in range(2):
        both = (0.25, nmce.vocab_parallel_cross_entropy(leaf, target, 0, v, ctx)), (4.0, nmce.vocab_parallel_distillation_loss(leaf, values, ids, 0, v, ctx))  # noqa: E501
        sum(a * loss for a, loss in both).backward()
    hints = [t for key, t in cross_entropy._upstream_hints.items() if key not in before]
    assert sorted(float(t) for t in hints) == [0.25, 4.0]
