"""Embedding lookup over a vocabulary shard, and its gradient, on gfx950 HIP kernels.

The input end of the matrix whose output end is the LM head: nano_megatron's
``VocabParallelEmbedding`` (tp_layers.py:91-132) holds rows ``[start, end)`` of
the vocabulary, looks up the ids that are its own, leaves zero rows for the
others, and sums (or reduce-scatters, under sequence parallelism) over the
tensor-parallel group.

    out[i] = scale * W[t_i - start]            start <= t_i < end, else 0
    dW[v]  = scale * sum of dY[i] over t_i = start + v

The product with ``scale`` and the sum are fp32 and are rounded once, to the
output's and the weight's type. The gradient is the whole shard's, dense: rows
that no id names are zero. Positions are sorted by id on the GPU and added in a
fixed order, without atomics on values, so the same inputs give the same bits
at every run, however often an id is repeated.

The autograd node is C++ (``_nmce_autograd``): with a node in Python a training
step of 512 tokens took 128 us, the host's, where it takes 53.

There is no CPU path.
"""

from __future__ import annotations

import torch

from . import _lib
from .cross_entropy import launch_target_check
from .mappings import (reduce_from_tensor_parallel_region,
                       reduce_scatter_to_sequence_parallel_region)
from .parallel import divide


def _check_embedding(tokens, weight, vocab_start, vocab_end, out_dtype) -> None:
    if not weight.is_cuda:
        raise RuntimeError("nmce: the embedding weight must be on a ROCm device "
                           "(there is no CPU path)")
    if tokens.device != weight.device:
        raise RuntimeError(f"nmce: tokens on {tokens.device}, weight on {weight.device}")
    if tokens.dtype != torch.int64:
        raise TypeError(f"nmce: tokens must be int64, got {tokens.dtype}")
    _lib.dtype_code(weight.dtype)
    _lib.dtype_code(out_dtype)
    if weight.dim() != 2 or weight.shape[1] == 0:
        raise ValueError(f"nmce: the embedding weight must be [vocabulary, hidden], got "
                         f"{tuple(weight.shape)}")
    if weight.shape[0] != vocab_end - vocab_start or weight.shape[0] == 0:
        raise ValueError(f"nmce: weight holds {weight.shape[0]} vocabulary rows but the shard "
                         f"[{vocab_start}, {vocab_end}) has {vocab_end - vocab_start}")


def _rows_of(t: torch.Tensor) -> tuple[torch.Tensor, int]:
    """``[..., H]`` as rows of contiguous elements, and their stride. A copy
    only where they do not lie so (a transposed or an expanded tensor)."""
    h = t.shape[-1]
    rows = None
    if t.stride(-1) == 1 or h == 1:
        try:
            rows = t.view(-1, h)
        except RuntimeError:
            pass
    if rows is None or (rows.shape[0] > 1 and rows.stride(0) < h):
        rows = t.contiguous().view(-1, h)
    return rows, rows.stride(0) if rows.shape[0] > 1 else h


def vocab_parallel_embedding(
    tokens: torch.Tensor,
    weight: torch.Tensor,
    vocab_start: int,
    vocab_end: int,
    ctx,
    *,
    scale: float = 1.0,
    out_dtype: torch.dtype | None = None,
    sequence_parallel: bool = False,
    validate: bool = True,
) -> torch.Tensor:
    """``scale * weight[tokens - vocab_start]`` over a vocabulary-sharded ``weight``.

    ``tokens`` is int64 of any shape and strides, ``weight`` ``[V/tp, H]`` fp32
    or bf16 (rows of any stride); returns ``[..., H]`` in ``out_dtype`` (fp32
    or bf16; by default the weight's). With ``tp_size > 1`` the ranks' rows are
    summed over ``ctx.tp_group`` (exactly: one rank holds each id), or, with
    ``sequence_parallel``, reduce-scattered along dim 1 of ``[B, S, H]``. The
    backward gives the weight its dense gradient, in its own type.

    An id outside ``[0, tp_size * V/tp)`` raises ``ValueError``;
    ``validate=False`` skips that check, which waits on the host for one small
    kernel, and gives such an id a zero row and no gradient. (Under graph
    capture the check has to be off.)
    """
    out_dtype = weight.dtype if out_dtype is None else out_dtype
    _check_embedding(tokens, weight, vocab_start, vocab_end, out_dtype)
    if sequence_parallel and tokens.dim() < 2:
        raise ValueError("nmce: sequence-parallel tokens must be [batch, seq], got "
                         f"{tuple(tokens.shape)}")
    pending = None
    if validate:
        pending = launch_target_check(tokens, ctx.tp_size * (vocab_end - vocab_start))
    try:
        out = _lib.autograd_ext().embedding(weight, tokens, vocab_start, float(scale),
                                            out_dtype == torch.float32)
    finally:
        if pending is not None:
            pending.wait()
    if pending is not None and pending.bad:
        raise ValueError("token id is outside the model vocabulary")
    if ctx.tp_size == 1:
        return out
    if sequence_parallel:
        return reduce_scatter_to_sequence_parallel_region(out, ctx)
    return reduce_from_tensor_parallel_region(out, ctx)


class VocabParallelEmbedding(torch.nn.Module):
    """Vocabulary-sharded embedding (tp_layers.py:91-132) on the HIP lookup.

    Takes ``FusedParallelLMHead``'s constructor arguments: ``config.vocab_size``,
    ``config.n_embd`` and ``config.sequence_parallel``, and has its weight
    (``[V/tp, n_embd]``, N(0, 0.02^2), ``tensor_parallel_sharded``), so that
    ``lm_head.weight = embedding.weight`` ties the two (model.py:235-236).
    ``forward(tokens, out_dtype=None)`` returns the scaled rows.
    """

    def __init__(self, config, ctx, scale: float = 1.0):
        super().__init__()
        self.ctx = ctx
        self.scale = float(scale)
        self.weight = torch.nn.Parameter(
            torch.empty(divide(config.vocab_size, ctx.tp_size), config.n_embd))
        self.weight.tensor_parallel_sharded = True
        self.sequence_parallel = bool(getattr(config, "sequence_parallel", False))
        self.validate = True
        torch.nn.init.normal_(self.weight, std=0.02)

    def vocab_range(self) -> tuple[int, int]:
        """This rank's global id range (model.py:242-245)."""
        per = self.weight.shape[0]
        return self.ctx.tp_rank * per, (self.ctx.tp_rank + 1) * per

    def forward(self, tokens: torch.Tensor, out_dtype: torch.dtype | None = None) -> torch.Tensor:
        start, end = self.vocab_range()
        return vocab_parallel_embedding(tokens, self.weight, start, end, self.ctx,
                                        scale=self.scale, out_dtype=out_dtype,
                                        sequence_parallel=self.sequence_parallel,
                                        validate=self.validate)
