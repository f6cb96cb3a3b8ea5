"""The largest logits of vocabulary-sharded rows, on gfx950 HIP kernels.

What a server returns as top log-probabilities, and what a teacher hands to a student
(:func:`~nmce.vocab_parallel_distillation_loss`): of every row the ``k`` largest logits
with their ids, in order, and ``log sum exp(x / T)`` over the whole vocabulary, so that
``values / T - log_normalizer`` are the log-probabilities. One read of the logits, no
sort of the row; the same inputs give the same bits at every run.

With ``tp_size > 1`` the ranks exchange ``8 (k + 1)`` bytes a row and no logits, and all
of them return the same. There is no derivative and no CPU path.
"""

from __future__ import annotations

import torch

from . import _lib
from .cross_entropy import _launch
from .embedding import _rows_of
from .mappings import _all_gather_rows

MAX_TOP = 512  # NMCE_TOP_MAX_K


def _check_top(logits, k, vocab_start, vocab_end, ctx, temperature) -> None:
    if not logits.is_cuda:
        raise RuntimeError("nmce: logits must be on a ROCm device (there is no CPU path)")
    _lib.dtype_code(logits.dtype)
    if logits.dim() == 0 or logits.shape[-1] == 0:
        raise ValueError(f"nmce: logits must be [..., vocabulary], got {tuple(logits.shape)}")
    v = logits.shape[-1]
    total = ctx.tp_size * v
    if vocab_end - vocab_start != v or vocab_start < 0 or vocab_end > total:
        raise ValueError(f"nmce: logits hold {v} vocabulary entries, which the shard "
                         f"[{vocab_start}, {vocab_end}) of {total} is not")
    if not 1 <= k <= min(MAX_TOP, total):
        raise ValueError(f"nmce: k must be from 1 to {min(MAX_TOP, total)} (at most {MAX_TOP}, and "
                         f"the vocabulary's {total}), got {k}")
    if not 1e-30 <= temperature <= 1e30:
        raise ValueError(f"nmce: temperature must be from 1e-30 to 1e30, got {temperature}")
    _lib.refuse_gradient(logits, "logits", "the top logits have")


def vocab_parallel_top_logits(
    logits: torch.Tensor,
    k: int,
    vocab_start: int,
    vocab_end: int,
    ctx,
    *,
    temperature: float = 1.0,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(values, ids, log_normalizer)`` of ``logits`` ``[..., V/tp]`` (fp32 or bf16).

    ``values`` ``[..., k]`` are the ``k`` largest logits (at most 512) in falling
    order, in the logits' type; ``ids`` ``[..., k]`` their global ids, int64, of
    equal logits the lowest first; ``log_normalizer`` ``[...]`` is the fp32
    ``log sum exp(x / temperature)``, temperatures from 1e-30 to 1e30. NaN counts as larger than +inf and makes the
    normaliser NaN; -inf is a logit like others (a masked row gives its lowest ids
    and the normaliser -inf); -0 comes back as 0.
    """
    _check_top(logits, k, vocab_start, vocab_end, ctx, temperature)
    temperature = float(temperature)
    tp = ctx.tp_size
    if tp == 1:
        return _lib.autograd_ext().top(logits, k, temperature)
    lib = _lib.load()
    dev = logits.device
    lead, v = tuple(logits.shape[:-1]), logits.shape[-1]
    values = torch.empty(lead + (k,), dtype=logits.dtype, device=dev)
    ids = torch.empty(lead + (k,), dtype=torch.int64, device=dev)
    norm = torch.empty(lead, dtype=torch.float32, device=dev)
    if logits.numel() == 0:
        return values, ids, norm
    rows, ld = _rows_of(logits)
    n = rows.shape[0]
    code = _lib.dtype_code(rows.dtype)
    ws = torch.empty(max(16, lib.nmce_top_workspace_bytes(n, v, k)), dtype=torch.uint8, device=dev)
    with torch.cuda.device(dev):
        stream = _lib.stream_handle(dev)
        part = torch.empty((1, n, k + 1), dtype=torch.int64, device=dev)
        _launch("nmce_top_logits", lib.nmce_top_logits, rows.data_ptr(), code, n, v, ld,
                vocab_start, k, temperature, part.data_ptr(), None, None, None, ws.data_ptr(),
                ws.numel(), stream)
        parts = _all_gather_rows(part, ctx.tp_group, tp)
        _launch("nmce_top_merge", lib.nmce_top_merge, parts.data_ptr(), tp, code, n, k,
                temperature, values.data_ptr(), ids.data_ptr(), norm.data_ptr(), stream)
    return values, ids, norm
