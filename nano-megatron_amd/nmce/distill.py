"""Distillation from a teacher's top logits over vocabulary-sharded logits, on gfx950
HIP kernels.

The student's ``q = softmax(z / T)`` is over the whole vocabulary; of the teacher, ``K``
logits ``t`` a token are at hand, at listed ids (what
:func:`~nmce.vocab_parallel_top_logits` keeps of a teacher's row). With its
log-normaliser, ``p = exp(t / T - log_normalizer)`` and ``r = 1 - sum p`` is the rest's
probability, one class more; without, ``p = softmax(t / T)`` over the list and ``r = 0``:

    loss = sum p (log p - log q) + r (log r - log s),   s = sum of q outside the list

the Kullback-Leibler divergence, whose gradient is ``(q - p) / T`` at the list's ids and
``(q - r q / s) / T`` outside. The logits are not upcast, and nothing of their size is
kept but themselves; the teacher's few values are worked on in 64 bits. With
``tp_size > 1`` the ranks exchange 40 bytes a token.

There is no CPU path.
"""

from __future__ import annotations

import ctypes
import sys

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .cross_entropy import (_as_rows, _check_hint, _grad_operand, _launch, _one_pass_ragged,
                            _one_pass_rows, _resolve_inplace, _save, _site_hint, _take)
from .embedding import _rows_of
from .mappings import _all_gather_rows

MAX_LISTED = 1024  # NMCE_DISTILL_MAX_K


def _check_distillation(logits, teacher_logits, teacher_ids, normalizer, vocab_start, vocab_end,
                        ctx, temperature, reduction) -> None:
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
    lead = tuple(logits.shape[:-1])
    if teacher_logits.dim() == 0 or tuple(teacher_logits.shape[:-1]) != lead:
        raise ValueError(f"nmce: teacher_logits {tuple(teacher_logits.shape)} are not a list for "
                         f"each of the tokens {lead}")
    k = teacher_logits.shape[-1]
    if not 1 <= k <= MAX_LISTED:
        raise ValueError(f"nmce: a teacher lists from 1 to {MAX_LISTED} logits a token, got {k}")
    if teacher_logits.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"nmce: teacher_logits must be float32 or bfloat16, got "
                        f"{teacher_logits.dtype}")
    others = [("teacher_logits", teacher_logits, lead + (k,), teacher_logits.dtype),
              ("teacher_ids", teacher_ids, lead + (k,), torch.int64)]
    if normalizer is not None:
        others.append(("teacher_log_normalizer", normalizer, lead, torch.float32))
    for name, t, shape, dtype in others:
        if t.device != logits.device:
            raise RuntimeError(f"nmce: {name} on {t.device}, logits on {logits.device}")
        if t.dtype != dtype:
            raise TypeError(f"nmce: {name} must be {dtype}, got {t.dtype}")
        if tuple(t.shape) != shape:
            raise ValueError(f"nmce: {name} must be {shape}, got {tuple(t.shape)}")
        if dtype != torch.int64:
            _lib.refuse_gradient(t, name, "the distillation loss has towards its teacher")
    if not 1e-6 <= temperature <= 1e6:
        raise ValueError(f"nmce: temperature must be from 1e-6 to 1e6, got {temperature}")
    if reduction not in ("mean", "none"):
        raise ValueError(f"nmce: reduction must be 'mean' or 'none', got {reduction!r}")


def _teacher(rows, ld, teacher_logits, teacher_ids, normalizer, vocab_start, total, temperature):
    """``(batch, what it points into)`` for the C entries."""
    t, t_ld = _rows_of(teacher_logits)
    ids, ids_ld = _rows_of(teacher_ids)
    norm = normalizer.reshape(-1).contiguous() if normalizer is not None else None
    n, v = rows.shape
    batch = _lib.DistillBatch(
        rows.data_ptr(), t.data_ptr(), ids.data_ptr(),
        norm.data_ptr() if norm is not None else None, ld, t_ld, ids_ld, n, v, vocab_start, total,
        temperature, t.shape[1], _lib.dtype_code(rows.dtype), _lib.dtype_code(t.dtype))
    return batch, (t, ids, norm)


class _VocabParallelDistillation(torch.autograd.Function):
    """Per-token loss (``mean`` False) or its mean over several ranks' shards, by two
    passes: statistics of the logits in the forward, exchanged, and their gradient from
    the logits in the backward. (One rank's nodes are C++, ``_nmce_autograd.distill`` and
    ``distill_mean``: in Python a step of 4 tokens took 135 us on the host.)"""

    @staticmethod
    def forward(ctx, logits, teacher_logits, teacher_ids, normalizer, vocab_start, group,
                world_size, temperature, mean, inplace):
        lib = _lib.load()
        dev = logits.device
        v = logits.shape[-1]
        n = logits.numel() // v
        k = teacher_logits.shape[-1]
        rows = _as_rows(logits) if n else logits.reshape(0, v)
        inplace = _resolve_inplace(logits, bool(inplace))
        if rows is None or (n > 1 and rows.stride(0) < v):
            rows, inplace = logits.contiguous().view(-1, v), False
        ld = rows.stride(0) if n > 1 else v
        loss = torch.empty((n,), dtype=torch.float32, device=dev)
        result = torch.empty((), dtype=torch.float32, device=dev) if mean and n else None
        size = int(lib.nmce_distill_state_bytes(n, k))
        state = torch.empty(max(16, size), dtype=torch.uint8, device=dev)
        if n:
            batch, held = _teacher(rows, ld, teacher_logits, teacher_ids, normalizer, vocab_start,
                                   world_size * v, temperature)
            stats = torch.empty((1, n, 5), dtype=torch.float64, device=dev)
            with torch.cuda.device(dev):
                stream = _lib.stream_handle(dev)
                _launch("nmce_distill_stats", lib.nmce_distill_stats, ctypes.addressof(batch),
                        state.data_ptr(), state.numel(), stats.data_ptr(), stream)
                if world_size > 1:
                    stats = _all_gather_rows(stats, group, world_size)
                _launch("nmce_distill_combine", lib.nmce_distill_combine, state.data_ptr(),
                        state.numel(), n, k, temperature, stats.data_ptr(), world_size,
                        loss.data_ptr(), result.data_ptr() if mean else None, stream)
            del held
        ctx.inplace, ctx.k, ctx.temperature, ctx.mean = inplace, k, temperature, mean
        ctx.shape = logits.shape
        _save(ctx, rows, state, logits if inplace else None)
        if mean:
            return result if n else loss.mean()  # (of no tokens: NaN)
        return loss.view(logits.shape[:-1])

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output):
        (rows, state, original), _ = _take(ctx)
        lib = _lib.load()
        n, v = rows.shape
        state = state.contiguous()
        if v > 1 and rows.stride(1) != 1:  # (what saved-tensor hooks handed back)
            rows = rows.contiguous()
        ld = rows.stride(0) if n > 1 else v
        out = _as_rows(original) if ctx.inplace and n else None
        if ctx.inplace and out is None:
            original = original.contiguous()
            out = original.view(n, v)
        if out is None:
            out = torch.empty((n, v), dtype=rows.dtype, device=rows.device)
        if ctx.mean:
            go, stride = grad_output.reshape(1).float(), 0
        else:
            go, stride = _grad_operand(grad_output)
        with torch.cuda.device(rows.device):
            _launch("nmce_distill_bwd", lib.nmce_distill_bwd, rows.data_ptr(), out.data_ptr(),
                    _lib.dtype_code(rows.dtype), n, v, ld, out.stride(0) if n > 1 else v, ctx.k,
                    ctx.temperature, state.data_ptr(), state.numel(), go.data_ptr(), stride,
                    float(max(n, 1)) if ctx.mean else 1.0, None, None,
                    _lib.stream_handle(rows.device))
        if ctx.inplace:
            # The logits hold the gradient: readers that saved them fail their version check.
            torch.autograd.graph.increment_version(original)
            grad = original.detach()
        else:
            grad = out.view(ctx.shape)
        return (grad,) + (None,) * 9


def vocab_parallel_distillation_loss(
    logits: torch.Tensor,
    teacher_logits: torch.Tensor,
    teacher_ids: torch.Tensor,
    vocab_start: int,
    vocab_end: int,
    ctx,
    *,
    teacher_log_normalizer: torch.Tensor | None = None,
    temperature: float = 1.0,
    reduction: str = "mean",
    inplace: bool = False,
    one_pass: bool = True,
    upstream_hint: torch.Tensor | None = None,
) -> torch.Tensor:
    """The divergence of the student's ``logits`` from a teacher's top logits.

    ``logits`` is ``[..., V/tp]`` (fp32 or bf16); ``teacher_logits`` ``[..., K]``
    (fp32 or bf16, at most 1024 a token) and ``teacher_ids`` ``[..., K]`` (int64
    global ids) are replicated over the tensor-parallel group. With
    ``teacher_log_normalizer`` ``[...]`` (fp32, ``log sum exp(t / temperature)`` of the
    teacher's whole row) the rest of the vocabulary is one class more. Returns the
    fp32 mean over all tokens, or with ``reduction="none"`` each token's loss
    ``[...]``. The usual factor ``temperature ** 2`` is the caller's.

    Shorter lists are padded with -1: an id outside the vocabulary stands for
    nothing. A token without a teacher (nothing else in its list, a normaliser of -inf, or
    without one only -inf) has loss and gradient 0, and counts in the mean. An id
    that comes several times adds up its probabilities. Where the student gives
    everything outside the list nothing (-inf), the rest has no term; a student's row
    of only -inf, or with a +inf or NaN, gives NaN.

    ``inplace=True`` writes the gradient into the logits' storage (they must not be a
    leaf, and nothing else may read them afterwards: not once this returns, on the
    one-pass path, whose backward cannot run twice then). Beside a cross entropy of the same
    logits neither may write in place: give that one ``inplace=False``. The teacher's
    tensors may not require grad; the loss cannot be differentiated twice.

    The mean at TP = 1, of rows of at most 131072 bf16 or 65536 fp32 columns, reads
    the logits once where a gradient is wanted: as in
    :func:`~nmce.vocab_parallel_cross_entropy` its forward also writes the gradient, for
    the upstream value that this call site's last backward received (``upstream_hint``
    replaces it), which another value makes the backward write again (in place: scale).
    ``one_pass=False`` writes it in the backward alone.
    """
    _check_distillation(logits, teacher_logits, teacher_ids, teacher_log_normalizer, vocab_start,
                        vocab_end, ctx, temperature, reduction)
    temperature = float(temperature)
    mean, inplace, tp = reduction == "mean", bool(inplace), ctx.tp_size
    if tp > 1:
        return _VocabParallelDistillation.apply(
            logits, teacher_logits, teacher_ids, teacher_log_normalizer, vocab_start,
            ctx.tp_group, tp, temperature, mean, inplace)
    inplace = _resolve_inplace(logits, inplace)
    ext = _lib.autograd_ext()
    if (mean and one_pass and torch.is_grad_enabled() and logits.requires_grad
            and (_one_pass_rows(logits, tp) is not None
                 or _one_pass_ragged(logits, tp, inplace))):
        if upstream_hint is None:
            caller = sys._getframe(1)
            # (Named: a cross entropy on the same line may have another upstream value.)
            hint = _site_hint(logits.device,
                              (caller.f_code.co_filename, caller.f_lineno, "distillation"))
        else:
            _check_hint(upstream_hint, logits.device)
            hint = upstream_hint
        return ext.distill_mean(logits, teacher_logits, teacher_ids, teacher_log_normalizer,
                                hint, temperature, inplace)
    return ext.distill(logits, teacher_logits, teacher_ids, teacher_log_normalizer, temperature,
                       mean, inplace)
