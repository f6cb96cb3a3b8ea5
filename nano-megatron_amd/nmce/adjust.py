"""Penalties, biases and masks on vocabulary-sharded logits, on a gfx950 HIP kernel.

What stands between the serving head and the sampler
(:func:`~nmce.vocab_parallel_verify_drafts`). With ``count`` = how often an id is
among a sequence's output tokens (and, for the row after its first ``i`` drafts,
among those),

* an id of the prompt, or with ``count > 0``: ``x / r`` where ``x > 0``, else ``x r``
  (``repetition_penalty``);
* with ``count > 0``: ``x - f count - p`` (``frequency_penalty``, ``presence_penalty``);
* then its biases are added, and an id that is not allowed gets ``-inf``.

An element that any of this touches is formed in 64 bits and rounded once to the
logits' type; every other one is copied. The lists hold global ids, so every rank of a
tensor-parallel group passes the same ones beside its own shard; nothing is
exchanged. There is no derivative and no CPU path.
"""

from __future__ import annotations

import math

import torch

from . import _lib

MAX_BIASES = 8192  # of one sequence (NMCE_ADJUST_MAX_BIASES)


def _check_adjust(logits, vocab_start, vocab_end, ctx, prompt, output, drafts, penalties, bias_ids,
                  bias_values, allowed) -> None:
    if not logits.is_cuda:
        raise RuntimeError("nmce: logits must be on a ROCm device (there is no CPU path)")
    _lib.dtype_code(logits.dtype)
    if logits.dim() != 3 or logits.shape[1] == 0 or logits.shape[2] == 0:
        raise ValueError(f"nmce: logits must be [batch, drafts + 1, vocabulary], got "
                         f"{tuple(logits.shape)}")
    b, rows, v = logits.shape
    total = ctx.tp_size * v
    if vocab_end - vocab_start != v or vocab_start < 0 or vocab_end > total:
        raise ValueError(f"nmce: logits hold {v} vocabulary entries, which the shard "
                         f"[{vocab_start}, {vocab_end}) of {total} is not")
    if drafts is None and rows != 1:
        raise ValueError(f"nmce: {rows} rows a sequence need their {rows - 1} draft_tokens")
    if (bias_ids is None) != (bias_values is None):
        raise ValueError("nmce: bias_ids and bias_values come together")
    i64, f32 = torch.int64, torch.float32
    others = []
    if prompt is not None:
        others.append(("prompt_tokens", prompt, (b, None), i64))
    if output is not None:
        others.append(("output_tokens", output, (b, None), i64))
    if drafts is not None:
        others.append(("draft_tokens", drafts, (b, rows - 1), i64))
    if bias_ids is not None:
        others.append(("bias_ids", bias_ids, (b, None), i64))
        others.append(("bias_values", bias_values, tuple(bias_ids.shape), f32))
    if allowed is not None:
        others.append(("allowed", allowed, (b, rows, -(-total // 32)), torch.int32))
    for name, value in penalties:
        if hasattr(value, "dim"):
            others.append((name, value, (b,), f32))
        elif not math.isfinite(value) or (name == "repetition_penalty" and value <= 0.0):
            raise ValueError(f"nmce: {name} must be a finite number"
                             f"{' above 0' if name == 'repetition_penalty' else ''}, got {value}")
    for name, t, shape, dtype in others:
        if t.device != logits.device:
            raise RuntimeError(f"nmce: {name} on {t.device}, logits on {logits.device}")
        if t.dtype != dtype:
            raise TypeError(f"nmce: {name} must be {dtype}, got {t.dtype}")
        if t.dim() != len(shape) or any(n is not None and n != m
                                        for n, m in zip(shape, t.shape)):
            raise ValueError(f"nmce: {name} must be {shape}, got {tuple(t.shape)}")
        if dtype == f32:
            _lib.refuse_gradient(t, name, "adjusting logits has")
    if bias_ids is not None and bias_ids.shape[1] > MAX_BIASES:
        raise ValueError(f"nmce: {bias_ids.shape[1]} biases a sequence; at most {MAX_BIASES} are "
                         "taken (a denser bias is a sum of two tensors)")
    _lib.refuse_gradient(logits, "logits", "adjusting logits has")


def _overlaps_itself(t: torch.Tensor) -> bool:
    """Whether rows of ``t`` [batch, rows, columns] may share elements (an expanded
    tensor, or rows nearer to one another than they are long)."""
    need = t.shape[2]
    for size, stride in sorted(((t.shape[0], t.stride(0)), (t.shape[1], t.stride(1))),
                               key=lambda d: d[1]):
        if size > 1:
            if stride < need:
                return True
            need = (size - 1) * stride + need
    return False


def vocab_parallel_adjust_logits(
    logits: torch.Tensor,
    vocab_start: int,
    vocab_end: int,
    ctx,
    *,
    prompt_tokens: torch.Tensor | None = None,
    output_tokens: torch.Tensor | None = None,
    draft_tokens: torch.Tensor | None = None,
    repetition_penalty: float | torch.Tensor = 1.0,
    frequency_penalty: float | torch.Tensor = 0.0,
    presence_penalty: float | torch.Tensor = 0.0,
    bias_ids: torch.Tensor | None = None,
    bias_values: torch.Tensor | None = None,
    allowed: torch.Tensor | None = None,
    inplace: bool = False,
) -> torch.Tensor:
    """``logits`` under penalties, biases and a mask; the same shape and type.

    ``logits`` is ``[B, K + 1, V/tp]`` (fp32 or bf16, the vocabulary contiguous,
    other strides any): after each of ``K`` drafted tokens, and before the first
    (``K = 0``: the next token's). ``prompt_tokens`` ``[B, P]``, ``output_tokens``
    ``[B, L]``, ``draft_tokens`` ``[B, K]`` and ``bias_ids`` ``[B, N]`` are int64
    global ids; an id outside the vocabulary (-1, the padding of shorter lists)
    stands for none. Row ``i`` counts the first ``i`` drafts as output. Each penalty
    is a number or fp32 ``[B]`` (a repetition penalty that is not a finite number
    above 0 leaves that sequence as 1 would). ``bias_values`` is fp32 ``[B, N]``, at
    most 8192 a sequence; an id that comes several times gets them all, added in
    their order (the caller adds them up first where a sequence has more than 512 within
    8192 neighbouring ids: there one such id costs milliseconds). ``allowed`` is int32 ``[B, K + 1, ceil(V / 32)]`` (any strides of
    the first two): id ``j`` is allowed where bit ``j % 32`` of word ``j // 32`` is
    set. A masked element is ``-inf`` whatever it held; a row may have none left.

    ``inplace=True`` writes into ``logits`` and returns it: only the touched and
    the masked elements are written. Its rows must not overlap. A call takes up to 2^23
    slabs: ``B (K + 1) ceil(V / tp / 8192)``.
    """
    _check_adjust(logits, vocab_start, vocab_end, ctx, prompt_tokens, output_tokens, draft_tokens,
                  (("repetition_penalty", repetition_penalty),
                   ("frequency_penalty", frequency_penalty),
                   ("presence_penalty", presence_penalty)), bias_ids, bias_values, allowed)
    v = logits.shape[2]
    if inplace:
        if v > 1 and logits.stride(2) != 1:
            raise ValueError("nmce: logits that are written in place must have a contiguous "
                             "vocabulary")
        if _overlaps_itself(logits):
            raise ValueError("nmce: logits that are written in place must not overlap themselves")
    penalties = (repetition_penalty, frequency_penalty, presence_penalty)
    tensors = [isinstance(t, torch.Tensor) for t in penalties]
    return _lib.autograd_ext().adjust(
        logits, prompt_tokens, output_tokens, draft_tokens,
        [t if is_tensor else None for t, is_tensor in zip(penalties, tensors)],
        [0.0 if is_tensor else float(t) for t, is_tensor in zip(penalties, tensors)],
        bias_ids, bias_values, allowed, vocab_start, ctx.tp_size * v, inplace)
