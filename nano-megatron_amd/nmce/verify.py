"""Verification of drafted tokens over vocabulary-sharded logits, on gfx950 HIP kernels.

Serving with a draft model: it proposes a few tokens, the target model's logits
at all of their positions come from one pass, and this decides from given
uniform numbers how many of them stand and which token follows, so that the
tokens are distributed as if the target model alone had drawn them. With
``p = softmax(target / T)`` and ``q = softmax(draft / T)`` at a position,

* the drafted token ``d`` stands while ``u q(d) < p(d)``;
* at the first that does not, the next token is drawn from ``max(p - q, 0)``: the
  first id whose running sum passes ``u'`` times all of it;
* after the last draft it is drawn from ``p`` (with no drafts at all: sampling).

The weights and sums are 64 bits wide, so that a token near the border of its
interval is the one that exact arithmetic gives. With ``tp_size > 1`` the ranks
exchange the statistics of their slabs of the vocabulary and no logits, and all
of them return the same tokens.

There is no CPU path.
"""

from __future__ import annotations

import ctypes

import torch
import torch.distributed as dist

from . import _lib
from .cross_entropy import _launch
from .mappings import _all_gather_rows, _use_host


def _check_verify(target, tokens, draft, accept_u, sample_u, vocab_start, vocab_end, ctx,
                  temperature) -> None:
    if not target.is_cuda:
        raise RuntimeError("nmce: target_logits must be on a ROCm device (there is no CPU path)")
    _lib.dtype_code(target.dtype)
    if target.dim() != 3 or target.shape[1] == 0 or target.shape[2] == 0:
        raise ValueError(f"nmce: target_logits must be [batch, drafts + 1, vocabulary], got "
                         f"{tuple(target.shape)}")
    b, rows, v = target.shape
    k = rows - 1
    if vocab_end - vocab_start != v or vocab_start < 0:
        raise ValueError(f"nmce: logits hold {v} vocabulary entries but the shard "
                         f"[{vocab_start}, {vocab_end}) has {vocab_end - vocab_start}")
    # The running sums go over the shards in the order of their ranks.
    rank = ctx.tp_rank if ctx.tp_size > 1 else 0
    if vocab_start != rank * v:
        raise ValueError(f"nmce: the shard [{vocab_start}, {vocab_end}) is not rank {rank}'s of "
                         f"the {ctx.tp_size * v} entries of {ctx.tp_size} shards")
    others = [("draft_tokens", tokens, (b, k), torch.int64),
              ("accept_uniform", accept_u, (b, k), torch.float32),
              ("sample_uniform", sample_u, (b,), torch.float32)]
    if draft is not None:
        others.append(("draft_logits", draft, (b, k, v), target.dtype))
    if isinstance(temperature, torch.Tensor):
        others.append(("temperature", temperature, (b,), torch.float32))
    elif not temperature >= 0.0:
        raise ValueError(f"nmce: temperature must not be negative, got {temperature}")
    for name, t, shape, dtype in others:
        if t.device != target.device:
            raise RuntimeError(f"nmce: {name} on {t.device}, target_logits on {target.device}")
        if t.dtype != dtype:
            raise TypeError(f"nmce: {name} must be {dtype}, got {t.dtype}")
        if tuple(t.shape) != shape:
            raise ValueError(f"nmce: {name} must be {shape}, got {tuple(t.shape)}")
    # (What the log-probabilities depend on smoothly, and the draft's logits.)
    for name, t in (("target_logits", target), ("draft_logits", draft),
                    ("temperature", temperature)):
        if isinstance(t, torch.Tensor):
            _lib.refuse_gradient(t, name, "verification has")


def vocab_parallel_verify_drafts(
    target_logits: torch.Tensor,
    draft_tokens: torch.Tensor,
    draft_logits: torch.Tensor | None,
    accept_uniform: torch.Tensor,
    sample_uniform: torch.Tensor,
    vocab_start: int,
    vocab_end: int,
    ctx,
    *,
    temperature: float | torch.Tensor = 1.0,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(tokens, accepted, logprobs)`` of ``K`` drafted tokens a sequence.

    ``target_logits`` is ``[B, K + 1, V/tp]`` (fp32 or bf16, the vocabulary
    contiguous, other strides any): the target model's after each drafted token,
    and before the first. ``draft_tokens`` is ``[B, K]`` of global ids;
    ``draft_logits`` ``[B, K, V/tp]``, what they were drawn from at the same
    temperature, or None (copied drafts: ``q`` is one at the drafted token).
    ``accept_uniform`` ``[B, K]`` and ``sample_uniform`` ``[B]`` are fp32 in
    ``[0, 1)``. ``temperature`` is a number (64 bits) or fp32 ``[B]``; 0 is greedy (so is
    what a tensor holds that is not above 0, NaN among it): a draft stands where
    it is the largest logit (the lowest id of equal ones), which is also the next
    token.

    ``tokens`` ``[B, K + 1]`` holds the drafts that stand, the next token, and -1
    behind it; ``accepted`` ``[B]`` how many stand; ``logprobs`` ``[B, K + 1]``
    fp32 the log-probability under ``p`` of each token (at temperature 1 where it
    is 0), 0 behind.

    Shorter drafts are padded with -1: an id outside the vocabulary ends its
    sequence's drafts, and the next token comes from ``p`` there. A draft row
    that is no distribution (only -inf, or an infinity or NaN) refuses its
    token, and the next comes from ``p``; such a target row gives the next token
    -1. A number outside ``[0, 1)`` is taken as the nearest inside, NaN as 0.
    Ranks of a tensor-parallel group must be given the same numbers and tokens, and
    each the shard of its rank, ``vocab_start = tp_rank * V/tp``.
    """
    _check_verify(target_logits, draft_tokens, draft_logits, accept_uniform, sample_uniform,
                  vocab_start, vocab_end, ctx, temperature)
    b, rows, v = target_logits.shape
    lib = _lib.load()
    dev = target_logits.device
    k = rows - 1
    tokens = torch.empty((b, k + 1), dtype=torch.int64, device=dev)
    accepted = torch.empty((b,), dtype=torch.int64, device=dev)
    logprobs = torch.empty((b, k + 1), dtype=torch.float32, device=dev)
    if b == 0:
        return tokens, accepted, logprobs
    x = target_logits if target_logits.stride(2) == 1 or v == 1 else target_logits.contiguous()
    y = draft_logits if k else None
    if y is not None and y.stride(2) != 1 and v != 1:
        y = y.contiguous()
    ids, au, su = draft_tokens.contiguous(), accept_uniform.contiguous(), \
        sample_uniform.contiguous()
    heat = temperature.contiguous() if isinstance(temperature, torch.Tensor) else None
    batch = _lib.VerifyBatch(
        x.data_ptr(), y.data_ptr() if y is not None else None, ids.data_ptr(), au.data_ptr(),
        su.data_ptr(), heat.data_ptr() if heat is not None else None,
        x.stride(0), x.stride(1), y.stride(0) if y is not None else 0,
        y.stride(1) if y is not None else 0, b, k, v, vocab_start, ctx.tp_size * v,
        1.0 if heat is not None else float(temperature), _lib.dtype_code(x.dtype))
    slabs = int(lib.nmce_verify_slabs(v))
    n = b * (k + 1) + (b * k if y is not None else 0)
    tp = ctx.tp_size
    stats = torch.empty((1, n, slabs, 4), dtype=torch.float64, device=dev)
    masses = torch.empty((1, b, slabs, 2), dtype=torch.float64, device=dev)
    ws = torch.empty(max(16, int(lib.nmce_verify_workspace_bytes(b))), dtype=torch.uint8,
                     device=dev)
    arg = ctypes.addressof(batch)
    out = tokens.data_ptr(), logprobs.data_ptr()
    with torch.cuda.device(dev):
        stream = _lib.stream_handle(dev)
        _launch("nmce_verify_stats", lib.nmce_verify_stats, arg, stats.data_ptr(), stream)
        if tp > 1:
            stats = _all_gather_rows(stats, ctx.tp_group, tp)
        _launch("nmce_verify_masses", lib.nmce_verify_masses, arg, stats.data_ptr(), tp,
                masses.data_ptr(), tokens.data_ptr(), accepted.data_ptr(), logprobs.data_ptr(),
                ws.data_ptr(), ws.numel(), stream)
        if tp == 1:
            _launch("nmce_verify_pick", lib.nmce_verify_pick, arg, masses.data_ptr(), 1, 0,
                    ws.data_ptr(), ws.numel(), *out, None, stream)
            return tokens, accepted, logprobs
        masses = _all_gather_rows(masses, ctx.tp_group, tp)
        picked = torch.empty((b, 2), dtype=torch.float64, device=dev)
        _launch("nmce_verify_pick", lib.nmce_verify_pick, arg, masses.data_ptr(), tp,
                ctx.tp_rank, ws.data_ptr(), ws.numel(), *out, picked.data_ptr(), stream)
        picked = _all_reduce_max(picked, ctx.tp_group)
        _launch("nmce_verify_finish", lib.nmce_verify_finish, picked.data_ptr(), ws.data_ptr(),
                ws.numel(), b, k, *out, stream)
    return tokens, accepted, logprobs


def _all_reduce_max(t: torch.Tensor, group) -> torch.Tensor:
    if _use_host(t, group):
        h = t.cpu()
        dist.all_reduce(h, op=dist.ReduceOp.MAX, group=group)
        return h.to(t.device)
    dist.all_reduce(t, op=dist.ReduceOp.MAX, group=group)
    return t
