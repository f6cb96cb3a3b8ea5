"""8-bit rows, their product, and the LM head made of it, on gfx950 HIP kernels.

Serving reads the LM head's weight once per step of a few tokens, and that read
is the step's time: held in 8 bits it is half of bf16's. Weight rows (one per
vocabulary entry) and tokens are quantised alike,

    s = max |x| / 127,   q = x / s to the nearest integer, halves to even

the weight once (:func:`quantize_rows`), the tokens within the call, and

    y[n, v] = (sum_k q[n, k] w[v, k]) * s_x[n] * s_w[v]

with the sum exact in 32-bit integers, the scales in fp32 and one rounding to
the output's type. A token that holds an infinity or a NaN gives a row of NaN.

There is no derivative (the training head is ``FusedParallelLMHead``; tensors that
one is wanted through are refused) and no CPU path.
"""

from __future__ import annotations

import torch

from . import _lib
from .cross_entropy import _launch
from .embedding import _rows_of
from .mappings import copy_to_tensor_parallel_region, gather_from_sequence_parallel_region
from .parallel import divide

# The product's rows of 8-bit weights lie a multiple of this many bytes apart.
_ROW_ALIGN = 16
_MAX_STRIDE = 1 << 23  # and at most this many
# Sums of this many products of two 8-bit integers fit 32 bits.
MAX_COLUMNS = 131072


def _check_rows(x: torch.Tensor, what: str) -> None:
    if not x.is_cuda:
        raise RuntimeError(f"nmce: {what} must be on a ROCm device (there is no CPU path)")
    _lib.dtype_code(x.dtype)
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"nmce: {what} must have columns, got {tuple(x.shape)}")
    _lib.refuse_gradient(x, what, "the 8-bit kernels have")


def quantize_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``(q, scale)`` of ``x`` ``[..., K]`` (fp32 or bf16): int8 ``[..., K]`` and
    fp32 ``[...]`` with ``x ~ q * scale[..., None]``.

    Rows of ``q`` lie a multiple of 16 bytes apart (zeros between), as
    :func:`int8_linear` takes its weight; with ``K`` a multiple of 16 ``q`` is
    contiguous. A row of zeros gets the scale 0; one with an infinity or a NaN
    gets NaN (and zeros).
    """
    _check_rows(x, "x")
    lib = _lib.load()
    k = x.shape[-1]
    rows, ld = _rows_of(x)
    ldq = -(-k // _ROW_ALIGN) * _ROW_ALIGN
    q = torch.empty(tuple(x.shape[:-1]) + (ldq,), dtype=torch.int8, device=x.device)
    scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    with torch.cuda.device(x.device):
        _launch("nmce_quantize_rows", lib.nmce_quantize_rows, rows.data_ptr(),
                _lib.dtype_code(x.dtype), rows.shape[0], k, ld, q.data_ptr(), ldq,
                scale.data_ptr(), _lib.stream_handle(x.device))
    return q[..., :k], scale


def _weight_rows(weight: torch.Tensor) -> tuple[torch.Tensor, int]:
    """``weight`` [V, K] int8 with rows a multiple of 16 bytes apart, each
    allocated to a whole 16 bytes, and their stride; a copy where they are not."""
    v, k = weight.shape
    ld = weight.stride(0) if v > 1 else -(-k // _ROW_ALIGN) * _ROW_ALIGN
    whole = (v - 1) * ld + -(-k // _ROW_ALIGN) * _ROW_ALIGN
    held = weight.untyped_storage().nbytes() - weight.storage_offset()
    if ((weight.stride(1) == 1 or k == 1) and k <= ld < _MAX_STRIDE and ld % _ROW_ALIGN == 0
            and weight.data_ptr() % _ROW_ALIGN == 0 and whole <= held):
        return weight, ld
    ld = -(-k // _ROW_ALIGN) * _ROW_ALIGN
    out = torch.zeros((v, ld), dtype=torch.int8, device=weight.device)
    out[:, :k] = weight
    return out, ld


def int8_linear(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, *,
                out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``x @ (weight * weight_scale[:, None]).t()`` with ``x`` quantised per row.

    ``x`` is ``[..., K]`` fp32 or bf16, ``weight`` int8 ``[V, K]`` and
    ``weight_scale`` fp32 ``[V]`` (:func:`quantize_rows` of a weight gives
    both); returns ``[..., V]`` in ``out_dtype`` (fp32 or bf16; ``x``'s by
    default). ``K`` is at most 131072. A weight whose rows are not a multiple
    of 16 bytes apart (one that ``quantize_rows`` did not make) is copied at
    every call.
    """
    _check_rows(x, "x")
    out_dtype = x.dtype if out_dtype is None else out_dtype
    _lib.dtype_code(out_dtype)
    if weight.device != x.device or weight_scale.device != x.device:
        raise RuntimeError(f"nmce: x on {x.device}, weight on {weight.device}, weight_scale on "
                           f"{weight_scale.device}")
    if weight.dtype != torch.int8 or weight_scale.dtype != torch.float32:
        raise TypeError(f"nmce: weight must be int8 and weight_scale float32, got {weight.dtype} "
                        f"and {weight_scale.dtype}")
    _lib.refuse_gradient(weight_scale, "weight_scale", "the 8-bit kernels have")
    k = x.shape[-1]
    if weight.dim() != 2 or weight.shape[1] != k or weight.shape[0] == 0:
        raise ValueError(f"nmce: x {tuple(x.shape)} and weight {tuple(weight.shape)} do not share "
                         "the column count")
    v = weight.shape[0]
    if tuple(weight_scale.shape) != (v,):
        raise ValueError(f"nmce: weight_scale {tuple(weight_scale.shape)} is not one per row of "
                         f"weight {tuple(weight.shape)}")
    if k > MAX_COLUMNS:
        raise ValueError(f"nmce: {k} columns; 8-bit products take at most {MAX_COLUMNS}")
    lib = _lib.load()
    rows, ld = _rows_of(x)
    w, ldw = _weight_rows(weight)
    ws = weight_scale if weight_scale.is_contiguous() else weight_scale.contiguous()
    n = rows.shape[0]
    dev = x.device
    out = torch.empty(tuple(x.shape[:-1]) + (v,), dtype=out_dtype, device=dev)
    buf = torch.empty(max(16, lib.nmce_int8_linear_workspace_bytes(n, k)), dtype=torch.uint8,
                      device=dev)
    with torch.cuda.device(dev):
        _launch("nmce_int8_linear", lib.nmce_int8_linear, rows.data_ptr(),
                _lib.dtype_code(x.dtype), n, k, ld, w.data_ptr(), v, ldw, ws.data_ptr(),
                out.data_ptr(), _lib.dtype_code(out_dtype), v, buf.data_ptr(), buf.numel(),
                _lib.stream_handle(dev))
    return out


class Int8ParallelLMHead(torch.nn.Module):
    """The vocabulary-sharded output projection with an 8-bit weight, for serving.

    Takes ``FusedParallelLMHead``'s constructor arguments and has its input
    mapping; ``forward(x)`` returns this rank's logits ``[..., V/tp]`` in
    ``x``'s type (fp32 or bf16). ``load_weight(w)`` quantises a ``[V/tp,
    n_embd]`` weight (on a ROCm device); ``FusedParallelLMHead.quantized()``
    makes one of a trained head. The buffers ``weight_q`` (rows padded to 16
    bytes) and ``weight_scale`` are what a checkpoint holds; a cast of the module
    (``.to(torch.bfloat16)``, ``.half()``) leaves them int8 and fp32.
    """

    def __init__(self, config, ctx):
        super().__init__()
        self.ctx = ctx
        self.n_embd = config.n_embd
        per_partition = divide(config.vocab_size, ctx.tp_size)
        self.sequence_parallel = bool(getattr(config, "sequence_parallel", False))
        padded = -(-self.n_embd // _ROW_ALIGN) * _ROW_ALIGN
        self.register_buffer("weight_q", torch.zeros(per_partition, padded, dtype=torch.int8))
        self.register_buffer("weight_scale", torch.zeros(per_partition))

    def _apply(self, fn, recurse=True):
        # Casts are not for quantised buffers: what one changed goes back to its
        # former bits, on the device that the call moved it to.
        held = {name: self._buffers[name] for name in ("weight_q", "weight_scale")}
        super()._apply(fn, recurse)
        for name, before in held.items():
            after = self._buffers[name]
            if after.dtype != before.dtype:
                self._buffers[name] = before.to(after.device)
        return self

    def vocab_range(self) -> tuple[int, int]:
        """This rank's global id range (model.py:242-245)."""
        per = self.weight_q.shape[0]
        return self.ctx.tp_rank * per, (self.ctx.tp_rank + 1) * per

    @torch.no_grad()
    def load_weight(self, weight: torch.Tensor) -> None:
        """Quantise ``weight`` into this head's buffers."""
        if tuple(weight.shape) != (self.weight_q.shape[0], self.n_embd):
            raise ValueError(f"nmce: weight {tuple(weight.shape)} is not this head's "
                             f"{(self.weight_q.shape[0], self.n_embd)}")
        q, scale = quantize_rows(weight)
        self.weight_q = torch.nn.functional.pad(q, (0, self.weight_q.shape[1] - self.n_embd))
        self.weight_scale = scale

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if self.sequence_parallel:
            x = gather_from_sequence_parallel_region(x, self.ctx)
        else:
            x = copy_to_tensor_parallel_region(x, self.ctx)
        return int8_linear(x, self.weight_q[:, :self.n_embd], self.weight_scale)
