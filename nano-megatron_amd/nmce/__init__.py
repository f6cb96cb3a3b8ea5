"""nmce: nano-megatron's vocabulary-parallel cross entropy on MI355X (gfx950).

Public API (mirrors nano_megatron/cross_entropy.py and parallel.py):

* ``vocab_parallel_cross_entropy(logits, target, vocab_start, vocab_end, ctx)``
  -> mean fp32 loss; backward yields the logits gradient.
* ``_VocabParallelCrossEntropy`` -- the autograd Function (per-token loss).
* ``lmhead_vocab_parallel_cross_entropy(hidden, weight, target, vocab_start,
  vocab_end, ctx)`` -> the same loss of ``hidden @ weight.t()`` (the LM head of
  model.py:192 fused in), never storing the logits; backward yields the hidden
  and weight gradients.
* ``FusedParallelLMHead(config, ctx)`` -- drop-in for model.py's
  ``ParallelLMHead`` whose ``forward(x, labels)`` returns that fused loss.
* ``vocab_parallel_embedding(tokens, weight, vocab_start, vocab_end, ctx)`` /
  ``VocabParallelEmbedding(config, ctx)`` -- the scaled lookup over the same
  shard (tp_layers.py:91-132), with the weight's dense gradient.
* ``quantize_rows(x)`` / ``int8_linear(x, weight, weight_scale)`` /
  ``Int8ParallelLMHead`` -- 8-bit rows, their product, and the serving head made
  of it (``FusedParallelLMHead.quantized()``).
* ``vocab_parallel_verify_drafts(...)`` -- drafted tokens against the target's
  sharded logits, from given uniform numbers; with no drafts, sampling.
* ``copy_to_tensor_parallel_region`` / ``gather_from_sequence_parallel_region``
  / ``gather_tokens_rank_major`` -- the collectives on the LM head's input side
  (mappings.py:83-94, :109-120); ``reduce_from_tensor_parallel_region`` /
  ``reduce_scatter_to_sequence_parallel_region`` -- on the embedding's output.
* ``ParallelContext`` / ``vocab_range`` / ``divide`` -- the topology fields and
  shard rule the loss reads.

All loss compute runs in ``libnmce.so`` (hand-written HIP for gfx950) through the C
ABI in ``include/nmce.h``; there is no CPU or PyTorch fallback.
"""

from .cross_entropy import (
    _VocabParallelCrossEntropy,
    validate_targets,
    vocab_parallel_cross_entropy,
)
from .embedding import VocabParallelEmbedding, vocab_parallel_embedding
from .int8 import Int8ParallelLMHead, int8_linear, quantize_rows
from .lmhead import (
    FusedParallelLMHead,
    _LMHeadVocabParallelCrossEntropy,
    lmhead_vocab_parallel_cross_entropy,
)
from .mappings import (
    copy_to_tensor_parallel_region,
    gather_from_sequence_parallel_region,
    gather_tokens_rank_major,
    reduce_from_tensor_parallel_region,
    reduce_scatter_to_sequence_parallel_region,
    targets_rank_major,
)
from .parallel import ParallelContext, divide, vocab_range
from .verify import vocab_parallel_verify_drafts

__all__ = [
    "FusedParallelLMHead",
    "Int8ParallelLMHead",
    "_LMHeadVocabParallelCrossEntropy",
    "_VocabParallelCrossEntropy",
    "ParallelContext",
    "VocabParallelEmbedding",
    "copy_to_tensor_parallel_region",
    "divide",
    "gather_from_sequence_parallel_region",
    "gather_tokens_rank_major",
    "int8_linear",
    "lmhead_vocab_parallel_cross_entropy",
    "quantize_rows",
    "reduce_from_tensor_parallel_region",
    "reduce_scatter_to_sequence_parallel_region",
    "targets_rank_major",
    "validate_targets",
    "vocab_parallel_cross_entropy",
    "vocab_parallel_embedding",
    "vocab_parallel_verify_drafts",
    "vocab_range",
]
