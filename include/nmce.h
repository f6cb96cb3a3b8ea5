/*
 * nmce.h -- C ABI of the MI355X (gfx950) vocabulary-parallel cross-entropy
 * library (libnmce.so).
 *
 * The library replaces the loss path of nano-megatron:
 *   nano_megatron/cross_entropy.py:16-85  (_VocabParallelCrossEntropy and
 *                                           vocab_parallel_cross_entropy)
 *   nano_megatron/model.py:169-192         (ParallelLMHead, fused variant)
 *   nano_megatron/tp_layers.py:91-132      (VocabParallelEmbedding's lookup)
 * and adds what serving with those weights needs beside it: 8-bit products for
 * the logits, and the verification of drafted tokens.
 *
 * Conventions shared by every entry point:
 *   - All tensor pointers are device memory owned by the caller. Unless an
 *     entry point says otherwise the library never allocates, frees or
 *     synchronises; work is enqueued on `stream` (a hipStream_t, NULL = the
 *     legacy default stream).
 *   - A "row" is one token: the logits of row r start at logits + r*ld
 *     (elements) and hold `vocab_local` contiguous entries.
 *   - A shard covers global vocabulary ids [vocab_start, vocab_start+vocab_local).
 *     Targets are global ids (int64). A target outside the shard contributes
 *     nothing on that shard (the reference's target_mask, cross_entropy.py:28-36).
 *   - Return value: NMCE_OK (0), a negative NMCE_E* argument error, or a
 *     positive hipError_t reported by the launch.
 */
#ifndef NMCE_H
#define NMCE_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* element types of logits / gradients / hidden states / weights */
#define NMCE_F32 0
#define NMCE_BF16 1

/* status codes (negative: argument errors detected before any launch) */
#define NMCE_OK 0
#define NMCE_EINVAL_DTYPE (-1)
#define NMCE_EINVAL_SHAPE (-2)
#define NMCE_EINVAL_ALIGN (-3)
#define NMCE_EINVAL_PTR (-4)
#define NMCE_EINVAL_TP (-5)
#define NMCE_EINVAL_WORKSPACE (-6)
#define NMCE_EINVAL_SCRATCH (-7)

/* Rows covered by one int32 count of nmce_validate_targets. */
#define NMCE_VALIDATE_ROWS_PER_SLOT 1024

/* Human-readable text for a status code (static storage). */
const char* nmce_status_string(int status);

/* Library version, (major << 16) | minor. */
int nmce_version(void);

/*
 * Per-shard row statistics, one read pass over the shard's logits.
 * Replaces cross_entropy.py:21 (row max), :28-36 (masked target pick) and
 * :40-41 (exp-sum) for one vocabulary shard.
 *
 *   row_max[r]       = max_j x[r, j]                            (fp32)
 *   row_sumexp_m1[r] = sum_j exp(x[r, j] - row_max[r]) - 1      (fp32)
 *   target_logit[r]  = x[r, target[r]-vocab_start] if the target is in this
 *                      shard, else 0.0  (raw logit, not shifted)
 * The exp-sum is carried minus the maximum's own term (exactly 1), so that
 * for a confident token, whose other terms are all small, it keeps its
 * relative precision; the loss is formed from it with log1p, and a target
 * at the maximum gets the gradient -(sum - 1)/sum * g from it directly. For
 * fp32 logits the sum is accumulated with
 * the terms equal to 1 kept apart (relative error a few 2^-24); bf16 rows
 * accumulate the plain sum and subtract 1 per lane (absolute error a few
 * 2^-24), which keeps the bf16 pass within its memory-bound time.
 * A row whose shard holds only -inf gives row_max = -1e38 and
 * row_sumexp_m1 = -1 (an empty sum), which the combine gives no weight.
 * dtype: NMCE_F32 or NMCE_BF16 (math is fp32 either way).
 */
int nmce_ce_fwd_stats(const void* logits, int dtype, int64_t n_rows,
                      int64_t vocab_local, int64_t ld, const int64_t* target,
                      int64_t vocab_start, float* row_max, float* row_sumexp_m1,
                      float* target_logit, void* stream);

/*
 * Single-shard forward (TP=1): the statistics pass with the combine folded
 * in. Same results as nmce_ce_fwd_stats(vocab_start = 0) followed by
 * nmce_ce_combine(tp = 1), bit for bit, in one read pass and one launch.
 * Replaces cross_entropy.py:17-50 at world_size == 1.
 *   g_max[r], g_sumexp_m1[r], loss[r] as defined for nmce_ce_combine.
 */
int nmce_ce_fwd(const void* logits, int dtype, int64_t n_rows, int64_t vocab,
                int64_t ld, const int64_t* target, float* loss, float* g_max,
                float* g_sumexp_m1, void* stream);

/*
 * Cross-shard combine of per-shard statistics, done locally.
 * Replaces the three TP all-reduces and the loss line of cross_entropy.py
 * (:22-23 MAX, :37-38 SUM of the target logit, :42-43 SUM of exp-sums, :45).
 *
 * Shard k's statistic for row r sits at [k*shard_stride + r] of each input
 * (a [tp, ...] stack, e.g. the all-gathered [tp, 3, n_rows] buffer of a real
 * TP group with row_max = base, row_sumexp_m1 = base + n_rows, target_logit =
 * base + 2*n_rows and shard_stride = 3*n_rows).
 *
 *   g_max[r]       = max_k row_max[k, r]
 *   g_sumexp_m1[r] = sum_k (1 + row_sumexp_m1[k, r]) * exp(row_max[k, r] - g_max[r]) - 1
 *                    (formed without the cancellation: a shard at the maximum
 *                    adds its row_sumexp_m1, each further one its full sum)
 *   loss[r]        = log1p(g_sumexp_m1[r]) - (sum_k target_logit[k, r] - g_max[r])
 * Any of loss / g_max / g_sumexp_m1 may be NULL if not wanted.
 */
int nmce_ce_combine(const float* row_max, const float* row_sumexp_m1,
                    const float* target_logit, int tp, int64_t shard_stride,
                    int64_t n_rows, float* loss, float* g_max, float* g_sumexp_m1,
                    void* stream);

/*
 * Target validation (cross_entropy.py:79-81: every target must lie in
 * [0, vocab_total)). Writes nmce_validate_slots(n_rows) int32 counts of bad
 * targets, one per NMCE_VALIDATE_ROWS_PER_SLOT rows; every slot is written,
 * so the buffer needs no clearing. The caller raises if any count is nonzero.
 * bad_counts may be device memory or pinned host memory (hipHostMalloc,
 * which the device addresses at its host address): the Python host writes
 * the counts straight to the host that way, with no copy after the kernel.
 */
int64_t nmce_validate_slots(int64_t n_rows);
int nmce_validate_targets(const int64_t* target, int64_t n_rows,
                          int64_t vocab_total, int32_t* bad_counts,
                          void* stream);

/*
 * The same check (cross_entropy.py:79-81) in one workgroup, for a loss
 * kernel that follows on the same stream and must leave its inputs untouched
 * on a bad target (the reference raises before touching anything, :80-81):
 * the number of bad targets, saturated at INT32_MAX, goes to bad_count[0]
 * (for the host; device or pinned host memory) and to bad_flag[0] (device
 * memory, passed to nmce_ce_fwd_bwd as target_bad). Both are written
 * unconditionally, so neither needs clearing.
 */
int nmce_validate_targets_once(const int64_t* target, int64_t n_rows,
                               int64_t vocab_total, int32_t* bad_count,
                               int32_t* bad_flag, void* stream);

/*
 * Backward over one shard: grad = (softmax - onehot(target)) * grad_output.
 * Replaces cross_entropy.py:53-65 plus the autograd cast back to the logits
 * dtype (the .float() at :83).
 *
 *   grad[r, j] = (exp(x[r, j] - g_max[r]) / (1 + g_sumexp_m1[r])
 *                 - [j == target[r] - vocab_start]) * grad_output[r*gout_stride]
 * with the target column, when it holds the row maximum, formed as
 *   -g_sumexp_m1[r] / (1 + g_sumexp_m1[r]) * g,
 * the same value without the cancellation of softmax - 1 near 1 (a target
 * below the maximum has softmax <= 1/2, where the plain form is exact enough).
 * gout_stride = 0 broadcasts grad_output[0] to every row (the loss.mean()
 * case). grad may equal logits (in place, ld_grad == ld); otherwise the two
 * must not overlap. grad has the same dtype as logits.
 */
int nmce_ce_bwd(const void* logits, void* grad, int dtype, int64_t n_rows,
                int64_t vocab_local, int64_t ld, int64_t ld_grad,
                const int64_t* target, int64_t vocab_start, const float* g_max,
                const float* g_sumexp_m1, const float* grad_output,
                int64_t gout_stride, void* stream);

/*
 * nmce_ce_bwd with the upstream gradient divided by gout_div (> 0) per row:
 * grad_output[r*gout_stride] / gout_div replaces grad_output[r*gout_stride].
 * With gout_stride = 0 and gout_div = N this is the backward of
 * loss.mean() (cross_entropy.py:85) folded in: the scalar gradient of the
 * mean is read directly, and the per-token value is the same fp32 quotient
 * torch's MeanBackward forms, so the result is bit-identical to nmce_ce_bwd
 * on the expanded gradient. gout_div = 1 is nmce_ce_bwd.
 */
int nmce_ce_bwd_scaled(const void* logits, void* grad, int dtype, int64_t n_rows,
                       int64_t vocab_local, int64_t ld, int64_t ld_grad,
                       const int64_t* target, int64_t vocab_start, const float* g_max,
                       const float* g_sumexp_m1, const float* grad_output,
                       int64_t gout_stride, float gout_div, void* stream);

/*
 * nmce_ce_bwd_scaled with gout_stride = 0, after nmce_ce_fwd_bwd. `assumed`
 * (device, one float) is the upstream value that forward computed the
 * gradient for: when grad_output[0] equals it every workgroup returns at
 * once, leaving `grad` as written; otherwise this is nmce_ce_bwd_scaled
 * exactly (cross_entropy.py:53-65 with the mean of :85). grad_output[0] is
 * also written to `observed` (device, one float; may be NULL), which a
 * caller can pass as the next forward's grad_expected.
 */
int nmce_ce_bwd_scaled_unless(const void* logits, void* grad, int dtype, int64_t n_rows,
                              int64_t vocab_local, int64_t ld, int64_t ld_grad,
                              const int64_t* target, int64_t vocab_start, const float* g_max,
                              const float* g_sumexp_m1, const float* grad_output, float gout_div,
                              const float* assumed, float* observed, void* stream);

/*
 * One-pass forward and backward at TP = 1 (cross_entropy.py:17-65 with the
 * mean of :85, world_size == 1). Each row is read once and held on chip; the
 * kernel writes g_max, g_sumexp_m1 and loss, and the gradient for the
 * upstream value u of the mean (u / gout_div per token) into `grad`, where
 * u = grad_expected[0], or 1.0 when that is zero, subnormal, infinite or NaN;
 * u goes to grad_assumed[0]. Both are device pointers to one float. `grad`
 * is either a separate buffer or the logits themselves (grad == logits,
 * ld_grad == ld): the row's target logit is read before the row is
 * overwritten. Every output is bit-identical to nmce_ce_fwd followed by
 * nmce_ce_bwd_scaled with grad_output = {u} and gout_stride = 0.
 * The backward is then, for a separate buffer,
 * nmce_ce_bwd_scaled_unless(..., assumed = grad_assumed, ...), which
 * rewrites `grad` from the logits only when the real upstream value differs;
 * in place, nmce_ce_grad_rescale_unless.
 * Requirements: vocab a whole number of 16-byte vectors and at most
 * nmce_ce_fwd_bwd_max_vocab(dtype) (131072 bf16, 65536 fp32); logits, grad
 * and both row strides 16-byte aligned. No counterpart call in the reference,
 * whose forward likewise computes the softmax that its backward returns.
 * target_bad (may be NULL): the bad_flag of nmce_validate_targets_once,
 * enqueued before on the same stream. When it is nonzero the kernel writes
 * nothing at all, so logits that were to receive their gradient in place
 * are left as they were.
 */
int64_t nmce_ce_fwd_bwd_max_vocab(int dtype);
int nmce_ce_fwd_bwd(const void* logits, void* grad, int dtype, int64_t n_rows, int64_t vocab,
                    int64_t ld, int64_t ld_grad, const int64_t* target, float* loss, float* g_max,
                    float* g_sumexp_m1, const float* grad_expected, float* grad_assumed,
                    const int32_t* target_bad, float gout_div, void* stream);

/*
 * Backward after an in-place nmce_ce_fwd_bwd (grad == logits), whose
 * gradient was written for the upstream value assumed[0]: when
 * grad_output[0] equals it, every workgroup returns at once; otherwise every
 * entry of `grad` is multiplied by grad_output[0] / assumed[0] in fp32 and
 * rounded back to the gradient's dtype (cross_entropy.py:64: the gradient is
 * linear in grad_output). The logits are gone, so this cannot recompute; the
 * result is within four (fp32) or two (bf16) units in the last place of the
 * recomputed one, and equal to it when the ratio is a power of two.
 * grad_output[0] also goes to `observed` (may be NULL), the next forward's
 * grad_expected. Same layout requirements as nmce_ce_fwd_bwd.
 */
int nmce_ce_grad_rescale_unless(void* grad, int dtype, int64_t n_rows, int64_t vocab,
                                int64_t ld_grad, const float* grad_output, const float* assumed,
                                float* observed, void* stream);

/*
 * The same for two contiguous gradients of one backward, count_a and count_b
 * elements (multiples of 16 bytes' elements; 16-byte aligned; either may be
 * empty), in one launch.
 */
int nmce_ce_grad_rescale_pair_unless(void* grad_a, int64_t count_a, void* grad_b, int64_t count_b,
                                     int dtype, const float* grad_output, const float* assumed,
                                     float* observed, void* stream);

/*
 * The two one-pass calls above (nmce_ce_fwd_bwd, nmce_ce_grad_rescale_unless)
 * for rows of any width and alignment: `vocab` up to the
 * same limit, logits and grad aligned to their element. In
 * nmce_ce_fwd_bwd_ragged every grad row must share its logits row's offset
 * from a 16-byte boundary (logits - grad a multiple of 16 bytes, ld - ld_grad
 * a multiple of 16 bytes' elements). Same results, bit for bit, as
 * nmce_ce_fwd followed by nmce_ce_bwd_scaled.
 */
int nmce_ce_fwd_bwd_ragged(const void* logits, void* grad, int dtype, int64_t n_rows,
                           int64_t vocab, int64_t ld, int64_t ld_grad, const int64_t* target,
                           float* loss, float* g_max, float* g_sumexp_m1,
                           const float* grad_expected, float* grad_assumed,
                           const int32_t* target_bad, float gout_div, void* stream);
int nmce_ce_grad_rescale_unless_ragged(void* grad, int dtype, int64_t n_rows, int64_t vocab,
                                       int64_t ld_grad, const float* grad_output,
                                       const float* assumed, float* observed, void* stream);

/*
 * Measurement support (no counterpart in the reference): a plain copy of
 * `bytes` (multiple of 16, both pointers 16-byte aligned) with the loss
 * kernels' access pattern -- 16-byte non-temporal loads and stores. Its HBM
 * traffic is known exactly, so hardware byte counters (FETCH_SIZE,
 * WRITE_SIZE) read for it give the scale factors for the same counters read
 * on the loss kernels.
 */
int nmce_stream_copy(const void* src, void* dst, int64_t bytes, void* stream);

/* ---------------------------------------------------------------------------
 * Fused LM head + cross entropy (bf16 only).
 *
 * Replaces ParallelLMHead.forward's projection logits = hidden @ weight.t()
 * (model.py:192, bf16 under autocast per model.py:255-257) followed by the
 * loss of cross_entropy.py:16-65, without storing the [n_rows, vocab_local]
 * logits. hidden is [n_rows, hidden_size] and weight (the vocabulary shard of
 * the tied embedding, tp_layers.py:108) is [vocab_local, hidden_size], both
 * row-major with row stride hidden_size, 16-byte aligned; hidden_size must be
 * a multiple of 64. Logits are accumulated in fp32 and not rounded to bf16.
 * The gradients that the entries below write, grad_hidden and grad_weight, need
 * be aligned to their element only (16-byte aligned ones leave faster).
 * --------------------------------------------------------------------------- */

/* Device workspace bytes needed by nmce_lmhead_ce_fwd_stats. */
int64_t nmce_lmhead_ce_fwd_workspace_bytes(int64_t n_rows, int64_t hidden_size,
                                           int64_t vocab_local);

/*
 * Per-shard statistics of the logits hidden @ weight^T, as nmce_ce_fwd_stats
 * computes them for a stored logit slab (cross_entropy.py:21, :28-36,
 * :40-41 on the shard [vocab_start, vocab_start + vocab_local)), the exp-sum
 * minus one accumulated with the terms equal to 1 kept apart. Combine the
 * shards with nmce_ce_combine (tp = 1 for a single shard).
 */
int nmce_lmhead_ce_fwd_stats(const void* hidden, const void* weight, int dtype, int64_t n_rows,
                             int64_t hidden_size, int64_t vocab_local, const int64_t* target,
                             int64_t vocab_start, float* row_max, float* row_sumexp_m1,
                             float* target_logit, void* workspace, int64_t workspace_bytes,
                             void* stream);

/*
 * nmce_lmhead_ce_fwd_stats without a workspace argument, for callers that
 * cannot allocate device memory (code under HIP graph capture, tight serving
 * loops, harnesses that forbid hipMalloc). No counterpart in the reference.
 * The partial statistics go to a fixed 64 MiB device array inside the
 * library (one per GPU, held until the process ends), and the tokens are
 * processed in as many launches as it takes to fit them there; the results
 * are bit-identical to nmce_lmhead_ce_fwd_stats. The call allocates nothing.
 * Limit: 3 * ceil(vocab_local / 128) * 4 bytes per token must fit in 64 MiB
 * (vocab_local up to 715,827,840); beyond that it returns
 * NMCE_EINVAL_SCRATCH before launching anything. Every call on one GPU uses
 * the same array: calls that overlap on one GPU (different streams, or
 * threads) race and must be serialised by the caller.
 */
int nmce_lmhead_ce_fwd_stats_noalloc(const void* hidden, const void* weight, int dtype,
                                     int64_t n_rows, int64_t hidden_size, int64_t vocab_local,
                                     const int64_t* target, int64_t vocab_start, float* row_max,
                                     float* row_sumexp_m1, float* target_logit, void* stream);

/* Device workspace bytes needed by nmce_lmhead_ce_bwd for a vocabulary chunk
 * of vocab_chunk rows (<= 0: the whole shard in one chunk). */
int64_t nmce_lmhead_ce_bwd_workspace_bytes(int64_t n_rows, int64_t hidden_size,
                                           int64_t vocab_local, int64_t vocab_chunk);

/*
 * Backward workspace layout (all values in elements of int64), written to
 * layout[0 .. NMCE_LMHEAD_LAYOUT_FIELDS-1]:
 *   [0] total workspace bytes
 *   [1] ldt      tokens rounded up to 64 (row stride of X^T and dZ^T)
 *   [2] vpad     vocab_local rounded up to 256 (row stride of W^T)
 *   [3] chunk    vocabulary rows per chunk (multiple of 256)
 *   [4] n_chunks
 *   [5] byte offset of X^T   bf16 [hidden_size, ldt], zero beyond n_rows
 *   [6] byte offset of W^T   bf16 [hidden_size, vpad], zero beyond vocab_local
 *   [7] byte offset of dZ^T  bf16 [chunk, ldt] of the current chunk
 *   [8] byte offset of dZ    bf16 [n_rows, chunk] of the current chunk
 *   [9] byte offset of the fp32 [n_rows, hidden_size] accumulator of
 *       nmce_lmhead_ce_bwd (present when n_chunks > 1)
 * for the caller-driven steps below. nmce_lmhead_ce_bwd by itself arranges the
 * same bytes as it needs them: X^T, one chunk's dZ^T and, where they fit, fp32
 * partial sums of grad_hidden in the place of W^T, dZ and the accumulator.
 */
#define NMCE_LMHEAD_LAYOUT_FIELDS 10
int nmce_lmhead_ce_bwd_layout(int64_t n_rows, int64_t hidden_size, int64_t vocab_local,
                              int64_t vocab_chunk, int64_t* layout);

/* Step 1 of a caller-driven backward: X^T and W^T into the workspace. */
int nmce_lmhead_ce_bwd_prepare(const void* hidden, const void* weight, int dtype, int64_t n_rows,
                               int64_t hidden_size, int64_t vocab_local, int64_t vocab_chunk,
                               void* workspace, int64_t workspace_bytes, void* stream);

/*
 * Step 2, once per chunk c (rows [c*chunk, c*chunk + chunk) of the shard):
 * recompute that slice of the logits and write the logit gradient
 *   dZ[r, j] = (exp(z[r, j] - g_max[r]) / (1 + g_sumexp_m1[r])
 *               - [j == target[r] - vocab_start]) * grad_output[r*gout_stride]
 * (target column without cancellation, as in nmce_ce_bwd)
 * as bf16 into the workspace's dZ^T and dZ (zeros in their padding). The
 * caller then forms grad_weight rows = dZ^T_c X and grad_hidden += dZ_c W_c
 * (e.g. with a library GEMM on X^T and W^T) before the next chunk overwrites
 * them. This is the fused part of cross_entropy.py:53-65 + the matmul
 * backward of model.py:192.
 */
int nmce_lmhead_ce_bwd_dz(const void* hidden, const void* weight, int dtype, int64_t n_rows,
                          int64_t hidden_size, int64_t vocab_local, const int64_t* target,
                          int64_t vocab_start, const float* g_max, const float* g_sumexp_m1,
                          const float* grad_output, int64_t gout_stride, int64_t vocab_chunk,
                          int64_t chunk_index, void* workspace, int64_t workspace_bytes,
                          void* stream);

/*
 * Backward of the fused LM head + loss (cross_entropy.py:53-65 followed by
 * the matmul backward of model.py:192):
 *   dZ[r, j]        = (exp(z[r, j] - g_max[r]) / (1 + g_sumexp_m1[r])
 *                      - [j == target[r] - vocab_start]) * grad_output[r*gout_stride]
 *   grad_hidden     = dZ @ weight          [n_rows, hidden_size] bf16
 *   grad_weight     = dZ^T @ hidden        [vocab_local, hidden_size] bf16
 * with z = hidden @ weight^T recomputed chunk by chunk (vocab_chunk rows of
 * the shard at a time) and dZ rounded to bf16 before the two products, as the
 * reference's autocast matmul backward consumes a bf16 gradient. g_max and
 * g_sumexp_m1 are the combined statistics of the forward (nmce_ce_combine).
 * grad_hidden is this shard's contribution only (the TP all-reduce of the
 * input gradient, mappings.py:83-94, belongs to the caller).
 */
int nmce_lmhead_ce_bwd(const void* hidden, const void* weight, int dtype, int64_t n_rows,
                       int64_t hidden_size, int64_t vocab_local, const int64_t* target,
                       int64_t vocab_start, const float* g_max, const float* g_sumexp_m1,
                       const float* grad_output, int64_t gout_stride, void* grad_hidden,
                       void* grad_weight, int64_t vocab_chunk, void* workspace,
                       int64_t workspace_bytes, void* stream);

/* ---------------------------------------------------------------------------
 * One-pass fused LM head + loss: forward and backward in the forward, for
 * the upstream value the caller assumes (bf16 only; same operand layout as
 * above). The tokens go in chunks of token_chunk (rounded up to 256; <= 0:
 * all at once). Per chunk the statistics GEMM keeps its exponentials
 * P = exp(z - block max) in the workspace; once the chunk's statistics are
 * combined across the TP group, dZ follows from P by one factor per
 * (128-row block, token), in place, and the dX rows of the chunk and its
 * share of dW are formed by libnmce's GEMM, which reads dZ^T and the weight
 * as they lie and the chunk's hidden rows transposed (hidden_size x
 * token_chunk bf16). The one buffer that grows with both sizes is a chunk's
 * P, then dZ^T: bf16 [vocab_local, token_chunk], the size of the bf16 logits
 * when the chunk holds every token. The logits are computed once: 6 * n_rows * vocab_local *
 * hidden_size flops in all. vocab_local is at most 8388352 (65535 blocks of
 * 128 rows once padded to 256); a larger shard is NMCE_EINVAL_SHAPE.
 * Replaces model.py:192 followed by cross_entropy.py:17-65 and the matmul
 * backward of model.py:192; with a caller that assumes the right upstream
 * value, as the reference's forward computes the softmax its backward
 * returns (cross_entropy.py:48-49).
 * --------------------------------------------------------------------------- */

/*
 * Workspace layout (int64 values) written to layout[0 .. 11]:
 *   [0] total bytes  [1] chunk (tokens per chunk)  [2] n_chunks
 *   [3] ldt (chunk padded to 64)  [4] vpad (vocab_local padded to 256)
 *   [5] nb (ceil(vocab_local / 128))  [6..9] byte offsets of P^T
 *   (= dZ_c^T, [vpad, ldt]: the only buffer that grows with the vocabulary
 *   and the chunk; both backward products read it), the partial statistics,
 *   the fp32 dW accumulator (present when n_chunks > 1) and the fp32 partials
 *   of a chunk's dX product when it is split over K  [10] the number of K
 *   ranges of that product (1: not split; more when a chunk's dX has too few
 *   256x256 tiles to fill the current device's compute units)  [11] byte
 *   offset of the chunk's hidden rows transposed, X_c^T [hidden_size, ldt]
 *   bf16 (the dW product's second operand), which runs to the end.
 */
#define NMCE_LMHEAD_FUSED_LAYOUT_FIELDS 12
int nmce_lmhead_ce_fused_layout(int64_t n_rows, int64_t hidden_size, int64_t vocab_local,
                                int64_t token_chunk, int64_t* layout);

/*
 * layout[0] above on a device of `compute_units` compute units (0: the current
 * device's count), or -1 for arguments that the layout refuses. Callers whose
 * ranks must agree on a chunk by its workspace ask for one count everywhere.
 */
int64_t nmce_lmhead_ce_fused_workspace_bytes(int64_t n_rows, int64_t hidden_size,
                                             int64_t vocab_local, int64_t token_chunk,
                                             int compute_units);

/* assumed[0] = hint[0], or 1.0 when hint[0] is zero, subnormal, infinite or
 * NaN (a gradient written for such a value could not be rescaled). Both are
 * device pointers to one float. */
int nmce_hint_assume(const float* hint, float* assumed, void* stream);

/*
 * Chunk c (tokens [c*chunk, min((c+1)*chunk, n_rows))): this shard's
 * statistics of those tokens, as nmce_lmhead_ce_fwd_stats computes them,
 * written at the tokens' positions of row_max / row_sumexp_m1 /
 * target_logit ([n_rows] each), and P of the chunk kept in the workspace.
 * Chunks run in order 0, 1, ..., each followed by its
 * nmce_lmhead_ce_fused_chunk_grads.
 */
int nmce_lmhead_ce_fused_chunk_stats(const void* hidden, const void* weight, int dtype,
                                     int64_t n_rows, int64_t hidden_size, int64_t vocab_local,
                                     const int64_t* target, int64_t vocab_start,
                                     int64_t token_chunk, int64_t chunk_index, float* row_max,
                                     float* row_sumexp_m1, float* target_logit, void* workspace,
                                     int64_t workspace_bytes, void* stream);

/*
 * The same where the shard is the whole vocabulary (target ids from 0): the
 * chunk's statistics are then the final ones, and its per-token loss is
 * written with them, as nmce_ce_combine over one shard would. `assumed`
 * (unless NULL) gets what nmce_hint_assume(hint, assumed) writes.
 */
int nmce_lmhead_ce_fused_chunk_loss(const void* hidden, const void* weight, int dtype,
                                    int64_t n_rows, int64_t hidden_size, int64_t vocab,
                                    const int64_t* target, int64_t token_chunk,
                                    int64_t chunk_index, float* loss, float* g_max,
                                    float* g_sumexp_m1, float* target_logit, const float* hint,
                                    float* assumed, void* workspace, int64_t workspace_bytes,
                                    void* stream);

/*
 * Chunk c's gradients, given the combined statistics g_max / g_sumexp_m1 of
 * its tokens (nmce_ce_combine over the TP group) and this shard's
 * target_logit from nmce_lmhead_ce_fused_chunk_stats:
 *   dZ[t, v]          = (softmax - onehot) * grad_output[t*gout_stride] / gout_div
 *                       (target column as in nmce_ce_bwd), rounded to bf16
 *   grad_hidden rows  = dZ_c @ weight                 (this shard's share)
 *   grad_weight      += dZ_c^T @ hidden_c             (fp32 across chunks,
 *                       bf16 when the last chunk is done)
 * grad_hidden is [n_rows, hidden_size], grad_weight [vocab_local,
 * hidden_size], both bf16.
 */
int nmce_lmhead_ce_fused_chunk_grads(const void* hidden, const void* weight, int dtype,
                                     int64_t n_rows, int64_t hidden_size, int64_t vocab_local,
                                     const int64_t* target, int64_t vocab_start,
                                     int64_t token_chunk, int64_t chunk_index, const float* g_max,
                                     const float* g_sumexp_m1, const float* target_logit,
                                     const float* grad_output, int64_t gout_stride,
                                     float gout_div, void* grad_hidden, void* grad_weight,
                                     void* workspace, int64_t workspace_bytes, void* stream);

/*
 * Embedding lookup over a vocabulary shard (tp_layers.py:91-132):
 *   out[i, :] = scale * weight[tokens[i] - vocab_start, :]   (in fp32, rounded once)
 * for ids in [vocab_start, vocab_start + vocab_local), and zeros for others
 * (any int64; nothing is read out of bounds). weight [vocab_local, ldw] and
 * out [n_tokens, ldo] are NMCE_F32 or NMCE_BF16 each, aligned to their
 * element; rows on the 16-byte grid go by 16-byte vectors. n_tokens and
 * vocab_local below 2^31, hidden at most 2^24.
 */
int nmce_embedding_fwd(const int64_t* tokens, int64_t n_tokens, const void* weight,
                       int weight_dtype, int64_t vocab_local, int64_t hidden, int64_t ldw,
                       int64_t vocab_start, float scale, void* out, int out_dtype, int64_t ldo,
                       void* stream);

/* Workspace of nmce_embedding_bwd in bytes (-1: sizes it does not take). */
int64_t nmce_embedding_bwd_workspace_bytes(int64_t n_tokens, int64_t vocab_local, int64_t hidden);

/*
 * The weight's gradient of nmce_embedding_fwd, written whole:
 *   grad_weight[v, :] = scale * sum of grad_out[i, :] over tokens[i] = vocab_start + v
 * (fp32 sums in an order that the tokens alone decide, rounded once; zeros
 * where no token is). grad_weight is [vocab_local, hidden] contiguous, 16-byte
 * aligned; grad_out [n_tokens, ldg] aligned to its element. The workspace
 * (16-byte aligned) belongs to this call until it is done on the stream.
 */
int nmce_embedding_bwd(const int64_t* tokens, int64_t n_tokens, const void* grad_out,
                       int grad_dtype, int64_t ldg, int64_t vocab_local, int64_t hidden,
                       int64_t vocab_start, float scale, void* grad_weight, int weight_dtype,
                       void* workspace, int64_t workspace_bytes, void* stream);

/*
 * 8-bit rows: scale[r] = max |x[r, :]| / 127 and q[r, k] = x[r, k] / scale[r]
 * to the nearest integer, halves to even (formed from 127 x / max |x|, whose
 * halves are exact). x [n_rows, ldx] NMCE_F32 or NMCE_BF16, aligned to its
 * element; q [n_rows, ldq] gets zeros in columns .. ldq - 1. A row of zeros
 * gets the scale 0; one with an infinity or a NaN the scale NaN and zeros.
 */
int nmce_quantize_rows(const void* x, int dtype, int64_t n_rows, int64_t columns, int64_t ldx,
                       int8_t* q, int64_t ldq, float* scale, void* stream);

/* Workspace of nmce_int8_linear in bytes (-1: sizes it does not take). */
int64_t nmce_int8_linear_workspace_bytes(int64_t n_rows, int64_t columns);

/*
 * Logits from an 8-bit weight: x quantised as nmce_quantize_rows does, then
 *   out[n, v] = (sum_k qx[n, k] * weight[v, k]) * sx[n] * w_scale[v]
 * with the sum exact in 32-bit integers (columns <= 131072), the rest in fp32,
 * rounded once to out_dtype. weight [vocab_local, ldw]: 16-byte aligned, ldw a
 * multiple of 16 below 2^23, each row allocated to a whole 16 bytes (what they
 * hold past `columns` does not matter). x and out are aligned to their
 * elements. The workspace (16-byte aligned) belongs to this call until it is
 * done on the stream.
 */
int nmce_int8_linear(const void* x, int dtype, int64_t n_rows, int64_t columns, int64_t ldx,
                     const int8_t* weight, int64_t vocab_local, int64_t ldw, const float* w_scale,
                     void* out, int out_dtype, int64_t ldo, void* workspace,
                     int64_t workspace_bytes, void* stream);

/*
 * Verification of drafted tokens over a vocabulary shard, from given uniform
 * numbers. With p = softmax(target / T), q = softmax(draft / T) at position i
 * (all in 64 bits), the drafted token d stands while accept_u q(d) < p(d). At
 * the first that does not, the next token is the first id whose running sum of
 * max(p - q, 0) passes sample_u times all of it; after the last draft, of p.
 *   - T not above 0 (or NaN): a draft stands where it is the lowest id of the
 *     largest logit, which is also the next token.
 *   - draft NULL: q is one at the drafted token.
 *   - A drafted token outside [0, vocab_total) ends its sequence's drafts (the
 *     padding of shorter ones); the next token comes from p there.
 *   - A draft row that is no distribution (all -inf, or an infinity or NaN in
 *     it) lets nothing stand; the next token comes from p. Such a target row
 *     gives the token -1.
 *   - Where max(p - q, 0) is nothing (adds up to 1e-14 or less, what rounding
 *     leaves of equal distributions), the next token comes from p.
 *   - Uniform numbers outside [0, 1) are taken as the nearest inside, NaN as 0.
 * Shapes: target [batch, drafts + 1, vocab_local], draft [batch, drafts,
 * vocab_local] with the given strides (elements; the vocabulary's is 1),
 * aligned to their elements; draft_tokens and accept_u [batch, drafts] and
 * sample_u [batch] contiguous; temperature [batch], or NULL: temperature_all
 * (64 bits wide, as all of the arithmetic is).
 * batch x (2 drafts + 1) x slabs (nmce_verify_slabs) is at most 2^23.
 */
typedef struct nmce_verify_batch {
  const void* target;
  const void* draft;
  const int64_t* draft_tokens;
  const float* accept_u;
  const float* sample_u;
  const float* temperature;
  int64_t target_batch_stride, target_row_stride;
  int64_t draft_batch_stride, draft_row_stride;
  int64_t batch, drafts;
  int64_t vocab_local, vocab_start, vocab_total;
  double temperature_all;
  int dtype;
} nmce_verify_batch;

/* Slabs that a shard's rows are cut into, and the decisions' workspace. */
int64_t nmce_verify_slabs(int64_t vocab_local);
int64_t nmce_verify_workspace_bytes(int64_t batch);

/*
 * The steps, in order. stats: doubles [rows][slabs][4] of this shard's rows
 * (batch x (drafts + 1) of the target, then batch x drafts of the draft). With
 * several ranks gather them to [ranks][rows][slabs][4] for the next step, and
 * its masses [batch][slabs][2] to [ranks][batch][slabs][2] for the one after.
 * nmce_verify_masses writes accepted [batch] (how many drafts stand) and
 * tokens, logprobs [batch][drafts + 1] but for the next token, whose place
 * holds -1 and 0 until nmce_verify_pick writes it (one rank, picked NULL), or
 * writes picked [batch][2], of which nmce_verify_finish takes the ranks'
 * elementwise maximum. Places behind the next token hold -1 and 0. logprobs
 * are log p of the tokens (of T = 1 where T is 0).
 */
int nmce_verify_stats(const nmce_verify_batch* batch, double* stats, void* stream);
int nmce_verify_masses(const nmce_verify_batch* batch, const double* stats, int ranks,
                       double* masses, int64_t* tokens, int64_t* accepted, float* logprobs,
                       void* workspace, int64_t workspace_bytes, void* stream);
int nmce_verify_pick(const nmce_verify_batch* batch, const double* masses, int ranks, int rank,
                     const void* workspace, int64_t workspace_bytes, int64_t* tokens,
                     float* logprobs, double* picked, void* stream);
int nmce_verify_finish(const double* picked, const void* workspace, int64_t workspace_bytes,
                       int64_t batch, int64_t drafts, int64_t* tokens, float* logprobs,
                       void* stream);

/*
 * Penalties, biases and masks on a vocabulary shard's logits, in one pass:
 * out[b, i, :] from logits[b, i, :], i < rows (after the first i drafts). With
 * count = how often an id is in output[b] and drafts[b][0 .. i - 1],
 *   in prompt[b] or count > 0:  x <- x / r where x > 0, else x r
 *   count > 0:                  x <- x - f count - p
 *   then x + the id's biases in their order, and -inf unless it is allowed.
 * What any of this touches is formed in 64 bits and rounded once; the rest is
 * copied. Ids are global; one outside [0, vocab_total) stands for none.
 *   - prompt [batch, n_prompt], output [batch, n_output], drafts [batch,
 *     rows - 1], bias_ids and bias [batch, n_bias] with the given strides
 *     between lists; repetition, frequency, presence [batch], or NULL: the
 *     *_all value of each. r that is not a finite number above 0 is taken as 1.
 *   - allowed: bit id % 32 of word id / 32, ceil(vocab_total / 32) words a row
 *     at the given strides (in words), or NULL (all are).
 *   - out may be logits (in place, the same strides): only touched and masked
 *     elements are written. Otherwise the two must not overlap.
 * n_bias at most NMCE_ADJUST_MAX_BIASES, n_output at most 2^29; batch x rows x
 * ceil(vocab_local / 8192) at most 2^23. More than 512 biases within 8192 neighbouring
 * ids (counted from vocab_start), one of whose ids comes again, are searched in n_bias
 * steps each: 2048 take 0.5 ms a row, 8192 7 ms, where different ids take 13 and 20 us.
 */
#define NMCE_ADJUST_MAX_BIASES 8192
typedef struct nmce_adjust_batch {
  const void* logits;
  void* out;
  const int64_t* prompt;
  const int64_t* output;
  const int64_t* drafts;
  const int64_t* bias_ids;
  const float* bias;
  const uint32_t* allowed;
  const float* repetition;
  const float* frequency;
  const float* presence;
  int64_t logits_batch_stride, logits_row_stride;
  int64_t out_batch_stride, out_row_stride;
  int64_t prompt_stride, output_stride, drafts_stride, bias_ids_stride, bias_stride;
  int64_t allowed_batch_stride, allowed_row_stride;
  int64_t n_prompt, n_output, n_bias;
  int64_t batch, rows;
  int64_t vocab_local, vocab_start, vocab_total;
  double repetition_all, frequency_all, presence_all;
  int dtype;
} nmce_adjust_batch;
int nmce_adjust_logits(const nmce_adjust_batch* batch, void* stream);

/*
 * The k largest logits of each row of a vocabulary shard with their ids, in order
 * (of equal ones the lowest id first; NaN above +inf; -0 as 0), and the row's
 * log sum exp(x / temperature). k at most NMCE_TOP_MAX_K, n_rows at most 2^22,
 * temperature from 1e-30 to 1e30.
 *   - list NULL: the results. values [n_rows, k] in the logits' type, ids
 *     [n_rows, k], log_normalizer [n_rows]; k is at most vocab_local.
 *   - otherwise list [n_rows, k + 1]: this shard's part (fewer than k entries
 *     where it has fewer columns), of which nmce_top_merge takes the ranks',
 *     [ranks, n_rows, k + 1], to the results.
 * logits [n_rows, ld] is aligned to its element. The workspace (16-byte aligned)
 * belongs to this call until it is done on the stream.
 */
#define NMCE_TOP_MAX_K 512
int64_t nmce_top_workspace_bytes(int64_t n_rows, int64_t vocab_local, int k);
int nmce_top_logits(const void* logits, int dtype, int64_t n_rows, int64_t vocab_local, int64_t ld,
                    int64_t vocab_start, int k, double temperature, int64_t* list, void* values,
                    int64_t* ids, float* log_normalizer, void* workspace, int64_t workspace_bytes,
                    void* stream);
int nmce_top_merge(const int64_t* lists, int ranks, int dtype, int64_t n_rows, int k,
                   double temperature, void* values, int64_t* ids, float* log_normalizer,
                   void* stream);

/*
 * Distillation from a teacher's top logits. With q = softmax(z / T) of a student's
 * row over the whole vocabulary and the teacher's p at its k listed ids,
 *   p = exp(t / T - teacher_log_normalizer), r = max(1 - sum p, 0), or, with
 *   teacher_log_normalizer NULL, p = softmax(t / T) over the list, r = 0:
 *   loss = sum p (log p - log q) + r (log r - log s)
 * where s is the sum of q outside the list (one class).
 *   - An id outside [0, vocab_total) is padding. A row without any other, or
 *     whose normaliser is -inf (with NULL, whose list holds only -inf), has no
 *     teacher: loss and gradient 0, whatever its logits are. An id that comes
 *     several times adds up its p.
 *   - Where the student gives everything outside the list nothing (-inf), the
 *     rest has no term. A student's row of only -inf, or with +inf or NaN: NaN.
 * logits [n_rows, ld] of this shard, teacher_logits and teacher_ids [n_rows, k]
 * at their own row strides, teacher_log_normalizer [n_rows]; aligned to their
 * elements. k at most NMCE_DISTILL_MAX_K, n_rows at most 2^22, vocab_total below
 * 2^31 - 1, temperature from 1e-6 to 1e6.
 */
#define NMCE_DISTILL_MAX_K 1024
typedef struct nmce_distill_batch {
  const void* logits;
  const void* teacher_logits;
  const int64_t* teacher_ids;
  const float* teacher_log_normalizer;
  int64_t ld, teacher_ld, ids_ld;
  int64_t n_rows;
  int64_t vocab_local, vocab_start, vocab_total;
  double temperature;
  int k;
  int dtype, teacher_dtype;
} nmce_distill_batch;

/* What a forward leaves for its backward, in bytes (16-byte aligned). */
int64_t nmce_distill_state_bytes(int64_t n_rows, int k);

/*
 * The forward in two steps: this shard's statistics, [n_rows, 5] doubles (with
 * several ranks gather them to [ranks, n_rows, 5]), and the per-token fp32 loss
 * from them, with what the backward needs, both in `state`; the losses' mean in
 * mean[0] unless it is NULL.
 */
int nmce_distill_stats(const nmce_distill_batch* batch, void* state, int64_t state_bytes,
                       double* stats, void* stream);
int nmce_distill_combine(void* state, int64_t state_bytes, int64_t n_rows, int k,
                         double temperature, const double* stats, int ranks, float* loss,
                         float* mean, void* stream);

/*
 * One rank (ids from 0, no exchange), rows of at most NMCE_DISTILL_ONE_PASS_BYTES:
 * the loss, the state and the gradient of its mean for the upstream value
 * expected[0] (1 if that is zero, subnormal or not finite), which goes to
 * assumed[0], in one read of the logits; mean[0] too unless it is NULL.
 * gout_div: the token count. Rows of grad lie against 16-byte boundaries as the
 * logits' rows do; grad may be logits (ld_grad == ld).
 */
#define NMCE_DISTILL_ONE_PASS_BYTES 262144
int nmce_distill_fwd_bwd(const nmce_distill_batch* batch, void* grad, int64_t ld_grad, void* state,
                         int64_t state_bytes, float* loss, float* mean, const float* expected,
                         float* assumed, float gout_div, void* stream);

/*
 * grad = d loss / d logits of each row times grad_output[row * gout_stride] /
 * gout_div, over this shard; the state is the forward's. grad may be logits
 * (ld_grad == ld), else the two must not overlap. With `assumed` (one float; the
 * gradient is there for that upstream value) nothing is done where
 * grad_output[0] equals it, and observed[0] gets grad_output[0].
 */
int nmce_distill_bwd(const void* logits, void* grad, int dtype, int64_t n_rows,
                     int64_t vocab_local, int64_t ld, int64_t ld_grad, int k, double temperature,
                     void* state, int64_t state_bytes, const float* grad_output,
                     int64_t gout_stride, float gout_div, const float* assumed, float* observed,
                     void* stream);

/*
 * The GEMM core of the fused path, exposed for testing and measurement (no
 * counterpart in the reference): c[i, j] = sum_l a[i, l] * b[j, l] for
 * i < m, j < n, l < k, with bf16 a [m, lda] and b [n, ldb], fp32
 * accumulation, and c [m, ldc] written as c_dtype (NMCE_BF16 or NMCE_F32).
 * k must be a multiple of 64; a and b 16-byte aligned, lda and ldb multiples
 * of 8.
 */
int nmce_gemm_nt_bf16(const void* a, int64_t lda, const void* b, int64_t ldb, int64_t m,
                      int64_t n, int64_t k, void* c, int c_dtype, int64_t ldc, void* stream);

/*
 * The same core with b MN-contiguous, as the fused backward products read
 * their operands (no counterpart in the reference; for tests):
 * c[i, j] = sum_l a(i, l) * b[l, j] with b [k, ldb], and a[i, l] ([m, lda],
 * K-contiguous) or, when a_mn, a[l, i] ([k, lda], MN-contiguous); bf16 c.
 * MN-contiguous operands need ld >= (columns rounded up to 8), 64 * ld < 2^31.
 * Bit-identical to nmce_gemm_nt_bf16 on the transposed operands.
 */
int nmce_gemm_mn_bf16(int a_mn, const void* a, int64_t lda, const void* b, int64_t ldb,
                      int64_t m, int64_t n, int64_t k, void* c, int64_t ldc, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* NMCE_H */
