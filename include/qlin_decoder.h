/*
 * qlin_decoder.h -- the glue around the quantized linears of a Qwen2-architecture decoder layer:
 * RMSNorm, rotary embedding with the KV-cache store, and causal grouped-query attention.
 *
 * These are not part of the quantized-linear path.  They let a whole decoder (benchmark configuration
 * C3, Qwen2.5-0.5B architecture with every linear in Q8_0) run its greedy decode on the path's kernels;
 * the linears, the embedding lookup and the argmax are the entry points of qlin.h.  Conventions as
 * in qlin.h: caller-owned device pointers, asynchronous on qlin_set_stream's stream, nothing
 * allocated, a qlin_status returned.
 *
 * Semantics restated from the reference engine (AI/codes/local-llm/src/backend/cuda/ops/):
 *   qlin_launch_rms_norm       launch_rms_norm (kernel.cuh:147-150, kernel.cu:112-150), same arguments:
 *                              y[r, j] = x[r, j] * rsqrt(mean_j x^2 + eps) * w[j], w bf16 (weight_type 0)
 *                              or f16 (1), plus one if one_plus.
 *   qlin_launch_rope_store_kv  the Qwen2 counterpart of launch_full_attention_q / _kv (kernel.cuh:162-184,
 *                              kernel.cu:186-340) without their q/k norms: rows at positions
 *                              *start_pos_dev + r; each head's pairs (i, i + head_dim/2) rotated by
 *                              pos / theta^(2i / head_dim); q in place, k rotated and v copied into the
 *                              caches [max_seq_len, kv_heads * head_dim] (f32) at the row's position.
 *   qlin_launch_attend         launch_full_attention_attend (kernel.cuh:186-189, kernel.cu:345-420) without
 *                              its output gate: attn[r, h] = softmax_j(q[r, h] . k[j, h / (n_heads /
 *                              kv_heads)] / sqrt(head_dim)) v[j, .] over positions j <= the row's.
 * A row's position is clamped to [0, max_seq_len - 1], and of the rows that a call has at one end then only the nearest is
 * stored (the one whose own position it is, if there is one); head_dim <= 256 and max_seq_len <= 32768
 * (else QLIN_ERR_LIMIT); n_heads a multiple of kv_heads and head_dim of 4 (else QLIN_ERR_SHAPE);
 * qlin_launch_attend reads q, the caches and attn as 16-byte vectors (16-byte aligned, else
 * QLIN_ERR_ALIGN).
 *
 * The RMSNorm fused into the decode linear that consumes it (no counterpart in the reference, whose
 * decode step runs launch_rms_norm and then launch_quant_gemv / launch_quant_swiglu on its output):
 *   qlin_launch_rms_norm_quant_gemv_multi  qlin_launch_quant_gemv_multi (one row, n_mats matrices that
 *                              share x) of rms_norm(x), the norm's arguments as qlin_launch_rms_norm's;
 *   qlin_launch_rms_norm_quant_swiglu      qlin_launch_quant_swiglu (gate and up of one row stride) of
 *                              rms_norm(x).
 * The decode kernels normalize x as they stage it (the normalized vector is not written), in one
 * launch instead of two.  They take the shapes of the matrix-core decode kernels (every format, in_dim
 * a multiple of 256, or 128 for Q8_0 and Q5_0, x 16-byte aligned); other shapes return
 * QLIN_ERR_LIMIT, for the two-launch form.
 *   qlin_launch_rope_attend    qlin_launch_rope_store_kv then qlin_launch_attend for one row (a decode
 *                              step), in one launch, with the same results: the rotated key and the
 *                              value are stored in the caches at the row's position as before, but q is
 *                              left as it is (the rotated q lives only in the launch).  Alignment as
 *                              qlin_launch_attend's for q, the caches and attn; k and v 4-byte aligned.
 *   qlin_launch_quant_gemv_argmax  the output head and the greedy pick: logits = W x, or W rms_norm(x) when
 *                              norm_weight is non-null, as qlin_launch_quant_gemv / ..._rms_norm_quant_gemv_multi
 *                              give them, then *out_idx as qlin_launch_argmax gives it for those logits (the
 *                              largest, the lowest index among equals, NaN never; 0 when nothing beats -inf).
 *                              Each workgroup of the GEMV reduces its own rows to one (value, index) pair in
 *                              scratch (QLIN_GEMV_ARGMAX_SCRATCH_BYTES of device memory, 4-byte aligned, used
 *                              by nothing else while the launches run), and one small launch reduces the pairs:
 *                              two launches instead of a GEMV and a one-workgroup scan of every logit.  Shapes
 *                              as the fused RMSNorm launches' (else QLIN_ERR_LIMIT); out_dim >= 1.
 */
#ifndef QLIN_DECODER_H
#define QLIN_DECODER_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- norms of queries and keys with the rotation, and an attention cache in 8 bits ---------------
 *
 * qlin_qk_rope says how a head of a query or key x becomes what the cache and the scores see:
 *   x'[j] = x[j] * (mean_j x^2 + eps)^(-1/2) * w[j]   over the head's head_dim values, with the weights q_norm
 *           or k_norm [head_dim] of norm_type 0 (bf16) or 1 (f16), plus one if one_plus; a NULL weight: x' = x;
 *   the first rotary_dim values of x' turned by the row table[p] of the position p, f32 cosines [rotary_dim / 2]
 *           and then sines: pairs (i, i + rotary_dim / 2), or (2i, 2i + 1) with pairing 1, become
 *           (a cos_i - b sin_i, b cos_i + a sin_i); the rest stays.  rotary_dim 0: no rotation (table unused).
 * Both are computed in 64 bits and rounded once.  The table (qlin_launch_rope_table, or a caller's own with
 * other frequencies) keeps far positions' angles exact, which powf and cosf of one f32 product do not.  Heads at a
 * position of the cache that the table does not have become NaN where they are turned (a position outside the cache is
 * taken as the nearest one in it).
 *
 * qlin_kv8_cache is one layer's cache of n_seqs sequences, up to blocks_per_seq blocks of QLIN_KV8_BLOCK
 * positions each (its capacity):
 *   - a block whose 32 positions are all there ("complete") is a record of 64 * head_dim + 16 bytes for each
 *     key head, pages[page][key head], in the page that block_table[seq][block] names (NULL table: page seq *
 *     blocks_per_seq + block).  Key codes (int8) come first: that of position t and dim 32 c + 8 g + j (j < 8) at
 *     byte 1024 c + 256 g + 16 (t % 16) + 8 (t / 16) + j.  Then, from byte 32 * head_dim, the value codes: that of
 *     position t and dim 4 e + j (j < 4), with w = e + (t % 2) * head_dim / 4, at byte 1024 (w / 16) + 256 (t / 4 % 4) +
 *     16 (w % 16) + 8 (t / 16) + 4 (t / 2 % 2) + j.  Then the two f32 scales, the keys' and the values', and 8 bytes
 *     that nothing reads or writes.
 *     scale = amax * (1.0f / 127.0f) over the 32 x head_dim values, code = clamp(round-to-even(x / scale), -127, 127),
 *     0 where the scale is 0; a block with a value that is not finite has scale NaN and codes 0.
 *   - recent holds the last positions in f32: [seq][key head][keys, values][64][head_dim], position p in row p % 64.
 *     The open block (the positions after the last complete block) is read from there.
 * So what a position's code is does not depend on whether its block came as a prompt or token by token, and
 * positions may be taken back: a store may start at a block's first position (0: another sequence), and from then on up
 * to 32 positions before the furthest end since (drafted tokens that were rejected), but not before that start.
 * A page number that is negative or >= n_pages, or a position outside [0, capacity), is not stored, and is not
 * seen by attention (a page taken out of the table is out of every score).  Sequences may share pages that none
 * of them is storing to.
 *
 * Rows come as [n_seqs, rows, heads, head_dim], row r of sequence s at position start_pos_dev[s] + r; with n_rows_dev
 * only the first n_rows_dev[s] (clamped to 0 .. rows) of them count: the others are not stored, and their outputs
 * stay as they were.  *_stride is the distance of a row's first head from the next row's, in
 * floats (>= heads * head_dim, so that q, k and v may be parts of one tensor); outputs are packed.
 * head_dim 64, 96, 128, 192 or 256 (else QLIN_ERR_LIMIT), pages and recent 16-byte aligned, blocks_per_seq <= 32768.
 *
 *   qlin_launch_rope_table      table[p][i], table[p][n / 2 + i] = cos, sin of p * theta^(-2i / n), n = rotary_dim, in
 *                               64 bits; n_pos rows.
 *   qlin_launch_qk_norm_rope_store_kv   q_out = the queries, and keys and values into the f32 caches of
 *                               qlin_launch_rope_store_kv, whose counterpart with norms it is (one sequence, positions
 *                               clamped as there, so that it is followed by qlin_launch_attend).  head_dim a
 *                               multiple of 8, <= 256.  q_out may be q (q_stride = n_heads * head_dim).
 *   qlin_launch_qk_norm_rope_store_kv8  the same into the 8-bit cache.
 *   qlin_launch_kv8_read        k_out, v_out [n_seqs, count, kv_heads, head_dim]: row r the values that position
 *                               first_dev[s] + r stands for, in a cache of lens_dev[s] positions; rows outside of it, or
 *                               of a page that the table does not have, stay as they were.
 *   qlin_launch_attend_kv8      attn[s, r, h] = sum_j p_j v_j, p = softmax_j(softmax_scale * q . k_j) over the positions
 *                               j <= the row's that the cache holds, which ends at start_pos_dev[s] + the sequence's rows
 *                               (their keys and values are stored first); heads and key heads as in qlin_launch_attend.
 *                               (A block that a later row of the call completes is seen in codes, whose scale is that of
 *                               all its positions.  Rows that must not depend on later ones, as those of drafted tokens, are
 *                               taken again by a second call whose n_rows_dev ends before the row that completes the block.)
 *                               A row that sees no position gives 0.  f32 accuracy: q softmax_scale log2(e) and p are
 *                               rounded to pairs of fp16 values, 22 bits and a sign each (what is below 2^-39 of a row's
 *                               largest q, or 2^-36 of its largest p, is lost), and their products with the codes are
 *                               exact; scores may be as large as f32 holds.  A row whose q softmax_scale log2(e) is beyond
 *                               f32 is NaN, and values are below 2^90 in magnitude.  workspace: qlin_attend_kv8_workspace_bytes(...) bytes, 16-byte aligned, used
 *                               by nothing else while the launches run (calls on one stream, or graphs that are not
 *                               replayed at the same time, may share it); its contents do not matter before or after.
 */
#define QLIN_KV8_BLOCK 32
#define QLIN_KV8_RECENT 64

typedef struct qlin_qk_rope {
    const uint16_t *q_norm, *k_norm; /* [head_dim], or NULL */
    int norm_type;                   /* 0 bf16, 1 f16 */
    float eps;
    int one_plus;
    const float *table;              /* [table_len, rotary_dim] */
    int table_len;                   /* positions 0 .. table_len - 1 */
    int rotary_dim;                  /* a multiple of 8, <= head_dim */
    int pairing;                     /* 0: (i, i + rotary_dim / 2), 1: (2i, 2i + 1) */
} qlin_qk_rope;

typedef struct qlin_kv8_cache {
    uint8_t *pages;         /* [n_pages, kv_heads, 64 * head_dim + 16] */
    float *recent;          /* [n_seqs, kv_heads, 2, QLIN_KV8_RECENT, head_dim] */
    const int *block_table; /* [n_seqs, blocks_per_seq], or NULL */
    int n_pages, n_seqs, blocks_per_seq, kv_heads, head_dim;
} qlin_kv8_cache;

/* ---- penalties, biases and a mask on logits, with the greedy pick --------------------------------
 *
 * qlin_launch_logits_controls: out[r, v] for a token v of row r from l = logits[r, v] and the count n of v among
 * history[r, 0 .. history_lens[r]):
 *   n > 0:  l > 0 ? l / repetition[r] : l * repetition[r];  then - frequency[r] * n;  then - presence[r]
 *   + the sum, in list order, of the bias_values[r, e] whose bias_ids[r, e] is v (if any is)
 *   -inf where bit v % 32 of mask[r * mask_stride + v / 32] is 0, whatever the above gives.
 * Every part is optional: history, bias_ids and mask NULL leave theirs out; history_lens NULL counts all max_history
 * tokens (a length is clamped to 0 .. max_history); repetition, frequency and presence NULL are 1, 0 and 0.  History
 * and bias ids outside [0, vocab) are no token's (padding).  repetition must be > 0.
 * picks (NULL: none): picks[r] as qlin_launch_argmax gives it for out[r] (the largest, the lowest index among equals,
 * NaN never; 0 when nothing beats -inf).
 * out may be logits itself (same pointer and stride), else they do not overlap.  Strides in floats, >= vocab.
 * scratch: qlin_logits_controls_scratch_bytes(rows, vocab) bytes, 4-byte aligned, needed only with picks, used by
 * nothing else while the launches run; its contents do not matter before or after.
 * vocab <= 1 << 28, max_history <= 1 << 20 and max_bias <= 4096 (else QLIN_ERR_LIMIT).
 */
typedef struct qlin_logits_controls {
    const int *history;      /* [rows, max_history] token ids, or NULL */
    const int *history_lens; /* [rows], or NULL */
    const float *repetition, *frequency, *presence; /* [rows] each, or NULL */
    const int *bias_ids;      /* [rows, max_bias], or NULL */
    const float *bias_values; /* [rows, max_bias] */
    const uint32_t *mask;     /* [rows, mask_stride], or NULL */
    size_t mask_stride;       /* in words, >= ceil(vocab / 32) */
    int max_history, max_bias;
} qlin_logits_controls;

/* ---- the residual's addition with the norm, into f32 or Q8_1 blocks ------------------------------
 *
 * qlin_launch_add_rms_norm, for each of rows rows of hidden values:
 *   s = x + delta (f32; delta NULL: s = x);   sum = s (sum NULL: not stored);
 *   y[j] = s[j] * (mean_j s^2 + eps)^(-1/2) * w[j], in 64 bits and rounded once, w of norm_type 0 (bf16) or 1 (f16), plus
 *   one if one_plus;   normed = y (NULL: not stored);
 *   q8_1 = the Q8_1 blocks of y (NULL: not stored), where qlin_launch_quantize_q8_1 (mmq 0) or qlin_launch_quantize_q8_1_mmq
 *   (mmq not 0) put theirs, with raw_sum as there.  The scale is the 8-bit cache's, d = amax * (1.0f / 127.0f), which is at
 *   most an f32 step from theirs, amax / 127.0f (of 2011 rows of 4096 3 codes of 8.2 million were one apart, no f16 scale); code = clamp(round-to-even(y * (1 / d)), -127, 127), 0 where d is below 2^-126; a block
 *   with a value that is not finite has scale NaN and codes 0.
 * normed or q8_1 or both.  *_stride: floats from a row to the next one, >= hidden.  sum may be x or delta (same pointer and
 * stride: the residual stream in place), and normed may be x or delta where sum is not; else outputs overlap nothing.
 * Norm weights 2-byte aligned, q8_1 and the rest 4-byte (else QLIN_ERR_ALIGN).  hidden <= 1 << 24, and rows < 1 << 22 (up to hidden
 * 4096 rows < 1 << 24) as what a launch holds (else QLIN_ERR_LIMIT).
 */

/* ---- low-rank adapters of many requests beside a shared projection -------------------------------
 *
 * qlin_launch_lora_add: for each row r with the adapter a = adapter_ids[r] and n_mats (1 .. 4) projections that read the same x,
 *   y[r, o] = base[r, o] + scales[a] * sum_{k < ranks[a]} B[a, o, k] * (sum_i A[a, k, i] x[r, i]).
 * A row whose id is negative or >= n_adapters has no adapter: y[r] = base[r].  y may be base (same pointer and stride: rows
 * without an adapter are then not touched), else it overlaps nothing.  Requests with adapters of their own stand in one
 * batch in any order, each adapter's weights are read for all the rows that have it.
 * The adapters stand in slots of max_rank: a [n_adapters, max_rank, in_dim] and b [n_adapters, out_dim, max_rank] of
 * weight_type 0 (bf16), 1 (f16) or 2 (f32).  ranks [n_adapters] (NULL: max_rank each; clamped to 0 .. max_rank) says how
 * much of a slot counts: the rest is not used, whatever it holds.  scales [n_adapters] or NULL (1).
 * Accuracy: exact products, sums in f32; A x is held in f32, then multiplied by the scale, and base is added to the sum in one
 * step.  bf16 and f16 weights are below 2^30 in magnitude, and sums of |A x| and |B z| below 2^100 (f32 weights, or an x or z of 2^60
 * or more: as far as f32 holds); an infinite weight gives NaN.  Infinities and NaN of x stay in their rows; a
 * row's result has the same bits whatever the others hold and wherever it stands among as many.
 * n_adapters >= 1, in_dim and max_rank are multiples of 8, from 8 on (else QLIN_ERR_SHAPE), max_rank <= 256, n_adapters <= 1024 and rows <= 65536 (else
 * QLIN_ERR_LIMIT); a and b 16-byte aligned, the rest 4-byte (else QLIN_ERR_ALIGN).  Strides in floats, >= the row.
 * workspace: qlin_lora_workspace_bytes(...) bytes, 16-byte aligned, used by nothing else while the launches run (calls
 * on one stream, or graphs that are not replayed at the same time, may share it); its contents do not matter before or after.
 * Fewer rows can take more of it.
 */
typedef struct qlin_lora {
    const void *a, *b;
    const float *base;
    float *y;
    size_t base_stride, y_stride;
    int out_dim;
} qlin_lora;

/* ---- drafted tokens against the target's probabilities -------------------------------------------
 *
 * qlin_launch_verify_drafts, for each of n_seqs sequences with n = n_drafts[s] drafted tokens x_0 .. x_{n-1} (n_drafts NULL:
 * max_drafts; clamped to 0 .. max_drafts):
 *   p_i = softmax(target row i / T), i <= n, and q_i = softmax(draft row i / T), i < n, T = temperature[s] (NULL: 1); without
 *     draft logits q_i is 1 at x_i (a draft by lookup).  T = 0 (or below, or NaN): all of it at the largest logit, the
 *     lowest index among equals;
 *   rates[s, i] = min(1, p_i(x_i) / q_i(x_i)) for i < n (where q_i(x_i) is 0: 1 if p_i(x_i) > 0, else 0), 0 after that;
 *   x_i is accepted if those before it were and uniform[s, i] * q_i(x_i) < p_i(x_i);
 *   accepted[s] = m, the number of accepted ones.  The next token y comes from max(p_m - q_m, 0) where x_m was rejected, and
 *     from p_n where all were accepted (from p_m, too, where the former is 0 everywhere): the first v at which the sum of
 *     the weights up to v is above uniform[s, max_drafts] times their sum over all v;
 *   tokens[s] = x_0 .. x_{m-1}, y, and -1 after that;  logprobs[s, i] = log p_i(tokens[s, i]) for i <= m, 0 after that.
 * So what comes out is distributed as the target alone would have it, and with max_drafts 0 the call is the draw of one
 * token for each sequence.  rates and logprobs may be NULL.
 * Everything is computed in 64 bits: a random number falls to one side of a border whatever the order of the sums is.
 * target [n_seqs, max_drafts + 1] rows and draft [n_seqs, max_drafts] rows of vocab logits, target_stride and draft_stride
 * floats from a row to the next (>= vocab); uniform [n_seqs, max_drafts + 1] in [0, 1) (below: 0; above: the largest f32
 * below 1; NaN: 0).  A logit that is NaN counts as -inf; tokens at +inf share a row's probability.  A row without any
 * logit above -inf accepts nothing; where y would come from it, y is 0 with logprob -inf.  A drafted token outside
 * [0, vocab) is not accepted (and by lookup takes nothing from p).
 * vocab <= 1 << 21, max_drafts <= 63, n_seqs < 1 << 22 and what the launches hold, 1 << 23 slices of rows (else QLIN_ERR_LIMIT).  Pointers 4-byte aligned, the workspace 16-byte
 * (qlin_verify_drafts_workspace_bytes(...) bytes; rules as qlin_launch_lora_add's).
 */

int qlin_launch_rms_norm(const float *input, float *output, const uint16_t *weight, int weight_type, int rows,
                         int hidden_size, float eps, int one_plus);
int qlin_launch_add_rms_norm(const float *x, size_t x_stride, const float *delta, size_t delta_stride, float *sum,
                             size_t sum_stride, const uint16_t *weight, int norm_type, float eps, int one_plus,
                             float *normed, size_t normed_stride, uint8_t *q8_1, int mmq, int raw_sum, int rows, int hidden);
size_t qlin_lora_workspace_bytes(int rows, int n_mats, int n_adapters, int max_rank, int in_dim);
int qlin_launch_lora_add(const qlin_lora *mats, int n_mats, int weight_type, int n_adapters, int max_rank, int in_dim,
                         const int *ranks, const float *scales, const float *x, size_t x_stride, const int *adapter_ids,
                         int rows, void *workspace, size_t workspace_bytes);
size_t qlin_verify_drafts_workspace_bytes(int n_seqs, int max_drafts, int vocab);
int qlin_launch_verify_drafts(const float *target, size_t target_stride, const float *draft, size_t draft_stride,
                              const int *drafts, const int *n_drafts, const float *temperature, const float *uniform,
                              int *tokens, int *accepted, float *logprobs, float *rates, int n_seqs, int max_drafts,
                              int vocab, void *workspace, size_t workspace_bytes);
int qlin_launch_rope_store_kv(float *q, const float *k, const float *v, float *key_cache, float *value_cache, int rows,
                              int n_heads, int kv_heads, int head_dim, int max_seq_len, const int *start_pos_dev,
                              float rope_theta);
int qlin_launch_attend(const float *q, const float *key_cache, const float *value_cache, float *attn, int rows,
                       int n_heads, int kv_heads, int head_dim, int max_seq_len, const int *start_pos_dev);
int qlin_launch_rope_attend(const float *q, const float *k, const float *v, float *key_cache, float *value_cache,
                            float *attn, int n_heads, int kv_heads, int head_dim, int max_seq_len,
                            const int *start_pos_dev, float rope_theta);
int qlin_launch_rms_norm_quant_gemv_multi(int type, int n_mats, const uint8_t *const *weights, size_t row_bytes,
                                          const float *x, const uint16_t *norm_weight, int norm_type, float eps,
                                          int one_plus, float *const *ys, const int *out_dims, int in_dim);
int qlin_launch_rms_norm_quant_swiglu(int type, const uint8_t *w_gate, const uint8_t *w_up, size_t row_bytes,
                                      const float *x, const uint16_t *norm_weight, int norm_type, float eps,
                                      int one_plus, float *act, int ffn_dim, int in_dim);
#define QLIN_GEMV_ARGMAX_SCRATCH_BYTES 8192
int qlin_launch_quant_gemv_argmax(int type, const uint8_t *weights, size_t row_bytes, const float *x,
                                  const uint16_t *norm_weight, int norm_type, float eps, int one_plus, float *logits,
                                  int out_dim, int in_dim, void *scratch, int *out_idx);
int qlin_launch_rope_table(float *table, int n_pos, int rotary_dim, float theta);
int qlin_launch_qk_norm_rope_store_kv(const qlin_qk_rope *how, const float *q, size_t q_stride, const float *k,
                                      size_t k_stride, const float *v, size_t v_stride, float *q_out, float *key_cache,
                                      float *value_cache, int rows, int n_heads, int kv_heads, int head_dim,
                                      int max_seq_len, const int *start_pos_dev);
int qlin_launch_qk_norm_rope_store_kv8(const qlin_qk_rope *how, const qlin_kv8_cache *cache, const float *q,
                                       size_t q_stride, const float *k, size_t k_stride, const float *v,
                                       size_t v_stride, float *q_out, int rows, int n_heads, const int *start_pos_dev,
                                       const int *n_rows_dev);
int qlin_launch_kv8_read(const qlin_kv8_cache *cache, const int *first_dev, const int *lens_dev, int count,
                         float *k_out, float *v_out);
size_t qlin_attend_kv8_workspace_bytes(int n_seqs, int rows, int n_heads, int kv_heads, int head_dim,
                                       int blocks_per_seq);
int qlin_launch_attend_kv8(const qlin_kv8_cache *cache, const float *q, float *attn, int rows, int n_heads,
                           const int *start_pos_dev, const int *n_rows_dev, float softmax_scale, void *workspace,
                           size_t workspace_bytes);
size_t qlin_logits_controls_scratch_bytes(int rows, int vocab);
int qlin_launch_logits_controls(const qlin_logits_controls *controls, const float *logits, size_t logits_stride,
                                float *out, size_t out_stride, int rows, int vocab, int *picks, void *scratch,
                                size_t scratch_bytes);

#ifdef __cplusplus
}
#endif

#endif /* QLIN_DECODER_H */
