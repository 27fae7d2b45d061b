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
 * A row's position is clamped to [0, max_seq_len - 1]; head_dim <= 256 and max_seq_len <= 32768
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

int qlin_launch_rms_norm(const float *input, float *output, const uint16_t *weight, int weight_type, int rows,
                         int hidden_size, float eps, int one_plus);
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
