/* Decode-step kernels for a Gemma-2 style decoder, in libse12_gfx950.so.
 *
 * No counterpart in the reference: its runtime leaves everything but the
 * linear layers to the framework (.spec/features/model-integration/spec.md,
 * "Out of scope: changes to attention, KV cache or sampling"). These exist so
 * that an end-to-end decode step is a few launches around the fused SE12
 * products (se12_amd/gemma2.py), with the framework's BF16 rounding sequence.
 *
 * All pointers are device memory; every call is asynchronous on `stream`
 * (a hipStream_t), allocates nothing and is graph-capturable. Returns
 * SE12_STEP_OK or a negative code; se12_step_last_error() gives the message.
 */
#ifndef SE12_STEP_H
#define SE12_STEP_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define SE12_STEP_OK 0
#define SE12_STEP_E_INVALID (-1)
#define SE12_STEP_E_HIP (-2)

/* element type of an input tensor (outputs are always BF16) */
#define SE12_STEP_BF16 0
#define SE12_STEP_F32 1
/* element type of a paged cache besides SE12_STEP_BF16: 8 bits (OCP E4M3, no
 * infinities), one FP32 scale per page and KV head */
#define SE12_STEP_E4M3 2
/* and 4 bits (E2M1: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign), one 8-bit scale per 32
 * columns of a token and KV head */
#define SE12_STEP_E2M1 3

const char* se12_step_last_error(void);

/* mode 0: out = norm(x) * (1 + w1), x = in (rounded to BF16, times in_scale
 *         when in_scale != 0, e.g. sqrt(hidden) for Gemma's embedding); when
 *         residual is not NULL it receives x.
 * mode 1: residual = bf16(residual + norm(bf16(in)) * (1 + w1));
 *         out = norm(residual) * (1 + w2).
 * norm(x) = x * rsqrt(mean(x^2) + eps) in FP32. in: [rows, in_stride];
 * residual, out: [rows, hidden] BF16; w1, w2: [hidden] BF16; hidden <= 8192. */
int se12_step_rmsnorm(const void* in, int32_t in_dtype, int64_t in_stride, const uint16_t* w1, uint16_t* residual,
                      const uint16_t* w2, uint16_t* out, int32_t rows, int32_t hidden, float eps, float in_scale,
                      int32_t mode, void* stream);

/* One decode step of grouped-query attention at position *pos for every
 * sequence: q [batch, q_stride] (heads x head_dim used), k and v
 * [batch, kv_stride]; rotary embedding with inv_freq[head_dim / 2]; the
 * rotated key and the value are written to k_cache_t [batch, kv_heads,
 * head_dim, max_len] and v_cache [batch, kv_heads, max_len, head_dim] at
 * *pos; scores = (q . k) * scaling, soft-capped tanh(s / softcap) * softcap
 * when softcap > 0, over positions max(0, *pos - window + 1) .. *pos
 * (window 0 = all); softmax in FP32, probabilities rounded to BF16; out
 * [batch, heads * head_dim] BF16. head_dim a multiple of 8 up to 256;
 * max_len a multiple of 8; heads / kv_heads in {1, 2, 4, 8}; both caches
 * 16-byte aligned. A *pos outside [0, max_len) writes zeros to out and
 * nothing to the caches.
 *
 * Two launches over (sequence, KV head, 64-position chunk). `workspace`
 * (device, 256-byte aligned, se12_step_attention_workspace() bytes for the
 * shape) holds scores, chunk statistics, partial sums and arrival counters:
 * zero-fill it once before its first use; each call leaves the counters at
 * zero again. Calls sharing a workspace must not run concurrently. */
int64_t se12_step_attention_workspace(int32_t batch, int32_t heads, int32_t kv_heads, int32_t head_dim,
                                      int32_t max_len);

int se12_step_attention(const void* q, const void* k, const void* v, int32_t dtype, int64_t q_stride, int64_t kv_stride,
                        uint16_t* k_cache_t, uint16_t* v_cache, const float* inv_freq, const int64_t* pos, uint16_t* out,
                        int32_t batch, int32_t heads, int32_t kv_heads, int32_t head_dim, int32_t max_len, float scaling,
                        float softcap, int32_t window, void* workspace, int64_t workspace_bytes, void* stream);

/* out[r, c] = bf16(gelu_tanh(bf16(gate[r, c])) * bf16(up[r, c])); gate and up
 * [rows, stride], out [rows, cols]. */
int se12_step_gelu_mul(const void* gate, const void* up, int32_t dtype, int64_t stride, uint16_t* out, int32_t rows,
                       int32_t cols, void* stream);

/* Per row: z = bf16(logits) soft-capped (softcap > 0), stored to logits_out
 * [rows, vocab] when not NULL; the first index of the maximum goes to ids[row]
 * and to tokens[row * token_stride + *step] (skipped when *step is outside
 * [0, token_stride)). rows <= 65535.
 *
 * Blocks over slices of 2,048 logits per row; `workspace` (device, 256-byte
 * aligned, se12_step_logits_workspace() bytes) holds their partial results
 * and arrival counters: zero-fill it once before its first use; each call
 * leaves the counters at zero again. Calls sharing a workspace must not run
 * concurrently. */
int64_t se12_step_logits_workspace(int32_t rows, int32_t vocab);

int se12_step_logits_argmax(const void* logits, int32_t dtype, int64_t stride, int32_t rows, int32_t vocab, float softcap,
                            uint16_t* logits_out, int64_t* ids, int64_t* tokens, int64_t token_stride,
                            const int64_t* step, void* workspace, int64_t workspace_bytes, void* stream);

/* *pos += 1, *step += 1 (device counters of a captured decode loop). */
int se12_step_advance(int64_t* pos, int64_t* step, void* stream);

/* se12_step_logits_argmax followed by se12_step_advance, in one launch: once
 * every row's pick is stored (the rows read *step first), the last row's
 * final block sets *pos += 1 and *step += 1. Same workspace. Saves the
 * decode loop the advance launch; no counterpart in the reference, whose
 * sampling is the framework's. */
int se12_step_logits_argmax_advance(const void* logits, int32_t dtype, int64_t stride, int32_t rows, int32_t vocab,
                                    float softcap, uint16_t* logits_out, int64_t* ids, int64_t* tokens,
                                    int64_t token_stride, int64_t* step, int64_t* pos, void* workspace,
                                    int64_t workspace_bytes, void* stream);

/* Attention of a whole prompt: qkv [batch, tokens, stride] BF16 holds each
 * token's heads query heads, then kv_heads key and kv_heads value heads of
 * head_dim (64, 128 or 256). q (in place) and k are rotated (x cos +
 * rotate_half(x) sin, each product and the sum rounded to BF16; cos, sin
 * [tokens, head_dim] BF16), the keys and values written to the caches of
 * se12_step_attention at positions 0 .. tokens - 1, and out [batch, tokens,
 * heads * head_dim] BF16 = softmax(softcap tanh(q . k scaling / softcap)) v over
 * positions max(0, t - window + 1) .. t (window 0 = all), scores and sums in
 * FP32, probabilities rounded to BF16. 0 < softcap <= 64; max_len >= tokens and
 * a multiple of 8; stride a multiple of 8; tensors 16-byte aligned (out 8).
 * `workspace`: se12_step_prefill_workspace() bytes, contents indifferent; calls
 * sharing it must not run concurrently. Two launches; not for use under
 * concurrent writes to the caches. */
int64_t se12_step_prefill_workspace(int32_t batch, int32_t tokens, int32_t heads, int32_t kv_heads, int32_t head_dim);

int se12_step_prefill_attention(uint16_t* qkv, int64_t stride, const uint16_t* cos, const uint16_t* sin,
                                uint16_t* k_cache_t, uint16_t* v_cache, uint16_t* out, int32_t batch, int32_t tokens,
                                int32_t heads, int32_t kv_heads, int32_t head_dim, int32_t max_len, float scaling,
                                float softcap, int32_t window, void* workspace, int64_t workspace_bytes, void* stream);

/* A key/value cache in pages of page_size tokens (16, 32, 64 or 128), any page
 * of the pool for any part of any sequence:
 *   k [pages, kv_heads, page_size, head_dim]
 *   v [pages, kv_heads, head_dim, page_size]
 *   k_scale, v_scale [pages, kv_heads] FP32 (SE12_STEP_E4M3; else ignored): a
 *   held value stands for itself times the scale of its page and head, a positive
 *   number (se12_step_paged_append writes powers of two)
 * SE12_STEP_E2M1, two values to a byte, the first in its low half:
 *   k [pages, kv_heads, page_size, head_dim / 2]
 *   v [pages, kv_heads, page_size / 16, head_dim, 8]: 16 tokens of a column
 *   k_scale, v_scale uint8 [pages, kv_heads, head_dim / 32, page_size], 16-byte
 *   aligned: the byte's bits are bits 14 .. 7 of an FP16 number (5 of exponent, 3
 *   of fraction), which 32 columns of a token are times, 0 to 226 (10240); 255: one
 *   of the 32 is no number, and all of them count as NaN. (Of slots that hold no
 *   token the bytes may be any.)
 * head_dim 64, 128 or 256; k and v 16-byte aligned. */
typedef struct se12_step_pages {
    void* k;
    void* v;
    float* k_scale;
    float* v_scale;
    int32_t dtype;
    int32_t pages, page_size, kv_heads, head_dim;
} se12_step_pages;

/* The new tokens of a call. Sequence s holds lengths[s] tokens before it, and
 * rows starts[s] .. starts[s + 1] - 1 of q, k, v and out are its next ones, at
 * positions lengths[s], lengths[s] + 1, ..; token j of a sequence lies in slot
 * j % page_size of page page_table[s * table_stride + j / page_size]. starts
 * [sequences + 1] ascends from 0; `tokens` is the number of rows of q, k, v and
 * out (rows from starts[sequences] on are neither read nor written), max_new at
 * least the most new tokens of a sequence (of more, the first max_new count).
 * Lengths are 0 to 2^30 - 1 (others are taken as the nearer of these).
 * All device memory, read when the kernels run, so a captured call follows what
 * they hold then. No entry can lead outside the memory given: a page outside
 * [0, pages), or a position outside the table, holds nothing and takes nothing.
 * sequences * table_width and so on are up to the caller; table_width *
 * page_size <= 2^30, sequences <= 65536. */
typedef struct se12_step_batch {
    const int32_t* page_table;
    int64_t table_stride;
    const int32_t* lengths;
    const int32_t* starts;
    int32_t table_width, sequences, tokens, max_new;
} se12_step_batch;

/* Appends k and v [tokens, kv_heads, head_dim] to the cache, k rotated to its
 * position, and writes the rotated q [tokens, heads, head_dim] to q_out (BF16,
 * contiguous; q itself where that is both, else apart from q, and apart from k and
 * v); q may be NULL, then nothing is. Rows `q_stride`, `k_stride`, `v_stride`
 * elements apart (multiples of 4), heads of a row side by side; dtype
 * SE12_STEP_BF16 or SE12_STEP_F32 for all three, aligned to four elements. The
 * rotation takes the pair (x[i], x[i + rotary / 2]) by position * inv_freq[i],
 * i < rotary / 2 (the angle in 64 bits, the rest in FP32); elements from
 * `rotary` on stay (a multiple of 8 up to head_dim, 0 for none).
 *
 * SE12_STEP_BF16: values are rounded once. SE12_STEP_E4M3: a page and head's
 * scale is the least power of two, 2^-100 or more, that holds the new finite
 * values (largest / scale <= 448); where older tokens share the page it is at
 * least the scale they have, and if it grows they are rounded again to the new
 * one (powers of two: exact but for values that become subnormal). NaN and
 * infinities are held as NaN. Slots behind the new tokens keep their bytes. A
 * page that a call writes under two entries of the table (of two sequences, or of
 * one), or that a concurrent call reads or writes, has undefined contents.
 * SE12_STEP_E2M1: as se12_step_paged_append_rotated. */
int se12_step_paged_append(const se12_step_pages* pages, const se12_step_batch* batch, const void* q, const void* k,
                           const void* v, int32_t dtype, int64_t q_stride, int64_t k_stride, int64_t v_stride,
                           int32_t heads, const float* inv_freq, int32_t rotary, uint16_t* q_out, void* stream);

/* How q and k are made from a projection's rows, head by head:
 *   n = x rsqrt(mean(x^2) + eps) (offset + w) where a norm weight w [head_dim] (BF16
 *   or FP32, 16-byte aligned) is given, q_norm for q and k_norm for k, else x;
 *   the pairs (n[i], n[i + rotary / 2]), or (n[2 i], n[2 i + 1]) where interleaved,
 *   i < rotary / 2, by position * inv_freq[i], sine and cosine times `scale` (below
 *   2^127);
 *   elements from `rotary` on stay (a multiple of 8 up to head_dim, 0 for none).
 * Sums of squares and angles in 64 bits, the rest in FP32. */
typedef struct se12_step_rotation {
    const float* inv_freq;
    const void* q_norm;
    const void* k_norm;
    double scale, eps;
    float offset;
    int32_t norm_dtype, rotary, interleaved;
} se12_step_rotation;

/* se12_step_paged_append for a cache of SE12_STEP_E2M1, with norms and any rotation.
 * Of 32 columns of a token the scale is the one nearest to a sixth of the largest
 * value (ties to the even byte; at most 10240, so values beyond 61440 are held as
 * that, and where the largest is 1.5 * 2^-16 or less all are zero); a value the nearest code,
 * ties to even. 32 columns with a NaN or an infinity are held as NaN. A token's codes and
 * scales depend on that token alone. One launch. */
int se12_step_paged_append_rotated(const se12_step_pages* pages, const se12_step_batch* batch, const void* q, const void* k,
                                   const void* v, int32_t dtype, int64_t q_stride, int64_t k_stride, int64_t v_stride,
                                   int32_t heads, const se12_step_rotation* rotation, uint16_t* q_out, void* stream);

/* What a cache of any type holds of the batch's tokens (rows starts[s] .. of
 * positions lengths[s] ..): k and v [tokens, kv_heads, head_dim] BF16, contiguous, 16-byte
 * aligned, apart from each other; rounded once (exact from SE12_STEP_E2M1 and
 * SE12_STEP_BF16, and from SE12_STEP_E4M3 under power-of-two scales). A token
 * held nowhere gives zeros; rows of no sequence are not written. One launch. */
int se12_step_paged_read(const se12_step_pages* pages, const se12_step_batch* batch, uint16_t* k, uint16_t* v, void* stream);

/* The batch's q [tokens, heads, head_dim] and k [tokens, kv_heads, head_dim] (none
 * where kv_heads is 0) normed and rotated, into q_out and k_out (out_dtype BF16 or
 * FP32, contiguous, 16-byte aligned; each may be its input where that has the same
 * type and rows, else all apart). The batch's page table is not read. head_dim a multiple of
 * 8 up to 256; strides multiples of 4, rows aligned to 4 values. An append's q may differ
 * in FP32's last bit (its angles are sums from the first of 16). One launch. */
int se12_step_rotate_heads(const se12_step_batch* batch, const void* q, const void* k, int32_t dtype, int64_t q_stride,
                           int64_t k_stride, int32_t heads, int32_t kv_heads, int32_t head_dim,
                           const se12_step_rotation* rotation, void* q_out, void* k_out, int32_t out_dtype, void* stream);

/* Attention of the new tokens over their sequences' pages, those of the call
 * itself included (appended before): the query at position p sees keys
 * max(0, p - window + 1) .. p (window 0 = all). s = q . k * scaling, soft-capped
 * tanh(s / softcap) * softcap when softcap > 0 (2^-60 to 1024; held to 2^-22 of
 * it); softmax and sums in FP32, weights rounded to BF16 for the product with v.
 * q BF16 [tokens, heads, head_dim], rows q_stride apart (a multiple of 8), 16-byte
 * aligned, already rotated; out BF16 [tokens, heads, head_dim] contiguous, 8-byte
 * aligned, apart from q. heads a multiple of kv_heads. What a query may not see
 * has no part in its row, whatever it holds (NaN too); a query that sees nothing
 * gives zeros. Any finite values of BF16 pages give finite results, those of E4M3
 * pages where none is above 2^112 / keys. SE12_STEP_E2M1 pages: the products' operands
 * are FP16, which holds keys and values exactly, a query to 2^-38 of its largest value, and a
 * weight to 2^-11 of itself or 2^-32 of the row's largest; scores beyond FP32's range
 * keep their order.
 *
 * `workspace`: se12_step_paged_attention_workspace() bytes for the shape (or for
 * one of more tokens), 256-byte aligned, contents indifferent; calls sharing it
 * (two captured graphs too) must not run concurrently. Two launches, four where
 * max_new allows a sequence more than 64 (token, query head) pairs to a KV head;
 * results do not depend on timing. */
int64_t se12_step_paged_attention_workspace(const se12_step_pages* pages, const se12_step_batch* batch, int32_t heads);

int se12_step_paged_attention(const se12_step_pages* pages, const se12_step_batch* batch, const uint16_t* q,
                              int64_t q_stride, uint16_t* out, int32_t heads, float scaling, float softcap,
                              int32_t window, void* workspace, int64_t workspace_bytes, void* stream);

/* What a serving program reports of logits [rows, stride] (BF16 or FP32, vocab
 * of a row used), with z = softcap tanh(logit / softcap) when softcap > 0 (2^-60 to
 * 1024; held to 2^-22 of itself), else the logit, and p = softmax(z) in FP32:
 *   logprobs[r]  log p of tokens[r] (-inf for a token outside [0, vocab))
 *   entropy[r]   -sum p log p
 *   top_logprobs, top_ids [rows, top]  the `top` (0 .. 32) most likely tokens,
 *                by logit from the highest, equal ones by the lower index
 * A logit of -inf without a cap has no part in the sums; a row of nothing else
 * has log probabilities of -inf and entropy 0. A row with a NaN, or +inf without
 * a cap, has NaN for all but its ids, in whose order a NaN comes last.
 * `workspace`: se12_step_logprobs_workspace() bytes (may be 0), 16-byte aligned,
 * contents indifferent; calls sharing it must not run concurrently. */
int64_t se12_step_logprobs_workspace(int32_t rows, int32_t vocab, int32_t top);

int se12_step_logprobs(const void* logits, int32_t dtype, int64_t stride, int32_t rows, int32_t vocab, float softcap,
                       const int64_t* tokens, int32_t top, float* logprobs, float* entropy, float* top_logprobs,
                       int64_t* top_ids, void* workspace, int64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* SE12_STEP_H */
