/*
 * litenn_kv.h — C ABI of the paged key/value cache: rotary positions applied while keys and values are
 * appended to pages, and attention that reads the pages, in fp16 or in GGUF's 8-bit and 4-bit blocks.
 *
 * LiteNN grows a cache by concatenation (src/LiteNN/Layer/KVCache.h:85-102), rotates with fp32 tables
 * (Layer/RoPE.h:22-117) and attends over the whole of it (Layer/FlashAttnExt.h:100-229).  Here the cache
 * lives in pages that a sequence takes as it grows, quantized by the same block rules as the weights:
 * a token of a head of 128 costs 144 bytes in Q4_0 where fp16 costs 512.
 *
 * Conventions are those of litenn_qmm.h: int status codes, qmm_last_error(), streams as void*, calls only
 * enqueue, *_dev pointers are on `device`.  Calls can be captured into a graph; the first one on a device makes its
 * status word (qmm_kernel_status) and comes before any capture.  Nothing else is allocated.
 *
 * The pool is caller-owned memory of qmm_kv_pool_bytes() bytes, 16-byte aligned, laid out
 *   [page][kv head][page_tokens / 16] tiles
 * so a page is one run of bytes that can be copied or moved.  A tile holds 16 consecutive tokens of one kv
 * head in four planes, one after the other: key quants, key scales, value quants, value scales.  With
 * NB = head_dim / 32 blocks, U = 4, 8, 16 bytes per eight values (Q4_0, Q8_0, fp16), L = NB * U bytes per
 * lane, V = 16, 8 or 4, the largest that divides L:
 *   quant plane  64 * L bytes.  Eight values that one lane of an attention warp multiplies lie together: byte x
 *                (0 <= x < U, of block b) of lane p (0..31), half j (0, 1) is byte
 *                j * 32 * L + (X / V) * 32 * V + p * V + X % V,  X = b * U + x.
 *       keys     token 8j + (p >> 2), dimension 32b + 8(p & 3) + 2r + e
 *       values   token 8j + 2(p & 3) + e, dimension 32b + 4(p >> 2) + r,      0 <= r < 4, 0 <= e < 2
 *       the value (r, e) is the fp16 at x = 2(2r + e), the byte q + 128 at x = 2r + e (Q8_0), or the nibble
 *       q + 8 at x = (r >> 1) + 2e, shifted by 4(r & 1) (Q4_0).
 *   scale plane  (Q4_0, Q8_0 only) 32 * NB bytes: fp16 scale of token 8j + 2t + e, block b, is number
 *                ((t * 2 + j) * NB + b) * 2 + e.
 * A value is q * scale.  Blocks are made as GGUF makes them, in fp32: Q4_0 d = m / -8 where m is the value of
 * largest magnitude (the first of equals), q + 8 = min(15, floor(x * (1 / d) + 8.5)); Q8_0 d = max|x| / 127, q =
 * x * (1 / d) rounded half away from zero.  |d| is held to 8188 and 515.5, so that every value lies within fp16's
 * range (larger ones saturate); a block with an infinity or a NaN gets a NaN scale and reads as NaN.  An fp16 cache holds
 * values rounded to fp16: past its range they are infinities.
 */
#ifndef LITENN_KV_H
#define LITENN_KV_H

#include "litenn_qmm.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Cache formats: QMM_FMT_Q4_0, QMM_FMT_Q8_0, or fp16. */
#define QMM_KV_F16 0

/* Element types of the rows: QMM_OUT_F32, QMM_OUT_BF16 (litenn_qmm.h). */

/* Bytes of workspace that qmm_kv_attention may use. */
#define QMM_KV_WORKSPACE_BYTES (16 * 1024 * 1024)

typedef struct qmm_kv_cache {
    int32_t fmt;         /* QMM_KV_F16, QMM_FMT_Q8_0, QMM_FMT_Q4_0 */
    int32_t kv_heads;
    int32_t head_dim;    /* 64, 96, 128 or 256 */
    int32_t page_tokens; /* tokens per page, a multiple of 16 */
    int64_t n_pages;
    void* pool_dev;
} qmm_kv_cache;

/* Which rows of a call belong to which sequence, and where the sequence's tokens are.  Row i of the n rows of
 * sequence s is the token at position kv_len[s] - n + i: kv_len counts the rows of the call.
 * The arrays (4-byte aligned) are read on the device when the call runs, so a captured call sees their values at replay.  What
 * cannot be right (a page outside the pool, rows outside the tensors, a length outside the table) is skipped and
 * reported through qmm_kernel_status: 21 a page, 22 rows or a length. */
typedef struct qmm_kv_batch {
    int32_t batch;                 /* sequences */
    int32_t table_width;           /* page numbers per sequence */
    const int32_t* page_table_dev; /* [batch][table_width]; entries past a sequence's length are not read */
    const int32_t* kv_len_dev;     /* [batch] */
    const int32_t* row_begin_dev;  /* [batch + 1] first row of each sequence, rising; NULL: one row per sequence */
    int64_t rows;                  /* rows of the tensors; those from row_begin[batch] on are left alone */
} qmm_kv_batch;

/* Rotary positions.  Pair i < dim / 2 of a head is turned by position * inv_freq[i]: (x, y) -> gain * (x cos - y sin,
 * x sin + y cos).  The angle and the product are taken in 64 bits and rounded to fp32 once. */
#define QMM_ROPE_PAIRS 0  /* pair i = dimensions 2i, 2i + 1 (Layer/RoPE.h:22-117) */
#define QMM_ROPE_HALVES 1 /* pair i = dimensions i, i + dim / 2 */
typedef struct qmm_rope {
    int32_t dim;    /* rotated dimensions, the first of the head; even, for QMM_ROPE_HALVES a multiple of 8; 0: none */
    int32_t layout; /* QMM_ROPE_PAIRS, QMM_ROPE_HALVES */
    const double* inv_freq_dev; /* [dim / 2] */
    double gain;
} qmm_rope;

/* How a context longer than the trained one is reached. */
#define QMM_ROPE_SCALE_NONE 0
#define QMM_ROPE_SCALE_LINEAR 1 /* every frequency / factor */
#define QMM_ROPE_SCALE_YARN 2   /* YaRN: pairs that turn more than beta_fast times over `trained` positions keep their
                                   frequency, below beta_slow it is / factor, a ramp between; gain 0.1 ln(factor) + 1 */
typedef struct qmm_rope_scaling {
    int32_t kind;
    float factor;    /* >= 1 */
    float trained;   /* YaRN: positions the model was trained on */
    float beta_fast; /* YaRN: usually 32 */
    float beta_slow; /* YaRN: usually 1 */
} qmm_rope_scaling;

/* Host helper: inv_freq_out[i] = theta^(-2i / dim), divided by factors[i] (GGUF's rope_freqs.weight; may be NULL), then
 * scaled (scaling may be NULL). */
int qmm_rope_frequencies(int dim, double theta, const float* factors, const qmm_rope_scaling* scaling,
                         double* inv_freq_out, double* gain_out);

/* Bytes of the pool of a cache (pool_dev is not looked at). */
int qmm_kv_pool_bytes(const qmm_kv_cache* cache, size_t* bytes);

/*
 * Rotates the rows' queries and keys and stores keys and values in their pages.
 *   type            element type of q, k and v
 *   q [rows, heads * head_dim], k and v [rows, kv_heads * head_dim], row strides in elements; one fused
 *                   projection is three pointers into the same rows.  q may be NULL (heads 0).
 *   q_out           rotated queries of type q_type; may be q itself, or lie apart from q, k and v
 *   rope            may be NULL: nothing is rotated
 * Pointers are 16-byte aligned and strides whole multiples of 16 bytes.  A page that is written to belongs to one
 * sequence of the batch.
 */
int qmm_kv_append(int device, const qmm_kv_cache* cache, const qmm_kv_batch* batch, const qmm_rope* rope, int heads,
                  int type, const void* q_dev, int64_t q_stride, const void* k_dev, int64_t k_stride,
                  const void* v_dev, int64_t v_stride, void* q_out_dev, int q_type, int64_t q_out_stride, void* stream);

/* What the cache holds for the rows' tokens: k_out and v_out [rows, kv_heads * head_dim] of `type`. */
int qmm_kv_read(int device, const qmm_kv_cache* cache, const qmm_kv_batch* batch, void* k_out_dev, int64_t k_stride,
                void* v_out_dev, int64_t v_stride, int type, void* stream);

/*
 * Attention of the rows over their sequences' pages: out = softmax(scale * q . K) V over the tokens at or before the
 * row's position (the last `window` of them if window > 0).  `heads` query heads share kv_heads, head h reads kv head
 * h / (heads / kv_heads).  A row that sees no token gives zeros.  Tokens that a row does not see do not reach it,
 * whatever their pages hold.  A value that is not finite (in quants its block of 32) makes its dimensions of the rows that
 * see it infinite or NaN, and no others.
 *   q [rows, heads * head_dim] of q_type, out the same shape of out_type.  fp32 results carry fp32's precision (scores
 *   and probabilities go through the tensor cores in two fp16 parts each, probabilities times a block's scale relative
 *   to the largest scale among the tokens: a value 2^-k of the largest keeps 28 - k bits); bf16 results of long prompts
 *   are computed with fp16 operands.
 *   workspace       QMM_KV_WORKSPACE_BYTES bytes, 256-byte aligned, zeroed once before their first use and left
 *                   zeroed where it matters by every call.  Calls that may run at the same time need one each.
 * Which kernel a call runs goes by its shape on the host: `rows` (all that the tensors have room for), heads and types, not by
 * lengths.  bf16 results of many rows go to one that reads a sequence's tokens once for 256 rows times heads, and does not
 * split them: long histories of few rows, single tokens above all, belong in a call of their own.
 * Pointers are 16-byte aligned and strides whole multiples of 16 bytes; out may not overlap q.
 */
int qmm_kv_attention(int device, const qmm_kv_cache* cache, const qmm_kv_batch* batch, int heads, const void* q_dev,
                     int q_type, int64_t q_stride, void* out_dev, int out_type, int64_t out_stride, float scale,
                     int window, void* workspace_dev, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* LITENN_KV_H */
