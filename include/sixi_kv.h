/*
 * sixi_kv.h - C ABI of the 8-bit paged key/value cache that sits before the logits-to-token path of
 * sixi_smp.h: rotary positions, writing the cache, reading it back, and attention over it for one or
 * several new tokens per sequence (a decode step, the 1 + k rows of speculative verification, a
 * chunk of a prompt). It has no counterpart in the engine, whose model execution is external.
 *
 * Conventions are those of sixi_smp.h: `extern "C"`, int32 status codes (the engine's ErrorCode
 * values), array arguments are DEVICE pointers aligned to their elements, every call is asynchronous on the caller's stream
 * and neither synchronises nor allocates (create excepted), and failures of a single sequence are
 * reported in out_status without affecting the other sequences. A cache handle owns a workspace: its
 * calls are serialised by the caller (one stream, or streams ordered by events). A rotary handle is
 * only read: several threads and streams may use one at a time.
 */
#ifndef SIXI_KV_H
#define SIXI_KV_H

#include <stddef.h>
#include <stdint.h>

#include "sixi_smp.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * The cache. Keys and values live in pages of `page_size` tokens, in buffers of the caller's:
 *   k_pages, v_pages    [n_pages][n_kv_heads][page_size][head_dim] bytes, e4m3 (4 exponent bits, bias
 *                       7, 3 mantissa bits, largest value 448, no infinities)
 *   k_scales, v_scales  [n_pages][n_kv_heads] fp32; a cached value is its byte's value times the
 *                       scale of its page and head
 * Scales are powers of two: 2^e with the least e >= -126 such that the largest magnitude written to
 * the page is at most 448 * 2^e. Multiplying by them is exact, and e4m3 is a floating-point format,
 * so a finer scale would not make the stored values more precise.
 */
typedef struct sixi_kv_config {
    uint32_t n_pages;
    uint32_t page_size;   /* tokens per page: 16, 32, 64 or 128 */
    uint32_t n_kv_heads;  /* 1..1024 */
    uint32_t head_dim;    /* a multiple of 16, 16..256 */
    uint32_t max_seqs;    /* most sequences of one call, 1..65535 */
    uint32_t reserved;
} sixi_kv_config;

typedef struct sixi_kv sixi_kv; /* opaque handle */

/* Binds a cache to `device` and the caller's buffers (pages 16-byte aligned; they must outlive the
 * handle), and allocates the workspace. The buffers' contents are not touched: pages need no
 * initialisation, whatever they hold beyond a sequence's length never reaches a result. */
SIXI_SMP_API int32_t sixi_kv_create(int32_t device, const sixi_kv_config* config, void* k_pages, void* v_pages,
                                    float* k_scales, float* v_scales, sixi_kv** out);
SIXI_SMP_API int32_t sixi_kv_destroy(sixi_kv* h);

/* Rows of heads: element (token t, head j, i) is data[t * token_stride + j * head_stride + i]; dtype
 * SIXI_SMP_F32 or SIXI_SMP_BF16, data aligned to its element size. */
typedef struct sixi_kv_tensor {
    void* data;
    uint32_t dtype;
    uint32_t n_heads;
    uint64_t token_stride; /* elements */
    uint64_t head_stride;  /* elements */
} sixi_kv_tensor;

/*
 * The tokens a call works on: for each sequence s the last n_s = offsets[s + 1] - offsets[s] of its
 * lens[s] positions. Token i of sequence s is row offsets[s] + i of the call's tensors and stands at
 * position lens[s] - n_s + i, in page page_table[s * table_stride + position / page_size].
 * The same batch serves an append and the attention that follows it: lens counts the new tokens.
 * After verification has kept a of the k drafted tokens of a stream, its next lens continues from
 * lens - k + a: positions behind it are written over by the next append. What a rejected token leaves is
 * the scale of its page, where it raised it (see sixi_kv_append): older tokens of that page stay as they
 * were rounded at it, until the page is written from its first slot again.
 */
typedef struct sixi_kv_batch {
    const int32_t* page_table;
    uint64_t table_stride;   /* entries between sequences, >= max_pages */
    const int64_t* offsets;  /* [n_seqs + 1], offsets[0] = 0, not decreasing */
    const int32_t* lens;     /* [n_seqs] */
    uint32_t n_seqs;         /* <= max_seqs */
    uint32_t max_pages;      /* page-table entries per sequence; max_pages * page_size <= 2^30 */
    uint32_t n_tokens;       /* offsets[n_seqs] */
    uint32_t max_new;        /* the largest n_s (picks a variant; results do not depend on it) */
} sixi_kv_batch;

/*
 * Rotary positions. Pair i < rot_dim / 2 of a head's first rot_dim elements, (x[i], x[i + rot_dim / 2])
 * in the half layout and (x[2i], x[2i + 1]) in the interleaved one, turns by position * f_i:
 *   (a, b) -> amp * (a cos - b sin, b cos + a sin)
 * The elements from rot_dim on are passed through. f_i = base^(-2i / rot_dim), and for long contexts
 *   LINEAR  f_i / factor
 *   NTK     base * factor^(rot_dim / (rot_dim - 2)) in the place of base
 *   YARN    f_i / factor * r_i + f_i * (1 - r_i), r_i = clamp((i - lo) / max(hi - lo, 0.001), 0, 1),
 *           lo = max(0, floor(d(beta_fast))), hi = min(rot_dim - 1, ceil(d(beta_slow))),
 *           d(t) = rot_dim ln(original_max_position / (2 pi t)) / (2 ln base)
 * amp is 1, and 0.1 ln(factor) + 1 for YARN. Angles are held as 64-bit fractions of a turn, so they
 * are as accurate at position 10^9 as at position 1.
 */
enum { SIXI_KV_ROPE_HALF = 0, SIXI_KV_ROPE_INTERLEAVED = 1 };
enum { SIXI_KV_ROPE_NONE = 0, SIXI_KV_ROPE_LINEAR = 1, SIXI_KV_ROPE_NTK = 2, SIXI_KV_ROPE_YARN = 3 };
typedef struct sixi_kv_rope_config {
    uint32_t rot_dim; /* even, 2..256 (4..256 for NTK) */
    uint32_t layout;
    uint32_t scaling;
    uint32_t original_max_position; /* YARN, >= 1 */
    double base;                    /* > 1 */
    double factor;                  /* >= 1 (LINEAR, NTK, YARN) */
    double beta_fast;               /* YARN (32 is usual) */
    double beta_slow;               /* YARN (1 is usual), <= beta_fast */
} sixi_kv_rope_config;

typedef struct sixi_kv_rope sixi_kv_rope; /* opaque: the frequencies, on the host and on the device */

SIXI_SMP_API int32_t sixi_kv_rope_create(int32_t device, const sixi_kv_rope_config* config, sixi_kv_rope** out);
SIXI_SMP_API int32_t sixi_kv_rope_destroy(sixi_kv_rope* r);

/*
 * Turns n_tokens rows of x by positions[t] into out (same dtype and heads; out may be x itself, and
 * otherwise may not overlap it). inverse != 0 turns back: with the same amp, it is the gradient of
 * the forward call, and without scaling it undoes it. head_dim >= rot_dim, at most 65,536.
 */
SIXI_SMP_API int32_t sixi_kv_rope_apply(const sixi_kv_rope* r, const sixi_kv_tensor* x, const int32_t* positions,
                                        uint32_t n_tokens, uint32_t head_dim, uint32_t inverse,
                                        const sixi_kv_tensor* out, void* stream);

/*
 * Writes the batch's keys and values (k, v: [n_tokens][n_kv_heads][head_dim]) to their pages, the
 * keys turned by their positions first when rope is not NULL (in 32 bits; they are rounded once).
 * A page that the call writes from its first slot gets the scale of the new tokens. A page that
 * holds older tokens of its sequence keeps the larger of its scale and the new tokens'; where that
 * grows, the older values are rounded again at it (exact unless they fall below 2^-6 of the scale).
 * NaN is written as 0 and +-Inf as +-448 * scale, scaled without them, as the clamp policy of
 * sixi_smp_numeric_policy does; out_status[s] = SIXI_NUMERIC_NAN_OR_INF then. It is
 * SIXI_OUT_OF_BOUNDS when the sequence's numbers or a page id do not fit (negative or beyond
 * n_pages, lens beyond max_pages * page_size, more new tokens than lens): nothing is written for bad
 * ids or numbers. Offsets that are negative, decrease or pass n_tokens leave no sequence its rows: every
 * sequence of the call reports it, and nothing is written. Pages of different sequences must differ
 * where they are written.
 */
SIXI_SMP_API int32_t sixi_kv_append(sixi_kv* h, const sixi_kv_tensor* k, const sixi_kv_tensor* v,
                                    const sixi_kv_batch* batch, const sixi_kv_rope* rope, int32_t* out_status,
                                    void* stream);

/*
 * Reads the batch's positions back: k and v [n_tokens][n_kv_heads][head_dim] as the values they stand
 * for (exact in fp32 and, within its range, in bf16). Rows of a sequence that reports
 * SIXI_OUT_OF_BOUNDS in out_status (as sixi_kv_append) are zero where its page id is bad, and
 * untouched where its numbers are.
 */
SIXI_SMP_API int32_t sixi_kv_read(sixi_kv* h, const sixi_kv_batch* batch, const sixi_kv_tensor* k,
                                  const sixi_kv_tensor* v, int32_t* out_status, void* stream);

/*
 * Attention of the batch's queries q [n_tokens][n_q_heads][head_dim] over their sequences' cached
 * tokens, the new ones included (append them first). Query head j reads key head j / (n_q_heads /
 * n_kv_heads); a query at position p attends to the positions t with
 *   t < lens, t <= p (unless SIXI_KV_ATTEND_ALL), and t > p - window (window > 0)
 *   s_t = scale * q . k_t,  out = sum_t exp(s_t - lse) v_t,  lse = ln sum_t exp(s_t)
 * A row that no position is left for gives out = 0 and lse = -inf. q is turned by its positions first
 * when rope is not NULL and rounded to its dtype, as sixi_kv_rope_apply would. A NaN or Inf in a query
 * makes its own row NaN only. Cached tokens inside a sequence's length must be finite (appended ones are).
 *   out       [n_tokens][n_q_heads][head_dim] of q's dtype
 *   out_lse   [n_tokens][n_q_heads] fp32 (natural logarithm), or NULL
 *   out_status [n_seqs]: SIXI_OUT_OF_BOUNDS for a sequence whose numbers (as sixi_kv_append; but lens
 *             may be below n_s, such rows are empty) or needed page ids do not fit; its out rows are
 *             unspecified. SIXI_BACKEND_ERROR for all if a wait inside a kernel ever runs out (and
 *             from then on for every call of the handle)
 * n_tokens * n_q_heads / n_kv_heads < 2^30, and the call's tiles of 8 rows by 64 positions < 2^40.
 * Queries and keys may have any finite magnitudes whose scores are within fp32's range. Values are
 * summed before they are divided by the weights' sum: what a row's |v_t| add up to has to stay within it too.
 * Pages that lie wholly before every row's window are not read, and their table entries may be anything.
 * Sums and softmax statistics are fp32. With fp32 queries everything is. With bf16 queries the products
 * run on the tensor cores straight from the cached bytes, and the weights exp(s_t - m) enter theirs
 * rounded: 8 significant bits (as bf16 weights would have) for those above 2^-13 of the largest of
 * their tile (positions 128 i to 128 i + 127), and an error of 2^-21.6 of that largest weight at most for
 * smaller ones. That is less than the output's own rounding, unless the tokens with the large weights
 * have values near zero and only the small ones' sum is left (fp32 queries keep it).
 */
enum { SIXI_KV_ATTEND_ALL = 1u };
SIXI_SMP_API int32_t sixi_kv_attend(sixi_kv* h, const sixi_kv_tensor* q, const sixi_kv_batch* batch, float scale,
                                    uint32_t window, uint32_t flags, const sixi_kv_rope* rope,
                                    const sixi_kv_tensor* out, float* out_lse, int32_t* out_status, void* stream);

#ifdef __cplusplus
} /* extern "C" */
#endif

#endif /* SIXI_KV_H */
