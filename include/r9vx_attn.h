/*
 * r9vx_attn.h -- attention over a paged key-value cache on MI355X: rotary
 * positions and the write into the cache, attention of the next tokens
 * (decode) and of prompts (prefill).  The operators between a layer's
 * projections (r9vx_matmul_launch, r9vx_matmul_fp8_launch); no counterpart in
 * the reference's device tier for this path.
 *
 * Conventions are r9vx.h's: caller-owned buffers and workspaces, nothing
 * allocated in a launch, stream order, refusals before anything is enqueued,
 * r9vx_last_error().  Strides are in elements; the last axis is dense.
 *
 * The cache.  Keys and values stand in pages of page_size tokens, each
 * [pages, page_size, kv_heads, head_dim] with strides of its own for pages,
 * tokens and heads (so [pages, kv_heads, page_size, head_dim], or keys and
 * values in one allocation, are read as well).  Token j of sequence b is at
 * place j % page_size of page table[b, j / page_size]; slot s of the whole cache
 * is place s % page_size of page s / page_size.  Query head h reads kv head
 * h / (heads / kv_heads).
 *
 * Attention.  A sequence of length L holds its new tokens already: the last n of
 * it are the queries, token i of them at position p = L - n + i.
 *     s[j] = scale * q . k[j];  softcap: s[j] = softcap * tanh(s[j] / softcap)
 *     slopes: s[j] -= slopes[h] * |p - j|
 *     seen: max(start, window ? p - window + 1 : 0) <= j,
 *           j < (causal ? min(L, max(p + 1, prefix)) : L)
 *     out = sum over the seen j of softmax(s)[j] * v[j]
 * A query that sees no key gets zeros.  What is not seen has no part in a row,
 * whatever its place in the cache holds (NaN and infinities too); a NaN that is
 * seen, or a softmax that is none (+infinity, all -infinity), makes the row NaN.  An
 * infinite value that is seen makes its column infinite, however small its probability.
 *
 * Numbers.  Products are summed in f32; scores, their maximum and sum are f32.
 * Probabilities are rounded to the cache's type before they are multiplied with
 * values (by up to 2^-8 of each for bf16, 2^-11 for f16: as much again as the
 * output's own rounding); attn_decode keeps a bf16 probability as two bf16
 * numbers.  One rounding to the output.  A cap adds up to 5 * 2^-23 of itself to a
 * score's error, one above 128 at most 21 * 2^-23 of the score; one above 2^100 is
 * taken as 2^100.
 *
 * Faulty data.  A page that is not in the cache, or a length below 0 or above
 * len_bucket, makes that sequence's outputs NaN, as far as they were to see it,
 * and leaves the others; or-ed into a status word of the caller's (or NULL),
 * which no launch clears.
 */
#ifndef R9VX_ATTN_H_
#define R9VX_ATTN_H_

#include "r9vx.h"

#ifdef __cplusplus
extern "C" {
#endif

#define R9VX_STATUS_BAD_PAGE 8u    /* a page of the table outside the cache */
#define R9VX_STATUS_BAD_LENGTH 16u /* a length or an offset outside its range */
#define R9VX_STATUS_BAD_SLOT 32u   /* a slot outside the cache */

/* ---------------------------------------------------------------- rope */

typedef struct r9vx_rope_kv_static {
    uint32_t heads;          /* query heads, 1 .. 1024 */
    uint32_t kv_heads;       /* 0: queries alone, no cache */
    uint32_t head_dim;       /* a multiple of 8, at most 512 */
    uint32_t rot;            /* leading columns that turn: a multiple of 16, at most head_dim */
    uint32_t interleaved;    /* pairs: 0 columns i and i + rot / 2, 1 columns 2i and 2i + 1 */
    uint32_t page_size;      /* a power of two (with kv_heads) */
    uint32_t in_dtype;       /* F32, BF16 or F16 */
    uint32_t out_dtype;      /* of q_out and the cache: in_dtype's, or BF16 or F16 of F32 */
    uint32_t amplitude_bits; /* f32: factor on cosine and sine */
} r9vx_rope_kv_static;

typedef struct r9vx_rope_kv_args {
    const void *q;            /* [t, heads, head_dim] */
    const void *k;            /* [t, kv_heads, head_dim] */
    const void *v;            /* [t, kv_heads, head_dim] */
    const int32_t *positions; /* [t] */
    const double *freqs;      /* f64 [rot / 2]: radians a position */
    void *q_out;              /* [t, heads, head_dim]; may be q with q's strides where the types agree */
    void *k_cache;            /* written at slots alone */
    void *v_cache;
    const int64_t *slots;     /* [t]: k's and v's place in the cache; -1: nowhere */
    uint32_t *status;         /* or NULL */
    uint64_t q_stride[2];     /* of a token, of a head */
    uint64_t k_stride[2];
    uint64_t v_stride[2];
    uint64_t q_out_stride[2];
    uint64_t k_cache_stride[3]; /* of a page, of a token, of a head */
    uint64_t v_cache_stride[3];
    uint32_t pages;
    uint32_t t;
} r9vx_rope_kv_args;

/* One launch: q and k turned by position * freqs (the angle in f64, its cosine
 * and sine in f32, one rounding of the result), q to q_out, k and v (copied) to
 * their slots.  Columns from rot on are copied.  A slot other than -1 outside
 * the cache writes nothing and sets R9VX_STATUS_BAD_SLOT; of two rows with one
 * slot either may be kept, 16 bytes by 16 bytes.  Pointers 16-byte aligned,
 * strides such that every head is; rows of q_out, of k_cache and of v_cache
 * apart from each other.  q in place may stand among k's and v's rows (of the same
 * token stride) and be none of them. */
int r9vx_rope_kv_launch(const r9vx_rope_kv_static *st, const r9vx_rope_kv_args *args, r9vx_stream_t stream);

/* ----------------------------------------------------------- attention */

typedef struct r9vx_attn_static {
    uint32_t b_bucket;     /* the launch's b <= b_bucket < 2^16 */
    uint32_t t_bucket;     /* decode: new tokens of each sequence, 1 .. 8; prefill: the launch's t <= t_bucket */
    uint32_t len_bucket;   /* the longest length; the table has a column for each of its pages */
    uint32_t heads;        /* a multiple of kv_heads */
    uint32_t kv_heads;
    uint32_t head_dim;     /* 64, 96, 128, 192 or 256 */
    uint32_t page_size;    /* a power of two, at least 8 */
    uint32_t dtype;        /* of q, the cache and out: BF16 or F16 */
    uint32_t causal;       /* decode: 1 */
    uint32_t window;       /* 0: none */
    uint32_t scale_bits;   /* f32, finite */
    uint32_t softcap_bits; /* f32, finite and not negative; 0: none */
} r9vx_attn_static;

typedef struct r9vx_attn_args {
    const void *q;          /* decode [b, t_bucket, heads, head_dim], prefill [t, heads, head_dim] */
    const void *k_cache;
    const void *v_cache;
    const int32_t *table;   /* [b, at least ceil(len_bucket / page_size)] */
    const int32_t *lengths; /* [b] */
    const int32_t *offsets; /* prefill: [b + 1], sequence i's rows of q are offsets[i] .. offsets[i + 1] - 1; decode: NULL */
    const int32_t *starts;  /* first key seen, decode [b], prefill [t], or NULL */
    const int32_t *prefix;  /* prefill: [b] or NULL: keys before it are seen by every row (a causal static's) */
    const float *slopes;    /* [heads] or NULL */
    void *out;              /* as q; overlaps no operand.  Prefill: rows outside every sequence are not written */
    uint8_t *workspace;     /* r9vx_attn_*_workspace_bytes, 256-byte aligned; NULL when 0 */
    uint32_t *status;       /* or NULL */
    uint64_t q_stride[3];   /* of a sequence (decode), of a token, of a head */
    uint64_t out_stride[3]; /* rows apart from each other */
    uint64_t k_stride[3];   /* of a page, of a token (below 2^27), of a head; all strides multiples of 8 below 2^40 */
    uint64_t v_stride[3];
    uint64_t table_stride;  /* of a sequence */
    uint32_t pages;
    uint32_t b;
    uint32_t t;             /* prefill: rows of q; decode: 0 */
    uint32_t _tail_pad;
} r9vx_attn_args;

/* The t_bucket new tokens of each sequence.  A row's output bits depend on the
 * static, its sequence's length and its operands alone.  A length below t_bucket
 * leaves the first rows without a place: zeros. */
int r9vx_attn_decode_launch(const r9vx_attn_static *st, const r9vx_attn_args *args, r9vx_stream_t stream);
size_t r9vx_attn_decode_workspace_bytes(const r9vx_attn_static *st);

/* Prompts, or chunks of prompts whose beginnings the cache holds, packed in q
 * without gaps: 0 <= offsets[0] <= offsets[1] <= ... <= t.  Offsets that are
 * not set R9VX_STATUS_BAD_LENGTH, and the rows they touch are undefined. */
int r9vx_attn_prefill_launch(const r9vx_attn_static *st, const r9vx_attn_args *args, r9vx_stream_t stream);
size_t r9vx_attn_prefill_workspace_bytes(const r9vx_attn_static *st);

#ifdef __cplusplus
}
#endif
#endif
