/*
 * ptc_serve.h -- device operators of a serving step over a paged KV cache:
 * page tables and slot maps of a batch, the rotary write of new keys and
 * values, attention of the new tokens over the cache, and token sampling.
 * They stand beside ptc_matvec and ptc_sgemm (ptc.h): DEVICE pointers,
 * asynchronous on `stream` (NULL = legacy default stream), no allocation,
 * capturable into CUDA graphs. A call runs on the device that holds its
 * output, whichever is current; the stream has to be that device's. No reference counterpart: the
 * reference answers one request with one contiguous cache.
 *
 * A step of a batch calls, in this order on one stream,
 *   ptc_plan_pages       who owns which page, where each new token goes
 *   ptc_kv_append        per layer, after the q/k/v products
 *   ptc_paged_attention  per layer
 *   ptc_sample_tokens    after the classifier
 *
 * Errors. A call with bad arguments (as far as the host can see them) or
 * one that the CUDA runtime rejects prints a message to stderr, does nothing
 * and returns -1; otherwise 0. What only the device can see -- lengths,
 * positions, page numbers -- is checked by the kernels: they OR a
 * PTC_SERVE_ERR_* bit into the device int *err (err may be NULL; the caller
 * clears it) and skip the access. Host threads may call at the same time, on
 * streams of their own; a refused call does not show in a later one.
 */
#ifndef PTC_SERVE_H
#define PTC_SERVE_H

#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Element types. Sums, softmax statistics and rotations are computed in 32
 * bits or more and rounded once to the type. What is rounded before that: the
 * probabilities of 16-bit attention (see there). */
enum { PTC_F32 = 0, PTC_F16 = 1, PTC_BF16 = 2 };

enum {
    PTC_SERVE_ERR_PAGES = 1,    /* fewer free pages than the step needs */
    PTC_SERVE_ERR_TABLE = 2,    /* a sequence needs more than max_pages pages */
    PTC_SERVE_ERR_TOKENS = 4,   /* more new tokens than max_tokens */
    PTC_SERVE_ERR_LENGTH = 8,   /* a negative or inconsistent length */
    PTC_SERVE_ERR_INDEX = 16,   /* a page, slot or position out of range */
    PTC_SERVE_ERR_WAIT = 32     /* a kernel's bounded wait ran out: its results are not valid */
};

#define PTC_SERVE_MAX_SEQS 4096   /* sequences of one call */

/* ---- page tables and slot maps -------------------------------------------- */

/* One step of n_seqs sequences, of which sequence r holds past_len[r] tokens
 * in the first ceil(past_len[r] / page_size) pages of its page_table row and
 * gets new_len[r] more (zero is fine for either). The pages it lacks are taken
 * from free_pages in order, sequence by sequence; a page that stands there
 * twice, or in the table too, is handed out all the same. Writes
 *   page_table[r][...]  the pages taken (entries that hold cached tokens and
 *                       entries behind the new ones are left as they are)
 *   kv_len[r]           past_len[r] + new_len[r]
 *   q_start[r]          first row of sequence r among the step's rows;
 *                       q_start[n_seqs] = their number
 *   positions[t]        position of row t in its sequence
 *   slots[t]            page * page_size + offset of that position
 *   pages_used          the number of free_pages taken
 * Rows from q_start[n_seqs] up to max_tokens get -1 in both maps, and so
 * does the slot of a row whose page number is outside [0, n_pages)
 * (PTC_SERVE_ERR_INDEX). A step that does not fit (PAGES, TABLE, TOKENS,
 * LENGTH) is refused as a whole: the table stays as it is, every row gets
 * -1, q_start is zero everywhere, kv_len = past_len and *pages_used = 0, so
 * that the operators below do nothing. No output may overlap another array. */
typedef struct {
    int n_seqs;             /* 0 .. PTC_SERVE_MAX_SEQS */
    int page_size;          /* tokens per page, >= 1 */
    int max_pages;          /* columns of page_table, >= 1 */
    int max_tokens;         /* entries of slots and positions, at most 2^30 */
    int n_free;             /* entries of free_pages */
    int n_pages;            /* pages of the cache; n_pages * page_size < 2^31 */
    const int *past_len;    /* [n_seqs] */
    const int *new_len;     /* [n_seqs] */
    const int *free_pages;  /* [n_free] */
    int *page_table;        /* [n_seqs][max_pages], updated */
    int *kv_len;            /* [n_seqs] */
    int *q_start;           /* [n_seqs + 1] */
    int *slots;             /* [max_tokens] */
    int *positions;         /* [max_tokens] */
    int *pages_used;        /* [1] */
    int *err;
} ptc_pages_args;

int ptc_plan_pages(const ptc_pages_args *a, void *stream);

/* ---- the paged cache -------------------------------------------------------- */

/* Keys and values of one layer. Element (page, head, offset, i) is at
 * page * page_stride + head * head_stride + offset * token_stride + i, in
 * elements, in both k and v. head_dim is a multiple of 8, at most 128; the
 * pointers and strides are multiples of 16 bytes. A contiguous cache
 * [n_kv][seq][head_dim] is one page of seq tokens. */
typedef struct {
    void *k, *v;
    int dtype;
    int n_pages;
    int page_size;
    int n_kv_heads;
    int head_dim;
    long long page_stride, head_stride, token_stride;
} ptc_paged_cache;

/* ---- rotary write of new keys and values ------------------------------------- */

/* For each of n_tokens rows: q_out = RoPE(q), the cache's slot gets RoPE(k)
 * and v. Pairs are adjacent elements (2i, 2i + 1), as in the decode kernels;
 * rope is a table [n_pos][head_dim / 2] of (cos, sin) indexed by positions[t]
 * (ptc_rope_table gives the decoder's), or NULL for no rotation. q rows hold
 * n_heads * head_dim elements, k and v rows n_kv_heads * head_dim, at their
 * strides (elements, multiples of 16 bytes), so they may be parts of one
 * packed row. q_out may be q with the same stride; otherwise nothing
 * overlaps. A row with position -1 is skipped, a row with slot -1 gets its
 * q_out but is not stored; other positions outside [0, n_pos) (with a
 * table) or slots outside [0, n_pages * page_size) are skipped alike and
 * reported (INDEX). Two rows of one call may not have the same slot. */
typedef struct {
    ptc_paged_cache cache;
    int n_tokens;
    int n_heads;
    const void *q, *k, *v;
    long long q_stride, k_stride, v_stride;
    const int *positions;   /* [n_tokens] */
    const int *slots;       /* [n_tokens] */
    const float *rope;
    int n_pos;
    void *q_out;
    long long q_out_stride;
    int *err;
} ptc_append_args;

int ptc_kv_append(const ptc_append_args *a, void *stream);

/* The decoder's rotation table: [n_pos][head_dim / 2] pairs (cos, sin). */
int ptc_rope_table(float *table, int n_pos, int head_dim, void *stream);

/* ---- attention of new tokens over the paged cache ----------------------------- */

/* A workspace of this size serves every ptc_paged_attention call. The caller
 * zeroes it once; each call leaves the flags at its front (4096 bytes) zero
 * again. Calls that may run
 * at the same time need workspaces of their own, and so do two graphs that
 * may be replayed at the same time. */
#define PTC_ATTN_WORKSPACE_BYTES ((size_t)64 << 20)

/* Row q_start[r] + j (j < q_start[r + 1] - q_start[r]) of q is the token of
 * sequence r at position p = kv_len[r] - (q_start[r + 1] - q_start[r]) + j;
 * its head h attends, through K/V head h / (n_heads / n_kv_heads), to the
 * cached positions t <= p, with window > 0 to those with t > p - window too:
 *   out = sum_t softmax_t(scale * q . k_t) v_t.
 * A row that sees no position (p < 0) becomes zeros. One token per sequence,
 * chunks and mixtures of both are all one call; sequences may have no rows.
 * max_q is the largest number of rows of a sequence as far as the caller
 * knows it: it selects the kernel, whatever the rows are. The kernels agree
 * up to their roundings: the one for few rows (16-bit types: up to 32 of a
 * K/V head, heads of its group times max_q, or a scale of 0 or less) takes
 * probabilities in two parts of the type, that for many rounds them to the type
 * for the product with v, not for their sum. f16 probabilities are held in
 * steps of 2^-31 of the largest weight or finer. Rows of q and out beyond
 * q_start[n_seqs] are neither read nor written. q_start has to rise from 0 to
 * at most n_tokens (LENGTH, the sequence is left out), kv_len may not pass
 * max_pages * page_size or 2^30 (LENGTH, positions behind it are left out), and
 * positions of pages outside [0, n_pages) are left out too (INDEX).
 * q and out have the cache's type; strides in elements, multiples of 16
 * bytes; n_tokens * n_heads at most 2^30. What lies behind a sequence's last
 * position may be anything, NaN included; its own cached values should be
 * finite, as one that is not can reach rows of that sequence which do not see
 * its position. The same inputs give the same bits in every call. */
typedef struct {
    ptc_paged_cache cache;
    int n_seqs;             /* 0 .. PTC_SERVE_MAX_SEQS */
    int n_tokens;           /* rows of q and out */
    int n_heads;            /* a multiple of n_kv_heads */
    int max_q;
    int max_pages;          /* columns of page_table */
    int window;             /* 0: none */
    float scale;
    const void *q;          /* [n_tokens][n_heads][head_dim] */
    long long q_stride;
    void *out;              /* [n_tokens][n_heads][head_dim] */
    long long out_stride;
    const int *page_table;  /* [n_seqs][max_pages] */
    const int *kv_len;      /* [n_seqs] */
    const int *q_start;     /* [n_seqs + 1] */
    void *workspace;        /* 256-byte aligned */
    size_t workspace_bytes; /* at least PTC_ATTN_WORKSPACE_BYTES */
    int *err;
} ptc_attn_args;

int ptc_paged_attention(const ptc_attn_args *a, void *stream);

/* ---- sampling ------------------------------------------------------------------ */

#define PTC_SAMPLE_MAX_VOCAB 262144

/* One token for each of `rows` rows of logits, from the caller's uniform
 * random number u[r] in [0, 1). With w_i = exp((x_i - max) / temperature):
 *   top_k   keep the k largest logits (among equals the lowest indexes);
 *           k <= 0 or k >= vocab: all
 *   top_p   of these, in descending order, keep a token while the mass
 *           before it is below top_p times their total (always the first);
 *           top_p >= 1: all
 *   min_p   of these keep w_i >= min_p (the largest weight is 1)
 *   token = the lowest index whose running sum of kept weights, in index
 *           order, exceeds u times their total.
 * temperature 0 (or less) gives the first maximum. NaN logits count as -inf,
 * which is never chosen; a row without any other logit gives -1. +inf logits
 * share the whole mass. The arrays are per row; temperature NULL means 1,
 * top_k, top_p or min_p NULL none of that rule. Weights are summed as 64-bit
 * integers (units of 2^-43 of the largest; what is below half of one is never
 * chosen), so the token does not depend on the order of any sum: the same
 * inputs give the same tokens. */
typedef struct {
    int dtype;              /* of the logits */
    int rows;
    int vocab;              /* 1 .. PTC_SAMPLE_MAX_VOCAB */
    const void *logits;
    long long stride;       /* elements between rows, >= vocab; no alignment needed */
    const float *temperature;
    const int *top_k;
    const float *top_p;
    const float *min_p;
    const float *u;
    int *tokens;            /* [rows] */
} ptc_sample_args;

int ptc_sample_tokens(const ptc_sample_args *a, void *stream);

#ifdef __cplusplus
}
#endif
#endif
