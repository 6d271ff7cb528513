/*
 * ar_pages.h -- C-ABI of the paged KV cache: pools of cache pages shared by many sequences, the rows of new
 * tokens on their way into them, and causal attention of those tokens over them.
 *
 * No counterpart in the reference, whose caches are one contiguous (seq, heads, size) block per model
 * (engine/ml/.../AttentionFeatures.java:823-826): it serves one sequence at a time.  The row preparation and the
 * attention compute what AttentionFeatures.attentionImpl (engine/ml/.../AttentionFeatures.java:785-929) computes
 * between the projections and the o_proj dense, as ar_hip_attention_decode does for one row of one sequence.
 *
 * Same conventions as ar_hip.h: plain C, device pointers, AR_HIP_* status codes, ar_hip_last_error().  Every call
 * enqueues on the context's stream and returns; nothing is allocated.  Calls that need scratch memory take `work`,
 * device memory of the caller's, 16-byte aligned, of at least the bytes that the matching *_work call reports; its
 * contents mean nothing between calls.  Calls ordered on one stream may share it, calls that may run at the same
 * time may not.
 */
#ifndef AR_PAGES_H
#define AR_PAGES_H

#include "ar_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* A pool of pages and the sequences that lie on them.  Row r of a sequence s lies on page
 * table[s * max_pages + r / page_rows], in that page's row r % page_rows, in every layer.  A table entry outside
 * 0..pages-1 (-1, by the calls below) is no page: rows there are not in the cache; they are dropped when written and
 * hidden from every query.
 * A pool that the caller manages without the calls below may leave rows and refs null. */
typedef struct ar_pages {
    void *k;            /* [layers][pages][kv_heads][page_rows][head_dim] of dtype, 16-byte aligned */
    void *v;            /* the same */
    int32_t *table;     /* [seqs][max_pages] */
    int32_t *rows;      /* [seqs]: rows each sequence holds */
    int32_t *refs;      /* [pages]: sequences that hold the page; 0: it is free */
    int32_t dtype;      /* AR_DTYPE_F32, AR_DTYPE_BF16 or AR_DTYPE_F16 */
    int32_t layers;
    int32_t pages;
    int32_t kv_heads;
    int32_t page_rows;  /* a power of two, 16 .. 256 */
    int32_t head_dim;   /* 64 or 128 */
    int32_t seqs;       /* table rows; 0 with a null table for a pool alone (ar_hip_pages_copy) */
    int32_t max_pages;  /* table columns; max_pages * page_rows <= 2^30 */
} ar_pages;

/* The new rows of a call, by sequence: chunk i is the rows start[i] .. start[i+1]-1 of the call's row arrays, and
 * they are the rows at[i], at[i]+1, ... of sequence seq[i].  Rows from start[n] on belong to no chunk: they are
 * neither read nor written.  A chunk of an unknown sequence or with a negative at is not in the cache: its rows are
 * dropped when written and see nothing.  A row past the table's last column is dropped, too.  A chunk that passes the
 * call's rows is empty; where starts descend it is not defined which chunks are (no access leaves the arrays, and rows
 * are left as they were or computed). */
typedef struct ar_chunks {
    const int32_t *seq;   /* device [n], or null: sequences 0 .. n-1 */
    const int32_t *start; /* device [n+1], not decreasing, from 0; or null: one row each */
    int32_t *at;          /* device [n]: read by ar_hip_pages_write and ar_hip_attention_paged, filled in by
                             ar_hip_pages_grow */
    int32_t n;            /* chunks, 1 .. 2^20 */
    int32_t rows;         /* rows of the call's row arrays, 0 .. 2^22, at least start[n] */
} ar_chunks;

/* Rotary positions with one to four axes (text; or time, height and width of images and video).  Frequency f of
 * head_dim / 2 turns dims (f, f + head_dim / 2) by positions[axis(f)][row] * theta^(-2 f / head_dim), the split-half
 * form of ar_hip_rope.  section[a] frequencies go by axis a, and the sections add up to head_dim / 2:
 *   AR_ROPE_SECTIONS:    the first section[0] by axis 0, the next section[1] by axis 1, ...
 *   AR_ROPE_INTERLEAVED: f by axis a = f % axes while f / axes < section[a], the others by axis 0;
 *                        for a > 0, section[a] is at most the number of f with f % axes == a
 * Angles are computed in double. */
#define AR_ROPE_SECTIONS 0
#define AR_ROPE_INTERLEAVED 1
typedef struct ar_rotary {
    double theta;
    const int32_t *positions; /* device [axes][chunks->rows], or null: a row's position in every axis is its cache row
                                 (0 where it has none) */
    int32_t axes;             /* 1 .. 4 */
    int32_t layout;           /* AR_ROPE_*; with one axis both are the same */
    int32_t section[4];
} ar_rotary;

/* Scratch bytes of ar_hip_pages_grow and _fork (of n entries) and of _compact (n = 0) on these pages. */
int ar_hip_pages_work(const ar_pages *pages, int n, size_t *bytes);

/* Makes room for every chunk's rows at its sequence's end: at[i] = rows[seq[i]], which then grows by the chunk's
 * rows.  Chunks are served in order, and new pages are the lowest-numbered free ones, one after another.  A last page
 * that is not full and that other sequences hold too is replaced by a copy of it; of several chunks on one such
 * page the last keeps it if no one else holds it.  A chunk that cannot be served, because the pool has no pages left
 * for it (then none that needs pages after it is served, either), its table row has no columns left, its sequence is
 * unknown or was named by an earlier chunk, leaves its sequence as it was and gets at[i] = -1.  *missing (device, or
 * null) receives the number of pages that were wanted beyond the free ones.  chunks->n at most 4096; needs rows and
 * refs. */
int ar_hip_pages_grow(ar_hip_ctx *ctx, const ar_pages *pages, const ar_chunks *chunks, int32_t *missing, void *work,
                      size_t work_bytes);

/* Sequence seq[i] (seq null: i) keeps its first keep[i] rows (keep null: none) and gives back the pages behind them.
 * A keep of more rows than there are changes nothing.  Unknown sequences, and all but the first mention of one, are
 * passed over.  n at most 4096; needs rows and refs. */
int ar_hip_pages_trim(ar_hip_ctx *ctx, const ar_pages *pages, const int32_t *seq, const int32_t *keep, int n);

/* Sequence dst[i] becomes what sequence src[i] was before the call, on the same pages; what it held is given back.
 * Sources may be targets as well (a search that reorders its sequences).  Entries with an unknown sequence, and all
 * but the first with one target, are passed over.  n at most 4096; needs rows and refs. */
int ar_hip_pages_fork(ar_hip_ctx *ctx, const ar_pages *pages, const int32_t *src, const int32_t *dst, int n,
                      void *work, size_t work_bytes);

/* Moves the pages in use to the front of the pool: the used pages past the number of used ones, in ascending order,
 * go to the free pages before it, in ascending order; table and refs follow.  *live (device, or null) receives the
 * number of pages in use: the pool is free from there on.  Needs refs. */
int ar_hip_pages_compact(ar_hip_ctx *ctx, const ar_pages *pages, int32_t *live, void *work, size_t work_bytes);

/* Copies page src[i] of `from` to page dst[i] of `to`, in every layer.  The pools may be one; they agree in dtype,
 * layers, kv_heads, page_rows and head_dim.  Entries with a page outside its pool, all but the first with one target
 * and, within one pool, entries whose target is an entry's source are passed over.  Tables and counts stay as they
 * are.  n at most 4096. */
int ar_hip_pages_copy(ar_hip_ctx *ctx, const ar_pages *from, const ar_pages *to, const int32_t *src,
                      const int32_t *dst, int n);

/* The rows of every chunk on their way to attention in one layer: QK-norm of the raw q and k projections (fp32;
 * gains of heads * head_dim and kv_heads * head_dim values, or null for none), rotary positions, k and v rounded to
 * the pool's dtype (to nearest; beyond fp16's range to infinity) and stored into their pages.  q_out (act_dtype:
 * AR_DTYPE_F32 or AR_DTYPE_BF16, [rows][heads * head_dim]) receives the queries; it may be q itself where both are
 * fp32 and q_stride is heads * head_dim.  q and q_out may both be null (keys and values only).  q_stride and
 * kv_stride are floats from one row to the next, multiples of 4, and the pointers are 16-byte aligned: the q | k | v
 * rows of one stacked projection are q, q + heads * head_dim and q + (heads + kv_heads) * head_dim.  Of several
 * chunks of one sequence only the first is written. */
int ar_hip_pages_write(ar_hip_ctx *ctx, const ar_pages *pages, int layer, const ar_chunks *chunks, const float *q,
                       const float *k, const float *v, int q_stride, int kv_stride, int heads, const float *q_norm,
                       const float *k_norm, float qk_eps, int qk_norm_mode, const ar_rotary *rotary, void *q_out,
                       int act_dtype);

/* Causal attention of every chunk's rows over their sequences' pages in one layer: the row at cache row p sees rows
 * 0 .. p (the chunk's own among them, written before), scores scaled by 1 / sqrt(head_dim), head h reads KV head
 * h / (heads / kv_heads).  q and out: [rows][heads * head_dim] of act_dtype (AR_DTYPE_F32 or AR_DTYPE_BF16), 16-byte
 * aligned; out may be q itself.  Rows that see nothing become 0.  What a hidden row holds (infinities, NaN) does not
 * reach the result; infinities and NaN that a row sees make it infinite or NaN.
 * Sums are in fp32, of weights up to 2^14: keys and values beyond 2^90 may overflow them.  With fp32 activations the products
 * keep 22 bits or more: relative to each factor over 16-bit caches (over fp16 ones a query value below 2^-17 of its row's
 * largest loses up to 2^-39 of that largest), to the largest value of its row of the cache over fp32 ones (if that is at
 * least 2^-122), and what a weight of less than 2^-30 of its row's largest loses is below 2^-30 of the value that it
 * weighs.  With bf16 activations the softmax weights are rounded to 16 bits (the cache's type; fp16 for fp32 caches)
 * for the second product.
 * chunks->rows * heads / 16 + chunks->n * kv_heads must be below 2^23. */
int ar_hip_attention_paged_work(ar_hip_ctx *ctx, const ar_pages *pages, const ar_chunks *chunks, int heads,
                                size_t *bytes);
int ar_hip_attention_paged(ar_hip_ctx *ctx, const ar_pages *pages, int layer, const ar_chunks *chunks, const void *q,
                           int act_dtype, int heads, void *out, void *work, size_t work_bytes);

#ifdef __cplusplus
}
#endif

#endif /* AR_PAGES_H */
