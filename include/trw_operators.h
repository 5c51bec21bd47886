/*
 * trw_operators.h -- C ABI of the operators that consume walks: attention
 * inside each walk (forward, backward, one new event over a cache) and the
 * learned bias by distance buckets.
 *
 * The sampler leaves walks padded in device memory; a sequence model over
 * them trains and answers through these calls.  They live in a library of
 * their own (libtrw_operators.so), because they work on the caller's tensors
 * and streams: the library binds to the HIP runtime that the caller's tensors
 * come from, and keeps no handle.
 *
 * Conventions
 *  - Every pointer is device memory of the current device.  Nothing is
 *    allocated and nothing is waited for: work is queued on `stream` (a
 *    hipStream_t, NULL = the default stream) and the caller's buffers are in
 *    use until it has run.  Scratch memory is the caller's; each operator has
 *    a call that says how much it needs.
 *  - Shapes, strides and alignments are checked on the host: a call that does
 *    not fit returns TRW_ERR_INVALID_ARGUMENT with a message
 *    (trw_ops_last_error, thread-local) and queues nothing.  Values that only
 *    the device knows (offsets, lengths, bucket ids) are clamped there, so
 *    that wrong ones give wrong results and never an access out of range.
 *  - Strides are in elements.  A row of D values is contiguous and 16-byte
 *    aligned, D is a multiple of 8 up to 128; rows lie at most 2^22 elements
 *    apart.
 */
#ifndef TRW_OPERATORS_H
#define TRW_OPERATORS_H

#include "trw_engine.h"

#ifdef __cplusplus
extern "C" {
#endif

#define TRW_OPS_ABI_VERSION 1

/* Longest reach of a distance bias (distances past it share the outermost
 * buckets) and most buckets of one. */
#define TRW_OPS_MAX_REACH 1024
#define TRW_OPS_MAX_BUCKETS 256
/* 16-bit types: softcaps above this have kernels of their own (walks of any
 * length go through those of tiles). */
#define TRW_OPS_WIDE_CAP 256

typedef enum trw_dtype { TRW_F32 = 0, TRW_F16 = 1, TRW_BF16 = 2 } trw_dtype;

typedef enum trw_mask_kind {
    TRW_MASK_FULL = 0,   /* every key of the walk */
    TRW_MASK_CAUSAL = 1, /* keys up to the query's own position */
    TRW_MASK_PREFIX = 2  /* those, and the walk's first `prefix` keys */
} trw_mask_kind;

/* [rows, heads, D] of one tensor. */
typedef struct trw_rows {
    void* data;
    int64_t row_stride;
    int64_t head_stride;
} trw_rows;

/* Which keys each query row sees, as an interval of key rows: documents
 * (walks) of query rows, each over a document of key rows of its own, of
 * which the queries are the last positions (a document of a queries over b
 * keys starts at position b - a; queries before position 0 see nothing).
 *
 * Padded (q_offsets NULL): document w has the rows [w * q_length,
 * w * q_length + min(q_lens[w], q_length)), keys alike.  Packed: the rows
 * [q_offsets[w], q_offsets[w + 1]).  Rows of no document see nothing.
 * k_lens / k_offsets NULL: the queries' own. */
typedef struct trw_walk_mask_params {
    int64_t docs;
    int64_t q_rows, k_rows;             /* below 2^30 */
    int64_t q_length, k_length;         /* padded */
    const int64_t *q_lens, *k_lens;     /* padded: [docs] */
    const int64_t *q_offsets, *k_offsets; /* packed: [docs + 1], ascending */
    const int64_t* prefix;              /* TRW_MASK_PREFIX: [docs] */
    int32_t kind;
    int32_t* q_rows_info; /* out: [q_rows, 4] first key, end key, key at the row's own position,
                             rows of its document (of queries or keys, whichever has more) */
    int32_t* k_rows_info; /* out: [k_rows, 4] first query, end query, 0, rows of its document */
    int32_t* docs_info;   /* out: [docs, 8] first query, queries, their rows with padding, first
                             key, keys, their rows with padding, prefix, kind */
} trw_walk_mask_params;
trw_status trw_ops_walk_mask(const trw_walk_mask_params* params, void* stream);

/* score(i, j) = cap(scale q_i . k_j) + table[h, buckets[reach + d]]
 *                 - slopes[h] |t_i - t_j|
 * with cap(x) = softcap tanh(x / softcap) (softcap 0: x), d the distance in
 * positions clamped to [-reach, reach], and t the times, or positions where
 * they are NULL. */
typedef struct trw_score {
    float scale;
    float softcap;
    const float* table;     /* [heads, num_buckets] or NULL */
    const int32_t* buckets; /* [2 reach + 1] bucket ids */
    int32_t num_buckets;
    int32_t reach;
    const float* slopes;    /* [heads] or NULL */
    const float* q_times;   /* [q_rows] or NULL */
    const float* k_times;   /* [k_rows], with q_times */
} trw_score;

typedef struct trw_attention_params {
    int32_t dtype; /* of q, k, v, out and their gradients */
    int32_t heads, kv_heads, dim; /* heads: a multiple of kv_heads, which it shares in order */
    int64_t q_rows, k_rows;
    const int32_t *q_rows_info, *k_rows_info, *docs_info; /* of trw_ops_walk_mask */
    int64_t docs;
    int64_t longest; /* no document has more queries or keys than this; 0: not known */
    int32_t own_causal; /* 1: the mask is causal, over the queries' own rows as keys */
    int32_t covered; /* 1: every row is a document's, its padding included (a padded mask); 0: rows
                        of no document are looked for, and left zero */
    trw_score score;
    trw_rows q, k, v, out;
    float* stats; /* [2, heads, q_rows], of the rows' softmax (base 2); written by the forward
                     pass where not NULL, read by the backward pass */
    trw_rows out_low; /* what rounding took from out, in the same type, for a backward pass that
                         takes sums of the output's products more exactly; data NULL: not kept */
    /* backward */
    trw_rows d_out, d_q, d_k, d_v;
    float* d_table; /* [heads, num_buckets], where score.table is given */
    void* workspace;
    uint64_t workspace_bytes;
} trw_attention_params;

/* Bytes of workspace of a pass (backward 0 or 1). */
trw_status trw_ops_attention_workspace(const trw_attention_params* params, int32_t backward,
                                       uint64_t* bytes);
/* out_i = sum_j softmax_j(score(i, j)) v_j over the keys that row i sees; 0
 * where it sees none. */
trw_status trw_ops_attention_forward(const trw_attention_params* params, void* stream);
/* Gradients of q, k, v and the table, from d_out and what the forward pass
 * left in out and stats.  Results do not depend on the order in which
 * workgroups run. */
trw_status trw_ops_attention_backward(const trw_attention_params* params, void* stream);

/* One new event of each of `batch` walks: its key and value go into the walk's
 * cache at position lens[b], and it attends to positions 0 .. lens[b].  A
 * negative length is an idle row: it writes nothing to the cache and its
 * output is 0 (as it is where the table masks every position); a length of
 * `capacity` or more (no room) gives NaN, and writes nothing to the cache
 * either. */
typedef struct trw_attention_step_params {
    int32_t dtype;
    int32_t heads, kv_heads, dim;
    int64_t batch, capacity;
    const int64_t* lens;     /* [batch] events already in the cache */
    trw_score score;         /* q_times [batch]; k_times [batch, capacity], row-major, written too */
    trw_rows q, k, v, out;   /* [batch, heads or kv_heads, D] */
    void *k_cache, *v_cache; /* element (b, position, head, 0) at the strides below */
    int64_t k_batch_stride, k_pos_stride, k_head_stride;
    int64_t v_batch_stride, v_pos_stride, v_head_stride;
    void* workspace;
    uint64_t workspace_bytes;
} trw_attention_step_params;
trw_status trw_ops_attention_step_workspace(const trw_attention_step_params* params,
                                            uint64_t* bytes);
trw_status trw_ops_attention_step(const trw_attention_step_params* params, void* stream);

/* out[h, i, j] = table[h, buckets[reach + clamp(i + q_offset - j)]], dense
 * [heads, q_len, k_len] of the table's type, and the table's gradient from a
 * dense d_out (rows contiguous; strides of heads and rows in elements). */
typedef struct trw_relative_bias_params {
    int32_t dtype; /* of table, out, d_out and d_table */
    int32_t heads, num_buckets, reach;
    int64_t q_len, k_len, q_offset;
    const void* table;
    const int32_t* buckets;
    void* out;
    const void* d_out;
    int64_t d_out_head_stride, d_out_row_stride;
    void* d_table;
    void* workspace; /* backward */
    uint64_t workspace_bytes;
} trw_relative_bias_params;
trw_status trw_ops_relative_bias(const trw_relative_bias_params* params, void* stream);
trw_status trw_ops_relative_bias_workspace(const trw_relative_bias_params* params,
                                           uint64_t* bytes);
trw_status trw_ops_relative_bias_backward(const trw_relative_bias_params* params, void* stream);

/* Message of the last failed call on this thread. */
const char* trw_ops_last_error(void);
int32_t trw_ops_abi_version(void);

#ifdef __cplusplus
}
#endif
#endif /* TRW_OPERATORS_H */
