/*
 * fa_window_hip.h — C ABI of libfa_hip.so for attention with a sliding window and sinks, over dense var-len
 * sequences (forward and backward) and over a cache held in pages (forward).
 *
 * One rule says what a query sees. Its position p is aligned to the end of its sequence's keys: query row i of
 * sq rows over sk keys stands at p = i + sk - sq. It sees key j when
 *     j <= p   and   (j > p - window   or   j < num_sinks).
 * window = 0 means no window (every key up to p). A query with p < 0 sees nothing: its output row is 0, its lse
 * -inf, its gradient 0. Query heads share key/value heads in groups: head h reads key/value head
 * h / (nheads / nheads_k).
 *
 * Conventions are those of fa_hip.h: plain C types, the caller allocates everything, every call is ordered on
 * `stream` and asynchronous, records no host work (so it can be captured into a HIP graph), returns 0 or an error
 * code, the message in fa_last_error().
 */
#ifndef FA_WINDOW_HIP_H_
#define FA_WINDOW_HIP_H_

#include "fa_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Dense sequences. Layouts and cu_seqlens as in FaFwdArgs; strides in elements, multiples of 8, rows 16-byte
 * aligned and not overlapping. Sequence bounds past total_q / total_k are cut off there. */
typedef struct FaWindowArgs {
    const void *q;                /* (total_q, nheads, head_dim) */
    const void *k, *v;            /* (total_k, nheads_k, head_dim) */
    void *o;                      /* forward: output; backward: the forward's output */
    float *softmax_lse;           /* (batch, nheads, lse_stride) natural log; backward: the forward's */
    const int32_t *cu_seqlens_q;  /* (batch + 1) device */
    const int32_t *cu_seqlens_k;  /* (batch + 1) device */
    /* backward only */
    const void *dout;             /* (total_q, nheads, head_dim) */
    void *dq, *dk, *dv;           /* outputs, shapes of q, k, v */
    void *workspace;              /* fa_window_bwd_workspace() bytes, 16-byte aligned, any contents */
    int64_t workspace_bytes;
    int64_t q_row_stride, q_head_stride;
    int64_t k_row_stride, k_head_stride;
    int64_t v_row_stride, v_head_stride;
    int64_t o_row_stride, o_head_stride;
    int64_t do_row_stride, do_head_stride;
    int64_t dq_row_stride, dq_head_stride;
    int64_t dk_row_stride, dk_head_stride;
    int64_t dv_row_stride, dv_head_stride;
    int64_t total_q, total_k;
    int32_t batch, nheads, nheads_k, head_dim;   /* head_dim: multiple of 8, <= 128 */
    int32_t max_seqlen_q, max_seqlen_k, lse_stride;   /* rows of a sequence past max_seqlen_q (dk, dv: keys past
                                     max_seqlen_k) are not computed and not written */
    int32_t window;               /* keys a query sees counting its own position; 0: all */
    int32_t num_sinks;            /* first keys that every later query sees */
    float softmax_scale;
    int32_t dtype;                /* FA_DTYPE_FP16 / FA_DTYPE_BF16 */
    int32_t reserved;             /* 0 */
} FaWindowArgs;

int fa_window_fwd(const FaWindowArgs *args, void *stream);
int fa_window_bwd(const FaWindowArgs *args, void *stream);
/* bytes fa_window_bwd needs for these sizes (only sizes are read); < 0: error code, negated */
int64_t fa_window_bwd_workspace(const FaWindowArgs *args);

/* A cache in pages. Key j of a sequence lies in row j % page_size of page block_table[seq][j / page_size].
 * The new tokens' keys are in the cache already, behind the context: keys 0 .. context_len + sq - 1. A table
 * entry outside [0, num_pages) is never read: its keys are seen by nobody.
 *
 * tree_mask (NULL: a chain, row i sees rows 0..i) gives for each new token the new tokens it sees, itself among
 * them, as bits (bit j & 63 of word j >> 6 for row j of its sequence). A token's position is then
 * context_len + (number of its bits) - 1, and a new key stands at its own token's position; the window goes by
 * these positions. Rows of a sequence: at most 64 * tree_words, at most 256. */
typedef struct FaPagedArgs {
    const void *q;                /* (total_q, nheads, head_dim) */
    void *o;                      /* (total_q, nheads, head_dim) */
    float *softmax_lse;           /* (batch, nheads, lse_stride) or NULL */
    const void *k_pages, *v_pages;    /* (num_pages, page_size, nheads_k, head_dim) */
    const int32_t *block_table;   /* (num_seqs, max_blocks) */
    const int32_t *context_lens;  /* (num_seqs) keys before the first new token */
    const int32_t *seq_ids;       /* (batch) rows of block_table / context_lens; NULL: 0 .. batch-1. An id outside
                                     [0, num_seqs) marks an unused entry: its output rows are 0 */
    const int32_t *cu_seqlens_q;  /* (batch + 1) */
    const uint64_t *tree_mask;    /* (total_q, tree_words) or NULL */
    void *workspace;              /* fa_paged_workspace() bytes, 16-byte aligned, any contents */
    int64_t workspace_bytes;
    int64_t q_row_stride, q_head_stride;
    int64_t o_row_stride, o_head_stride;
    int64_t k_page_stride, k_row_stride, k_head_stride;
    int64_t v_page_stride, v_row_stride, v_head_stride;
    int64_t table_stride;
    int64_t total_q;
    int32_t batch, nheads, nheads_k, head_dim;
    int32_t num_pages, page_size; /* page_size: a power of two, 16 or more */
    int32_t num_seqs, max_blocks;
    int32_t max_seqlen_q, max_context_len;   /* max_seqlen_q as above. max_context_len only decides how the keys are
                                     split: results differ in the order of their sums, in the last bits */
    int32_t tree_words, lse_stride;
    int32_t window, num_sinks;
    float softmax_scale;
    int32_t dtype;
} FaPagedArgs;

int fa_paged_fwd(const FaPagedArgs *args, void *stream);
int64_t fa_paged_workspace(const FaPagedArgs *args);

/* sizeof(FaWindowArgs) (what = 0) or sizeof(FaPagedArgs) (what = 1), for bindings that check their layout */
int64_t fa_window_args_size(int what);

#ifdef __cplusplus
}
#endif

#endif /* FA_WINDOW_HIP_H_ */
