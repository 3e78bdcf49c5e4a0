/*
 * fa_cache_hip.h — C ABI of libfa_hip.so for a key/value cache held in pages: room for new tokens, writing them,
 * sharing pages between sequences, keeping the accepted ones of drafted tokens, giving pages back.
 *
 * A page holds page_size tokens of one sequence in every layer. block_table[slot][b] names the page of a sequence's
 * tokens b * page_size ..; a page may belong to several sequences (refcount of them), then it is only read. A page
 * is free when its refcount is 0; the lowest-numbered free pages are given out first, in the order of the call's
 * slots, so that equal calls give equal tables.
 *
 * Everything lives on the device and every call is asynchronous on `stream`: no call reads a length on the host.
 * So a call that cannot be done on the device's values sets a bit of *status (FA_CACHE_*, bits are only ever
 * added) and leaves the sequence it concerns as it was (fa_cache_reserve: every sequence). Slot -1 marks an unused
 * entry and is passed over. Calls on one cache have to be ordered (one stream, or events between streams).
 */
#ifndef FA_CACHE_HIP_H_
#define FA_CACHE_HIP_H_

#include "fa_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct FaCache {
    void *k_pages, *v_pages;      /* (layers, num_pages, page_size, nheads, head_dim), 16-bit, contiguous */
    int32_t *block_table;         /* (max_seqs, max_blocks): page, or -1 */
    int32_t *seqlens;             /* (max_seqs): tokens held */
    int32_t *nblocks;             /* (max_seqs): table entries in use (evicted ones, -1, among them) */
    int32_t *refcount;            /* (num_pages): sequences that hold the page */
    int32_t *status;              /* (1) */
    int32_t *scratch;             /* fa_cache_scratch_words() words, any contents */
    int32_t layers, num_pages, page_size, nheads, head_dim, max_seqs, max_blocks;
    int32_t window, num_sinks;    /* what the attention over this cache sees (fa_window_hip.h); 0: no window */
} FaCache;

enum {
    FA_CACHE_NO_PAGES = 1,        /* reserve: not enough free pages; nothing was reserved */
    FA_CACHE_TOO_LONG = 2,        /* reserve: a sequence would pass max_blocks pages; nothing was reserved */
    FA_CACHE_BAD_SLOT = 4,        /* a slot out of range, or named twice */
    FA_CACHE_NOT_RESERVED = 8,    /* write, compact: no page of the sequence's own there */
    FA_CACHE_BAD_KEEP = 16,       /* compact: indices not ascending, or a count out of range */
    FA_CACHE_BAD_LENGTH = 32,     /* reserve: a negative count; truncate: longer than the sequence, or keys that the
                                     shorter one would see are evicted */
    FA_CACHE_NOT_EMPTY = 64,      /* fork: the child holds tokens or pages */
};

/* most slots of one call, most slots of a cache */
enum { FA_CACHE_MAX_SLOTS = 4096, FA_CACHE_MAX_SEQS = 65536 };

int64_t fa_cache_scratch_words(int32_t num_pages);
/* sizeof(FaCache) */
int64_t fa_cache_struct_size(void);

/* Room for counts[i] (NULL: `count`) more tokens behind the tokens of slots[i]. A partly full last page that other
 * sequences hold too is left to them (the call's last holder keeps it): its rows are copied into a page of the
 * sequence's own. */
int fa_cache_reserve(const FaCache *cache, const int32_t *slots, int32_t n, const int32_t *counts, int32_t count,
                     void *stream);
/* Stores the rows cu_seqlens[i] .. cu_seqlens[i+1]-1 of k, v (rows, nheads, head_dim; element strides, multiples of 8)
 * behind the tokens of slots[i], in one layer. Lengths stay as they are. */
int fa_cache_write(const FaCache *cache, int32_t layer, const int32_t *slots, int32_t n, const void *k,
                   int64_t k_row_stride, int64_t k_head_stride, const void *v, int64_t v_row_stride,
                   int64_t v_head_stride, const int32_t *cu_seqlens, int64_t total, int32_t max_seqlen, void *stream);
/* Keeps the tokens keep[i][0 .. counts[i]-1] (ascending, counted from the sequence's length) of those written behind
 * slots[i], moved together; the length grows by counts[i], pages behind the new end are given back. */
int fa_cache_compact(const FaCache *cache, const int32_t *slots, int32_t n, const int32_t *keep, int64_t keep_stride,
                     int32_t max_keep, const int32_t *counts, void *stream);
/* children[i] (empty) begins with the tokens of parents[i], in the same pages */
int fa_cache_fork(const FaCache *cache, const int32_t *parents, const int32_t *children, int32_t n, void *stream);
/* shortens slots[i] to lens[i] tokens (NULL: 0) and gives the pages behind back */
int fa_cache_truncate(const FaCache *cache, const int32_t *slots, int32_t n, const int32_t *lens, void *stream);
/* gives back the pages that no later token sees: past the sinks and wholly behind the window */
int fa_cache_evict(const FaCache *cache, const int32_t *slots, int32_t n, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* FA_CACHE_HIP_H_ */
