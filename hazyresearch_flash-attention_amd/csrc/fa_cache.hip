// fa_cache.hip — the paged key/value cache's upkeep (include/fa_cache_hip.h): kernels and their C ABI.
//
// Tables are small (a few thousand words), so their kernels are bound by launch and by the latency of a few
// dependent loads; rows are moved by copies of 16 bytes a lane, bound by HBM. Everything is a function of the
// tables alone: pages are chosen by rank among the free ones (prefix sums), never by which atomic came first.
#include <hip/hip_runtime.h>

#include "fa_window_launch.h"
#include "../../include/fa_cache_hip.h"

namespace fa {
namespace {

typedef uint32_t u32x4v __attribute__((ext_vector_type(4)));

constexpr int SCR_COPIES = 0;              // scratch[0]: copies to make
constexpr int SCR_LIST = 4;                // then src, dst, rows of each copy (FA_CACHE_MAX_SLOTS triples)
constexpr int SCR_FREE = SCR_LIST + 3 * FA_CACHE_MAX_SLOTS;   // then the free pages taken, lowest first

__device__ __forceinline__ int blocks_of(int64_t tokens, int page_size) { return (int)((tokens + page_size - 1) / page_size); }
__device__ __forceinline__ void flag(const FaCache &c, int bit) { atomicOr(c.status, bit); }

// whether slots[i] may be worked on: in range and named once in the call (a WG asks with all its threads)
__device__ bool slot_ok(const FaCache &c, const int32_t *slots, int n, int i, int slot) {
    int twice = 0;
    for (int j = threadIdx.x; j < n; j += blockDim.x) twice |= j != i && slots[j] == slot;
    const bool bad = __syncthreads_or(twice) || slot < 0 || slot >= c.max_seqs;
    if (bad && threadIdx.x == 0) flag(c, FA_CACHE_BAD_SLOT);
    return !bad;
}

// gives back the table entries [from, to) of a sequence
__device__ void release(const FaCache &c, int32_t *tbl, int from, int to) {
    for (int b = from + (int)threadIdx.x; b < to; b += blockDim.x) {
        const int page = tbl[b];
        tbl[b] = -1;
        if (page >= 0 && page < c.num_pages) atomicSub(c.refcount + page, 1);
    }
}

// exclusive prefix sums of one value per thread over a workgroup of 1024; total to all. tmp: 16 words, free again after
// the next barrier
template <typename V>
__device__ V scan1024(V v, V *tmp, V &total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    V x = v;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
        const V y = __shfl_up(x, s);
        if (lane >= s) x += y;
    }
    if (lane == 63) tmp[wave] = x;
    __syncthreads();
    V before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const V y = tmp[i];
        before += i < wave ? y : 0;
        all += y;
    }
    total = all;
    return before + x - v;
}

// One workgroup: what each slot needs, the lowest free pages that cover it, then the tables. Nothing is written to
// them before all is known to fit. Bound by the chain of dependent loads (slots, lengths, entries, counts), so the first
// 4096 pages' counts are on their way from the start, and each thread keeps its slots in registers. 9 us for 32 slots, 15 for
// 256 beams that share their last page.
constexpr int RES_PER = FA_CACHE_MAX_SLOTS / 1024;
__global__ __launch_bounds__(1024) void cache_reserve_kernel(const FaCache c, const int32_t *slots, int n,
                                                             const int32_t *counts, int count) {
    __shared__ uint32_t named[FA_CACHE_MAX_SEQS / 32];
    __shared__ __attribute__((aligned(16))) int shared_page[FA_CACHE_MAX_SLOTS];      // a partly full page that others hold too, or -1
    __shared__ int sbad;
    __shared__ long long tmp[2][16];
    __shared__ int tmp32[2][16];
    const int tid = threadIdx.x, lane = tid & 63, ps = c.page_size;
    auto free_at = [&](int p) -> bool { return p < c.num_pages && c.refcount[p] == 0; };
    bool is_free[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) is_free[x] = free_at(tid * 4 + x);
    const int per = (n + 1023) / 1024;                   // consecutive slots to a thread
    int slot[RES_PER], cnt[RES_PER];
#pragma unroll
    for (int x = 0; x < RES_PER; ++x) {
        const int i = tid * per + x;
        slot[x] = x < per && i < n ? slots[i] : -1;
        cnt[x] = x < per && i < n && counts ? counts[i] : count;
    }
    if (tid == 0) {
        c.scratch[SCR_COPIES] = 0;
        sbad = 0;
    }
    for (int i = tid; i < FA_CACHE_MAX_SEQS / 32; i += 1024) named[i] = 0;
    for (int i = tid; i < FA_CACHE_MAX_SLOTS; i += 1024) shared_page[i] = -1;
    __syncthreads();
    int bad = 0, len[RES_PER], have[RES_PER], page[RES_PER], refs[RES_PER];
#pragma unroll
    for (int x = 0; x < RES_PER; ++x) {
        const int s = slot[x];
        len[x] = have[x] = refs[x] = 0;
        page[x] = -1;
        if (s == -1) continue;
        slot[x] = -1;
        if (s < 0 || s >= c.max_seqs || (atomicOr(&named[s >> 5], 1u << (s & 31)) >> (s & 31) & 1)) {
            bad |= FA_CACHE_BAD_SLOT;
        } else if (cnt[x] < 0) {
            bad |= FA_CACHE_BAD_LENGTH;
        } else if (cnt[x] > 0) {
            len[x] = c.seqlens[s];
            have[x] = c.nblocks[s];
            if (((int64_t)len[x] + cnt[x] + ps - 1) / ps > c.max_blocks) {
                bad |= FA_CACHE_TOO_LONG;
                continue;
            }
            slot[x] = s;
            if (len[x] % ps) {
                const int p = c.block_table[(int64_t)s * c.max_blocks + len[x] / ps];
                if (p < 0 || p >= c.num_pages) {
                    bad |= FA_CACHE_NOT_RESERVED;        // the last token's page was given back
                } else if ((refs[x] = c.refcount[p]) > 1) {
                    page[x] = p;
                    shared_page[tid * per + x] = p;
                }
            }
        }
    }
    if (bad) atomicOr(&sbad, bad);
    __syncthreads();
    if (sbad) {
        if (tid == 0) flag(c, sbad);
        return;
    }
    // a shared page is copied unless this is its last holder: earlier slots of the call leave it first
    long long mine = 0;                                  // pages needed (4096 times 2^26 at most), copies above them
    constexpr int COPY_BIT = 48;
    int need[RES_PER];
    bool copy[RES_PER];
#pragma unroll
    for (int x = 0; x < RES_PER; ++x) {
        const int i = tid * per + x;
        need[x] = 0;
        copy[x] = false;
        if (slot[x] < 0) continue;
        if (page[x] >= 0) {
            int before = 0;
            typedef int i32x4s __attribute__((ext_vector_type(4)));
            for (int j = 0; j < i; j += 4) {
                const i32x4s o = *(const i32x4s *)(shared_page + j);
#pragma unroll
                for (int e = 0; e < 4; ++e) before += j + e < i && o[e] == page[x];
            }
            copy[x] = refs[x] - before > 1;
        }
        const int more = blocks_of((int64_t)len[x] + cnt[x], ps) - have[x];
        need[x] = (copy[x] ? 1 : 0) + (more > 0 ? more : 0);
        mine += need[x] + ((long long)copy[x] << COPY_BIT);
    }
    long long sums;
    const long long at0 = scan1024<long long>(mine, tmp[0], sums);
    const int ncopies = (int)(sums >> COPY_BIT);
    const long long wanted = sums & ((1ll << COPY_BIT) - 1);
    if (wanted == 0) return;
    if (wanted > c.num_pages) {
        if (tid == 0) flag(c, FA_CACHE_NO_PAGES);
        return;
    }
    const int total = (int)wanted;
    // the `total` lowest free pages, in order
    int32_t *list = c.scratch + SCR_FREE;
    int found = 0;
    for (int p0 = 0, round = 0; p0 < c.num_pages && found < total; p0 += 4096, round ^= 1) {
        if (p0 > 0) {
#pragma unroll
            for (int x = 0; x < 4; ++x) is_free[x] = free_at(p0 + tid * 4 + x);
        }
        const int f = (int)is_free[0] + is_free[1] + is_free[2] + is_free[3];
        int here, at = found + scan1024<int>(f, tmp32[round], here);
#pragma unroll
        for (int x = 0; x < 4; ++x)
            if (is_free[x]) {
                if (at < total) list[at] = p0 + tid * 4 + x;
                ++at;
            }
        found += here;
    }
    if (found < total) {
        if (tid == 0) flag(c, FA_CACHE_NO_PAGES);
        return;
    }
    if (tid == 0) c.scratch[SCR_COPIES] = ncopies;
    __threadfence();
    __syncthreads();
    // the tables: a thread sets its slots' copies and first new blocks, its wave the rest of long ones
    constexpr int OWN = 4;
    int rank = (int)(at0 & ((1ll << COPY_BIT) - 1)), crank = (int)(at0 >> COPY_BIT);
#pragma unroll
    for (int x = 0; x < RES_PER; ++x) {
        const int64_t row = (int64_t)slot[x] * c.max_blocks;
        if (copy[x]) {
            const int p = list[rank++];
            c.block_table[row + len[x] / ps] = p;
            c.refcount[p] = 1;
            atomicSub(c.refcount + page[x], 1);
            int32_t *e = c.scratch + SCR_LIST + 3 * crank++;
            e[0] = page[x];
            e[1] = p;
            e[2] = len[x] % ps;
        }
        const int more = need[x] - (copy[x] ? 1 : 0);
        for (int b = 0; b < more && b < OWN; ++b) {
            const int p = list[rank + b];
            c.block_table[row + have[x] + b] = p;
            c.refcount[p] = 1;
        }
        if (more > 0) c.nblocks[slot[x]] = have[x] + more;
        uint64_t longer = __builtin_amdgcn_ballot_w64(more > OWN);
        while (longer) {
            const int src = __builtin_ctzll(longer);
            longer &= longer - 1;
            const int s = __shfl(slot[x], src), h = __shfl(have[x], src), m = __shfl(more, src), r = __shfl(rank, src);
            for (int b = OWN + lane; b < m; b += 64) {
                const int p = list[r + b];
                c.block_table[(int64_t)s * c.max_blocks + h + b] = p;
                c.refcount[p] = 1;
            }
        }
        rank += more;
    }
}

// The copies that reserve found: the first `rows` rows of page src into page dst, K and V of every layer. A fixed
// grid walks pieces of 16 KiB, so a call with nothing to copy costs an empty launch. Bound by memory: 1.06 GB read and
// written in 158 us (much of it still in the last cache).
constexpr int COPY_PIECE = 16384;
__global__ __launch_bounds__(256) void cache_copy_kernel(const FaCache c) {
    const int ncopies = c.scratch[SCR_COPIES];
    if (ncopies == 0) return;
    const int64_t row = (int64_t)c.nheads * c.head_dim * 2, page = row * c.page_size, layer = page * c.num_pages;
    const int pieces = (int)((page + COPY_PIECE - 1) / COPY_PIECE);
    const int64_t jobs = (int64_t)ncopies * c.layers * 2 * pieces;
    for (int64_t j = blockIdx.x; j < jobs; j += gridDim.x) {
        const int piece = (int)(j % pieces);
        const int64_t r = j / pieces;
        const int l = (int)(r / 2 % c.layers);
        const int32_t *e = c.scratch + SCR_LIST + 3 * (r / 2 / c.layers);
        const int64_t bytes = e[2] * row, beg = (int64_t)piece * COPY_PIECE;
        const int64_t end = bytes < beg + COPY_PIECE ? bytes : beg + COPY_PIECE;
        char *pool = (char *)(r & 1 ? c.v_pages : c.k_pages) + l * layer;
        const char *src = pool + e[0] * page;
        char *dst = pool + e[1] * page;
        u32x4v v[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const int64_t o = beg + (threadIdx.x + 256 * x) * 16;
            if (o < end) v[x] = *(const u32x4v *)(src + o);
        }
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const int64_t o = beg + (threadIdx.x + 256 * x) * 16;
            if (o < end) *(u32x4v *)(dst + o) = v[x];
        }
    }
}

// New rows into their pages: blockIdx.y the slot; a block takes `lines` tokens, a lane one 16-byte piece of a row, in K
// and in V. Bound by HBM for long calls (16 sequences of 8192 tokens, 8 heads of 128: 209 us, 5.1 TB/s; with four tokens
// to a lane, and a quarter of the blocks, 226), by launch and three dependent loads (length, table, count) for short
// ones (32 sequences of 64 tokens, 8 heads of 128: 6.1 us against 7.5).
__global__ __launch_bounds__(256) void cache_write_kernel(const FaCache c, int layer, const int32_t *slots,
                                                          const uint16_t *k, int64_t k_rs, int64_t k_hs,
                                                          const uint16_t *v, int64_t v_rs, int64_t v_hs,
                                                          const int32_t *cu, int64_t total, int n, int lines) {
    const int i = blockIdx.y, s = slots[i];
    int beg = cu[i], end = cu[i + 1];
    if (s == -1 || !slot_ok(c, slots, n, i, s)) return;
    beg = beg < 0 ? 0 : beg;
    end = end > total ? (int)total : end;
    const int hc = c.head_dim / 8, chunks = c.nheads * hc;
    const int t0 = beg + blockIdx.x * lines;
    if (t0 >= end) return;
    const int len = c.seqlens[s], have = c.nblocks[s], shift = __builtin_ctz(c.page_size);
    const int64_t row = (int64_t)c.nheads * c.head_dim, layer0 = (int64_t)layer * c.num_pages * c.page_size * row;
    // rows wider than a block: several pieces to a lane
    const int line = lines > 1 ? threadIdx.x / chunks : 0, t = t0 + line;
    const int at = len + t - beg, blk = at >> shift;
    if (line >= lines || t >= end) return;
    const int page = at >= 0 && blk < have ? c.block_table[(int64_t)s * c.max_blocks + blk] : -1;
    const bool own = page >= 0 && page < c.num_pages && c.refcount[page] == 1;
    const int64_t to = layer0 + (((int64_t)page << shift) + (at & (c.page_size - 1))) * row;
    for (int ch = threadIdx.x - line * chunks; ch < chunks; ch += 256) {
        const int h = ch / hc, d = (ch - h * hc) * 8;
        const u32x4v x = *(const u32x4v *)(k + (int64_t)t * k_rs + (int64_t)h * k_hs + d);
        const u32x4v y = *(const u32x4v *)(v + (int64_t)t * v_rs + (int64_t)h * v_hs + d);
        if (own) {
            *(u32x4v *)((uint16_t *)c.k_pages + to + ch * 8) = x;
            *(u32x4v *)((uint16_t *)c.v_pages + to + ch * 8) = y;
        }
    }
    if (!own) flag(c, FA_CACHE_NOT_RESERVED);
}

// What compact asks of slots[i]; the same answer in both of its kernels, since the first changes no table. Writes
// the rows (page * page_size + row) of the kept tokens and of their new places to LDS. -1: leave the slot alone.
__device__ int keep_ok(const FaCache &c, const int32_t *slots, int n, int i, const int32_t *keep, int max_keep,
                       const int32_t *counts, int *src, int *dst) {
    const int s = slots[i];
    if (s == -1) return -1;
    if (!slot_ok(c, slots, n, i, s)) return -1;
    const int m = counts[i], len = c.seqlens[s], have = c.nblocks[s];
    int bad = m < 0 || m > max_keep ? FA_CACHE_BAD_KEEP : 0;
    if (!bad)
        for (int j = threadIdx.x; j < m; j += blockDim.x) {
            const int from = keep[j];
            if (from < j || (j > 0 && keep[j - 1] >= from)) {
                bad |= FA_CACHE_BAD_KEEP;
                continue;
            }
            const int64_t a = (int64_t)len + from, b = (int64_t)len + j;
            const int64_t room = (int64_t)have * c.page_size;
            const int pa = a < room ? c.block_table[(int64_t)s * c.max_blocks + a / c.page_size] : -1;
            const int pb = b < room ? c.block_table[(int64_t)s * c.max_blocks + b / c.page_size] : -1;
            if (pa < 0 || pa >= c.num_pages || pb < 0 || pb >= c.num_pages || c.refcount[pb] != 1) {
                bad |= FA_CACHE_NOT_RESERVED;
                continue;
            }
            src[j] = pa * c.page_size + (int)(a % c.page_size);
            dst[j] = pb * c.page_size + (int)(b % c.page_size);
        }
    const int keep_bad = __syncthreads_or(bad & FA_CACHE_BAD_KEEP), room_bad = __syncthreads_or(bad & FA_CACHE_NOT_RESERVED);
    if (keep_bad || room_bad) {
        if (threadIdx.x == 0) flag(c, keep_bad ? FA_CACHE_BAD_KEEP : FA_CACHE_NOT_RESERVED);
        return -1;
    }
    return m;
}

// Moves the kept rows together, in place. A lane owns 16 bytes of a row in one layer of K or V and moves them in
// ascending order: a row's new place is at or before its old one and before every later row's, so nothing is
// overwritten before it is read; sixteen rows are read before the first of them is written. 10 us for 32 slots, 12 layers of
// 8 heads of 128: mostly the chain of loads to the rows' places.
__global__ __launch_bounds__(128) void cache_move_kernel(const FaCache c, const int32_t *slots, int n,
                                                         const int32_t *keep, int64_t keep_stride, int max_keep,
                                                         const int32_t *counts) {
    extern __shared__ int rows[];
    const int i = blockIdx.x;
    int *src = rows, *dst = rows + max_keep;
    const int m = keep_ok(c, slots, n, i, keep + i * keep_stride, max_keep, counts, src, dst);
    if (m <= 0) return;
    const int chunks = c.nheads * c.head_dim / 8;
    const int ch = blockIdx.z * 128 + threadIdx.x;
    if (ch >= chunks) return;
    const int64_t row = (int64_t)c.nheads * c.head_dim;
    uint16_t *pool = (uint16_t *)(blockIdx.y & 1 ? c.v_pages : c.k_pages) +
                     (int64_t)(blockIdx.y >> 1) * c.num_pages * c.page_size * row + ch * 8;
    for (int j = 0; j < m; j += 16) {
        u32x4v v[16];
#pragma unroll
        for (int x = 0; x < 16; ++x)
            if (j + x < m && src[j + x] != dst[j + x]) v[x] = *(const u32x4v *)(pool + src[j + x] * row);
#pragma unroll
        for (int x = 0; x < 16; ++x)
            if (j + x < m && src[j + x] != dst[j + x]) *(u32x4v *)(pool + dst[j + x] * row) = v[x];
    }
}

__global__ __launch_bounds__(128) void cache_kept_kernel(const FaCache c, const int32_t *slots, int n,
                                                         const int32_t *keep, int64_t keep_stride, int max_keep,
                                                         const int32_t *counts) {
    extern __shared__ int rows[];
    const int i = blockIdx.x;
    const int m = keep_ok(c, slots, n, i, keep + i * keep_stride, max_keep, counts, rows, rows + max_keep);
    if (m < 0) return;
    const int s = slots[i], len = c.seqlens[s] + m, have = c.nblocks[s], need = blocks_of(len, c.page_size);
    __syncthreads();
    release(c, c.block_table + (int64_t)s * c.max_blocks, need, have);
    if (threadIdx.x == 0) {
        c.seqlens[s] = len;
        if (need < have) c.nblocks[s] = need;
    }
}

__global__ __launch_bounds__(128) void cache_truncate_kernel(const FaCache c, const int32_t *slots, int n,
                                                             const int32_t *lens) {
    const int i = blockIdx.x, s = slots[i];
    if (s == -1 || !slot_ok(c, slots, n, i, s)) return;
    int32_t *tbl = c.block_table + (int64_t)s * c.max_blocks;
    const int len = lens ? lens[i] : 0, old = c.seqlens[s];
    int have = c.nblocks[s];
    have = have < 0 ? 0 : (have > c.max_blocks ? c.max_blocks : have);
    bool bad = len < 0 || (lens && len > old);
    if (!bad && len > 0 && c.window > 0) {
        // the next token sees the keys from len - window + 1 on; pages are evicted from the front
        const int lo = len - c.window + 1 > 0 ? len - c.window + 1 : 0;
        if (lo < len && tbl[lo / c.page_size] < 0) bad = true;
    }
    __syncthreads();
    if (bad) {
        if (threadIdx.x == 0) flag(c, FA_CACHE_BAD_LENGTH);
        return;
    }
    const int need = blocks_of(len, c.page_size);
    release(c, tbl, need, have);
    if (threadIdx.x == 0) {
        c.seqlens[s] = len;
        c.nblocks[s] = need < have ? need : have;
    }
}

__global__ __launch_bounds__(128) void cache_evict_kernel(const FaCache c, const int32_t *slots, int n) {
    const int i = blockIdx.x, s = slots[i];
    if (s == -1 || !slot_ok(c, slots, n, i, s)) return;
    const int gone = c.seqlens[s] - c.window + 1;     // keys before it are behind the window of every later token
    int end = gone > 0 ? gone / c.page_size : 0;
    end = end < c.nblocks[s] ? end : c.nblocks[s];
    release(c, c.block_table + (int64_t)s * c.max_blocks, blocks_of(c.num_sinks, c.page_size), end);
}

__global__ __launch_bounds__(128) void cache_fork_kernel(const FaCache c, const int32_t *parents,
                                                         const int32_t *children, int n) {
    const int i = blockIdx.x, p = parents[i], s = children[i];
    if (p == -1 && s == -1) return;
    if (!slot_ok(c, children, n, i, s)) return;
    int crossed = p < 0 || p >= c.max_seqs;
    for (int j = threadIdx.x; j < n; j += 128) crossed |= parents[j] == s;   // a child is nobody's parent here
    if (__syncthreads_or(crossed)) {
        if (threadIdx.x == 0) flag(c, FA_CACHE_BAD_SLOT);
        return;
    }
    const bool full = c.nblocks[s] != 0 || c.seqlens[s] != 0;
    const int len = c.seqlens[p], need = blocks_of(len, c.page_size);
    __syncthreads();
    if (full) {
        if (threadIdx.x == 0) flag(c, FA_CACHE_NOT_EMPTY);
        return;
    }
    const int32_t *from = c.block_table + (int64_t)p * c.max_blocks;
    int32_t *to = c.block_table + (int64_t)s * c.max_blocks;
    for (int b = threadIdx.x; b < need; b += 128) {
        const int page = from[b];
        to[b] = page;
        if (page >= 0 && page < c.num_pages) atomicAdd(c.refcount + page, 1);
    }
    if (threadIdx.x == 0) {
        c.seqlens[s] = len;
        c.nblocks[s] = need;
    }
}

int check_cache(const char *fn, const FaCache *c, const int32_t *slots, int n) {
    if (!c) return set_error(FA_ERR_INVALID_ARGUMENT, "%s: cache is NULL", fn);
    if (c->layers <= 0 || c->num_pages <= 0 || c->nheads <= 0 || c->head_dim <= 0 || c->max_seqs <= 0 || c->max_blocks <= 0)
        return set_error(FA_ERR_INVALID_ARGUMENT, "%s: sizes of the cache must be positive", fn);
    if (c->page_size < 16 || (c->page_size & (c->page_size - 1)))
        return set_error(FA_ERR_UNSUPPORTED, "%s: page_size must be a power of two, 16 or more (got %d)", fn, c->page_size);
    if (c->head_dim % 8 || c->head_dim > 128)
        return set_error(FA_ERR_UNSUPPORTED, "%s: head_size must be a multiple of 8 and <= 128 (got %d)", fn, c->head_dim);
    if (c->max_seqs > FA_CACHE_MAX_SEQS) return set_error(FA_ERR_UNSUPPORTED, "%s: more than %d sequences", fn, (int)FA_CACHE_MAX_SEQS);
    if ((int64_t)c->num_pages * c->page_size >= (int64_t)1 << 31 || (int64_t)c->max_blocks * c->page_size >= (int64_t)1 << 30)
        return set_error(FA_ERR_UNSUPPORTED, "%s: 2^31 rows of pages, or 2^30 tokens in a sequence, or more", fn);
    if (c->window < 0 || c->num_sinks < 0) return set_error(FA_ERR_INVALID_ARGUMENT, "%s: window and num_sinks must be >= 0", fn);
    if (!c->k_pages || !c->v_pages || !c->block_table || !c->seqlens || !c->nblocks || !c->refcount || !c->status || !c->scratch)
        return set_error(FA_ERR_INVALID_ARGUMENT, "%s: NULL pointer in the cache", fn);
    if ((((uintptr_t)c->k_pages | (uintptr_t)c->v_pages) & 15) != 0)
        return set_error(FA_ERR_INVALID_ARGUMENT, "%s: pages must be 16-byte aligned", fn);
    if (n < 0 || n > FA_CACHE_MAX_SLOTS)
        return set_error(FA_ERR_UNSUPPORTED, "%s: 0 to %d slots a call (got %d)", fn, (int)FA_CACHE_MAX_SLOTS, n);
    if (n > 0 && !slots) return set_error(FA_ERR_INVALID_ARGUMENT, "%s: slots is NULL", fn);
    return FA_OK;
}

int launched(const char *fn) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? FA_OK : set_error(FA_ERR_LAUNCH, "%s: HIP error %d (%s)", fn, (int)e, hipGetErrorString(e));
}

}  // namespace
}  // namespace fa

using namespace fa;

extern "C" {

int64_t fa_cache_struct_size(void) { return (int64_t)sizeof(FaCache); }
int64_t fa_cache_scratch_words(int32_t num_pages) { return (int64_t)SCR_FREE + (num_pages > 0 ? num_pages : 0); }

int fa_cache_reserve(const FaCache *c, const int32_t *slots, int32_t n, const int32_t *counts, int32_t count, void *stream) {
    clear_error();
    const int rc = check_cache("fa_cache_reserve", c, slots, n);
    if (rc) return rc;
    if (!counts && count < 0) return set_error(FA_ERR_INVALID_ARGUMENT, "fa_cache_reserve: count must be >= 0");
    if (n == 0) return FA_OK;
    hipLaunchKernelGGL(cache_reserve_kernel, dim3(1), dim3(1024), 0, (hipStream_t)stream, *c, slots, n, counts, count);
    const int64_t page = (int64_t)c->nheads * c->head_dim * 2 * c->page_size;
    const int64_t most = (int64_t)n * c->layers * 2 * ((page + COPY_PIECE - 1) / COPY_PIECE);
    hipLaunchKernelGGL(cache_copy_kernel, dim3((uint32_t)(most < 2048 ? most : 2048)), dim3(256), 0, (hipStream_t)stream, *c);
    return launched("fa_cache_reserve");
}

int fa_cache_write(const FaCache *c, int32_t layer, const int32_t *slots, int32_t n, const void *k, int64_t k_rs,
                   int64_t k_hs, const void *v, int64_t v_rs, int64_t v_hs, const int32_t *cu, int64_t total,
                   int32_t max_seqlen, void *stream) {
    clear_error();
    const int rc = check_cache("fa_cache_write", c, slots, n);
    if (rc) return rc;
    if (layer < 0 || layer >= c->layers)
        return set_error(FA_ERR_INVALID_ARGUMENT, "fa_cache_write: layer %d of %d", layer, c->layers);
    if (total < 0 || total >= (int64_t)1 << 30 || max_seqlen < 0 || max_seqlen >= 1 << 30)
        return set_error(FA_ERR_INVALID_ARGUMENT, "fa_cache_write: lengths must be in [0, 2^30)");
    if (n == 0 || total == 0 || max_seqlen == 0) return FA_OK;
    if (!k || !v || !cu) return set_error(FA_ERR_INVALID_ARGUMENT, "fa_cache_write: NULL pointer");
    if ((((uintptr_t)k | (uintptr_t)v) & 15) != 0 || (k_rs | k_hs | v_rs | v_hs) % 8)
        return set_error(FA_ERR_INVALID_ARGUMENT, "fa_cache_write: k and v must be 16-byte aligned with strides multiple of 8");
    const int chunks = c->nheads * c->head_dim / 8;
    const int lines = chunks < 256 ? 256 / chunks : 1;       // tokens a block takes at a time
    const dim3 grid((max_seqlen + lines - 1) / lines, n);
    hipLaunchKernelGGL(cache_write_kernel, grid, dim3(256), 0, (hipStream_t)stream, *c, layer, slots, (const uint16_t *)k,
                       k_rs, k_hs, (const uint16_t *)v, v_rs, v_hs, cu, total, n, lines);
    return launched("fa_cache_write");
}

int fa_cache_compact(const FaCache *c, const int32_t *slots, int32_t n, const int32_t *keep, int64_t keep_stride,
                     int32_t max_keep, const int32_t *counts, void *stream) {
    clear_error();
    const int rc = check_cache("fa_cache_compact", c, slots, n);
    if (rc) return rc;
    if (max_keep < 0 || max_keep > 4096 || keep_stride < max_keep)
        return set_error(FA_ERR_UNSUPPORTED, "fa_cache_compact: 0 to 4096 tokens kept a call (got %d)", max_keep);
    if (c->layers > 32767) return set_error(FA_ERR_UNSUPPORTED, "fa_cache_compact: more than 32767 layers");
    if (n == 0) return FA_OK;
    if (!counts || (max_keep > 0 && !keep)) return set_error(FA_ERR_INVALID_ARGUMENT, "fa_cache_compact: NULL pointer");
    const int lds = 8 * max_keep;
    const dim3 grid(n, 2 * c->layers, (c->nheads * c->head_dim / 8 + 127) / 128);
    hipLaunchKernelGGL(cache_move_kernel, grid, dim3(128), lds, (hipStream_t)stream, *c, slots, n, keep, keep_stride, max_keep, counts);
    hipLaunchKernelGGL(cache_kept_kernel, dim3(n), dim3(128), lds, (hipStream_t)stream, *c, slots, n, keep, keep_stride, max_keep, counts);
    return launched("fa_cache_compact");
}

int fa_cache_fork(const FaCache *c, const int32_t *parents, const int32_t *children, int32_t n, void *stream) {
    clear_error();
    int rc = check_cache("fa_cache_fork", c, parents, n);
    if (rc) return rc;
    if (n == 0) return FA_OK;
    if (!children) return set_error(FA_ERR_INVALID_ARGUMENT, "fa_cache_fork: children is NULL");
    hipLaunchKernelGGL(cache_fork_kernel, dim3(n), dim3(128), 0, (hipStream_t)stream, *c, parents, children, n);
    return launched("fa_cache_fork");
}

int fa_cache_truncate(const FaCache *c, const int32_t *slots, int32_t n, const int32_t *lens, void *stream) {
    clear_error();
    const int rc = check_cache("fa_cache_truncate", c, slots, n);
    if (rc) return rc;
    if (n == 0) return FA_OK;
    hipLaunchKernelGGL(cache_truncate_kernel, dim3(n), dim3(128), 0, (hipStream_t)stream, *c, slots, n, lens);
    return launched("fa_cache_truncate");
}

int fa_cache_evict(const FaCache *c, const int32_t *slots, int32_t n, void *stream) {
    clear_error();
    const int rc = check_cache("fa_cache_evict", c, slots, n);
    if (rc) return rc;
    if (c->window == 0) return set_error(FA_ERR_INVALID_ARGUMENT, "fa_cache_evict: the cache has no window");
    if (n == 0) return FA_OK;
    hipLaunchKernelGGL(cache_evict_kernel, dim3(n), dim3(128), 0, (hipStream_t)stream, *c, slots, n);
    return launched("fa_cache_evict");
}

}  // extern "C"
