// fa_window_fwd_kernel.h — forward attention with a sliding window and sinks, dense or over a paged cache.
//
// For each query row: m = max_j s_j over the keys it sees (s_j = scale q.k_j), l = sum exp(s_j - m),
// O = sum exp(s_j - m) v_j / l, lse = m + log l, in one pass over the keys with running m, l and O (fp32).
//
// A workgroup has NWR row waves (32 packed rows each, fa_window_common.h) times KG key groups. Tiles of BN keys
// go HBM -> LDS by LDS-DMA into two buffers per key group; the scores are computed swapped (S^T = K Q^T), so a
// lane owns a row: its mask is one 32-bit word per 32 keys, its max and sum need one lane exchange per tile, and
// P feeds O^T += V^T P^T from registers (rounded to 16 bits, the operand type of the matrix instruction, or in two
// such parts, see FINE; the sum l takes P unrounded). Key groups walk every KG-th tile and are joined through LDS at the end; a split walks a
// contiguous share of the tiles and leaves O, m and l in the workspace for fa_window_join_kernel.
//
// What bounds it. Dense, head_dim 128: 32768 tokens, 8 heads on 2, window 4096: 562 us, 931 TFLOP/s of the 1273 that a
// large library product reaches here; matrix units 52 % busy, vector units 52 %, LDS 27 %, at two waves a SIMD, whose
// phases hide each other hardly more: one half tile's exponentials placed between the other's products, and priorities
// for either phase, changed nothing. At head_dim 64 the softmax takes twice the matrix instructions' time (vector units
// 65 % busy, matrix units 23 %), and short windows the latency of a workgroup's start and end: 8 x 2048 tokens, 12 heads,
// window 256: 39 us. Paged, few rows: HBM; 64 single tokens over caches of up to 8191, 32 heads of 128 on 8: 232 us,
// 4.8 TB/s (a copy of 2 GiB: 4.9).
//
// Tiles that a wave sees whole take no mask; a tile at the window's edge, the diagonal or the end takes the mask
// path, as does one with drafted tokens or a page that is not there.
#pragma once

#include "fa_window_careful.h"

namespace fa {

struct WinFwdArgs {
    const uint16_t *q, *k, *v;
    uint16_t *o;
    float *lse;
    const int32_t *cu_q, *cu_k;
    const int32_t *table, *ctx, *seq_ids;
    const uint64_t *tree;
    float *ws_o, *ws_ml;          // [nsplit][total_q * nheads][D], [nsplit][total_q * nheads][2]
    int64_t q_rs, q_hs, o_rs, o_hs;
    int64_t k_ps, k_rs, k_hs, v_ps, v_rs, v_hs;
    int64_t table_stride, total_q, total_k;
    int batch, nheads, nheads_k, head_dim, group;
    int num_pages, page_shift, num_seqs, max_blocks, tree_words;
    int max_q, lse_stride, window, sinks, nrb, nsplit;
    int fine;                     // dense: which of the two kernels
    float scale;
    Div dgroup, dheads, dsplit;   // by group, nheads_k, nsplit
    BlockOrder order;             // dense; paged: its blk divides by nrb
};

__device__ __forceinline__ float wmax3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

template <int D, int NWR, int KG, int BN>
struct WinFwdCfg {
    static constexpr int NT = 64 * NWR * KG;
    static constexpr int BM = 32 * NWR;
    static constexpr int NS = BN / 32;
    static constexpr int NC = D / 8;
    static constexpr int TILE = BN * D * 2;            // bytes of one K or V tile
    static constexpr int GROUP_LDS = 4 * TILE;         // K[2], V[2]
    static constexpr int PIECES = TILE / 1024;
    static constexpr int PPW = (PIECES + NWR - 1) / NWR;
    static constexpr int RPP = 1024 / (2 * D);         // rows per 1-KiB piece
    static constexpr int MERGE = KG > 1 ? (KG - 1) * NWR * (32 * D * 4 + 64 * 8) : 0;
    static constexpr int TREE_OFF = KG * GROUP_LDS > MERGE ? KG * GROUP_LDS : MERGE;
    static constexpr int lds(bool tree) { return TREE_OFF + (tree ? 256 * 4 : 0); }
};

// P stays below 2^8: the running maximum is moved only when a tile passes it by that much, so O and l are
// rarely rescaled. The same relative rounding, and fp16's smallest P is 2^8 times nearer to the row's largest.
constexpr float WIN_RESCALE = 8.0f;

//
// FINE: P goes to the product in two 16-bit parts, what the first leaves in the second, with half as many matrix
// instructions more. Rounded once, P brings as much error as the rounding of the output (rms, together 1.41 of it);
// so 1.0. Taken where it costs nothing or little: few rows over a cache (HBM or latency bounds them: 64 single
// tokens over caches of up to 8191 take 235 us for 233) and small dense calls (takes_fine, fa_window_api.cpp).
template <int D, typename T, int NWR, int KG, int BN, bool PAGED, bool TREE, bool FINE>
__global__ __launch_bounds__(64 * NWR * KG) void fa_window_fwd_kernel(const WinFwdArgs a) {
    using C = WinFwdCfg<D, NWR, KG, BN>;
    using S = Swz<D>;
    constexpr float LOG2E = 1.4426950408889634f;
    constexpr float LN2 = 0.6931471805599453f;
    extern __shared__ __attribute__((aligned(16))) char smem[];

    // ---- block -> (row block, split, key/value head, sequence). The row blocks of one split of a paged call share
    // its K/V and follow each other.
    int rb, split = 0, w;
    if constexpr (PAGED) {
        w = xcd_contiguous(blockIdx.x, gridDim.x);
        int x = a.order.blk.div(w);
        rb = w - x * a.nrb;
        w = a.dsplit.div(x);
        split = x - w * a.nsplit;
    } else {
        a.order.get(blockIdx.x, rb, w);
    }
    const int b = a.dheads.div(w);
    const int kvh = w - b * a.nheads_k;

    int q_start, len_q, klen, off;
    const uint16_t *kbase, *vbase;
    const int32_t *tbl = nullptr;
    seq_bounds(a.cu_q, b, a.total_q, q_start, len_q);
    const int sq = len_q < a.max_q ? len_q : a.max_q;             // lse's rows (masks, depth_s) end at max_q
    const int G = a.group;
    const int R = sq * G;
    const int r0 = rb * C::BM;
    if (r0 >= R) {
        zero_tail(a.o, a.o_rs, a.o_hs, a.nheads, a.head_dim, a.total_q, a.cu_q, a.batch);
        return;
    }
    if constexpr (PAGED) {
        const int row = a.seq_ids ? a.seq_ids[b] : b;
        const bool used = row >= 0 && row < a.num_seqs;
        int ctx = used ? a.ctx[row] : 0;
        ctx = ctx < 0 ? 0 : ctx;
        const int64_t room = (int64_t)a.max_blocks << a.page_shift;
        if (ctx > room) ctx = (int)room;
        off = ctx;
        const int64_t end = (int64_t)ctx + len_q;
        klen = used ? (int)(end < room ? end : room) : 0;
        tbl = a.table + (int64_t)(used ? row : 0) * a.table_stride;
        kbase = a.k + (int64_t)kvh * a.k_hs;
        vbase = a.v + (int64_t)kvh * a.v_hs;
    } else {
        int k_start;
        seq_bounds(a.cu_k, b, a.total_k, k_start, klen);
        off = klen - len_q;
        kbase = a.k + (int64_t)k_start * a.k_rs + (int64_t)kvh * a.k_hs;
        vbase = a.v + (int64_t)k_start * a.v_rs + (int64_t)kvh * a.v_hs;
    }

    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wr = wave % NWR, kg = wave / NWR;
    const int l32 = lane & 31, hi = lane >> 5;
    const int head_dim = a.head_dim;

    // ---- this lane's row
    const int rw = r0 + 32 * wr;                              // first row of the wave
    const int row = rw + l32;
    const int rc = row < R ? row : R - 1;                     // rows behind the end compute what nobody stores
    const int t = a.dgroup.div(rc), g = rc - t * G;
    int pos = off + t;
    // positions of the wave
    int pmin = off + a.dgroup.div(rw), pmax = off + a.dgroup.div(rw + 31 < R ? rw + 31 : R - 1);
    if (rw >= R) pmin = pmax = pos;
    int bmin = off + a.dgroup.div(r0);                        // of the workgroup
    int k_end = off + a.dgroup.div(r0 + C::BM < R ? r0 + C::BM - 1 : R - 1) + 1;
    int *depth_s = (int *)(smem + C::TREE_OFF);
    const uint64_t *my_mask = nullptr;
    if constexpr (TREE) {
        // positions by depth; drafted rows reach from context - 1 (an empty mask) to the last token
        for (int i = tid; i < sq; i += C::NT) {
            int n = 0;
            for (int x = 0; x < a.tree_words; ++x) n += __popcll(a.tree[(int64_t)(q_start + i) * a.tree_words + x]);
            depth_s[i] = n;
        }
        __syncthreads();
        pos = off + depth_s[t] - 1;
        my_mask = a.tree + (int64_t)(q_start + t) * a.tree_words;
        pmin = bmin = off - 1;
        pmax = off + sq - 1;
        k_end = klen;
    }
    k_end = k_end < klen ? k_end : klen;
    const TileWalk walk = tile_walk(bmin, k_end, a.window, a.sinks, BN);
    const int per = a.dsplit.div(walk.n + a.nsplit - 1);
    const int i_beg = split * per;
    const int i_end = walk.n < i_beg + per ? walk.n : i_beg + per;
    const int steps = i_end > i_beg ? (i_end - i_beg + KG - 1) / KG : 0;

    // ---- staging. Piece p (1 KiB = RPP rows) is written by row wave p % NWR of its group; lane l lands at byte
    // 16 l of the piece, so the swizzle goes onto the source: slot l % NC of row RPP p + l / NC holds chunk
    // slot ^ x(row). Descriptors end at the last key, and rows behind it land as zeros, so that whatever a page
    // holds there (an old token, a NaN) never meets a weight of 0.
    char *const gsm = smem + kg * C::GROUP_LDS;
    int k_off[C::PPW], v_off[C::PPW];
#pragma unroll
    for (int i = 0; i < C::PPW; ++i) {
        const int p = wr + NWR * i;
        const int r = C::RPP * p + lane / C::NC;
        const int c = (lane % C::NC) ^ S::x(r);
        const bool ok = c * 8 < head_dim;
        k_off[i] = ok ? (r * (int)a.k_rs + c * 8) * 2 : OOB;
        v_off[i] = ok ? (r * (int)a.v_rs + c * 8) * 2 : OOB;
    }
    constexpr int NU = BN / 16;                               // a page holds 16 rows or more
    const bool one_page = PAGED && (1 << a.page_shift) >= BN; // pages of whole tiles: one entry to a tile
    int ent[NU];                                              // table entries of the tile to be staged next
    auto load_entries = [&](int i) __attribute__((always_inline)) {
        if constexpr (PAGED) {
            const int j0 = walk.tile(i) * BN;
            const int last = a.max_blocks - 1, b0 = j0 >> a.page_shift;
            ent[0] = uniform_load(tbl + (b0 < last ? b0 : last));
            if (!one_page) {
#pragma unroll
                for (int u = 1; u < NU; ++u) {
                    const int blk = (j0 + 16 * u) >> a.page_shift;
                    ent[u] = uniform_load(tbl + (blk < last ? blk : last));
                }
            }
        }
    };
    // stages tile i into buffer `buf`; returns the keys whose page is there, as bits of 16
    auto stage = [&](int i, int buf) __attribute__((always_inline)) -> uint32_t {
        const int j0 = walk.tile(i) * BN;
        char *kb = gsm + buf * C::TILE, *vb = gsm + (2 + buf) * C::TILE;
        uint32_t there = 0;
        if constexpr (PAGED) {
            // rows of a page from row `rin` on stand at the tile's rows from `r0` on; what is not there is not read
            auto rows_of = [&](int e, int r0, int n, i32x4 &ks, i32x4 &vs) __attribute__((always_inline)) {
                const bool ok = (uint32_t)e < (uint32_t)a.num_pages;
                int rows = klen - (j0 + r0);
                rows = !ok || rows < 0 ? 0 : (rows > n ? n : rows);
                const int64_t pg = ok ? e : 0, rin = ((j0 + r0) & ((1 << a.page_shift) - 1)) - r0;
                const int end = rows > 0 ? r0 + rows : 0;
                ks = make_srd(kbase + pg * a.k_ps + rin * a.k_rs, end * (int)a.k_rs * 2);
                vs = make_srd(vbase + pg * a.v_ps + rin * a.v_rs, end * (int)a.v_rs * 2);
            };
            i32x4 ks, vs;
            if (one_page) {
                there = (uint32_t)ent[0] < (uint32_t)a.num_pages ? (1u << NU) - 1 : 0u;
                rows_of(ent[0], 0, BN, ks, vs);
#pragma unroll
                for (int n = 0; n < C::PPW; ++n) {
                    const int p = wr + NWR * n;
                    if (C::PIECES % NWR == 0 || p < C::PIECES) {
                        dma16(ks, k_off[n], 0, lds_addr(kb + 1024 * p));
                        dma16(vs, v_off[n], 0, lds_addr(vb + 1024 * p));
                    }
                }
            } else {
#pragma unroll
                for (int u = 0; u < NU; ++u) there |= ((uint32_t)ent[u] < (uint32_t)a.num_pages ? 1u : 0u) << u;
#pragma unroll
                for (int n = 0; n < C::PPW; ++n) {
                    const int p = wr + NWR * n;
                    if (C::PIECES % NWR == 0 || p < C::PIECES) {
                        const int u = C::RPP * p / 16;
                        int e = 0;             // ent[u], u the wave's: by masks (an index would put ent in memory)
#pragma unroll
                        for (int x = 0; x < NU; ++x) e |= ent[x] & -(int)(u == x);
                        rows_of(e, C::RPP * p, C::RPP, ks, vs);
                        dma16(ks, k_off[n], 0, lds_addr(kb + 1024 * p));
                        dma16(vs, v_off[n], 0, lds_addr(vb + 1024 * p));
                    }
                }
            }
        } else {
            there = (1u << NU) - 1;
            int rows = klen - j0;
            rows = rows < 0 ? 0 : (rows > BN ? BN : rows);
            const i32x4 ks = make_srd(kbase + (int64_t)j0 * a.k_rs, rows * (int)a.k_rs * 2);
            const i32x4 vs = make_srd(vbase + (int64_t)j0 * a.v_rs, rows * (int)a.v_rs * 2);
#pragma unroll
            for (int n = 0; n < C::PPW; ++n) {
                const int p = wr + NWR * n;
                if (C::PIECES % NWR == 0 || p < C::PIECES) {
                    dma16(ks, k_off[n], 0, lds_addr(kb + 1024 * p));
                    dma16(vs, v_off[n], 0, lds_addr(vb + 1024 * p));
                }
            }
        }
        return there;
    };

    // ---- the first tile is on its way before the rows are read
    auto idx = [&](int n) __attribute__((always_inline)) -> int { return i_beg + KG * n + kg; };
    uint32_t there[2] = {0, 0};
    if (idx(0) < i_end) {
        load_entries(idx(0));
        there[0] = stage(idx(0), 0);
    }
    if (idx(1) < i_end) load_entries(idx(1));

    // ---- Q: B operand of S^T = K Q^T, element j of k-step ks is Q[row][16 ks + 8 hi + j]. A negative scale
    // turns Q's sign, a zero scale makes it 0, so that the running maximum is always of c * s with c > 0.
    const float c_log2 = (a.scale == 0.f ? 1.f : fabsf(a.scale)) * LOG2E;
    typename T::frag qf[D / 16];
    {
        const uint16_t *qp = a.q + (int64_t)(q_start + t) * a.q_rs + (int64_t)(kvh * G + g) * a.q_hs;
        const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
            const int c = 2 * ks + hi;
            u32x4 x = {0u, 0u, 0u, 0u};
            if (c * 8 < head_dim && a.scale != 0.f) {
                x = gload128(qp + c * 8);
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] ^= flip;
            }
            qf[ks] = as_frag<T>(x);
        }
    }

    // ---- lane-constant LDS offsets: K rows, and V^T by transposed reads
    const int grp = (lane >> 4) & 1, qq = (lane & 15) >> 2, pp = lane & 3;
    int k_rd[C::NS][D / 16];
#pragma unroll
    for (int st = 0; st < C::NS; ++st)
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) k_rd[st][ks] = S::off(32 * st + l32, 2 * ks + hi);
    int v_rd[D / 32][C::NS][2][2];
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
        for (int st = 0; st < C::NS; ++st)
#pragma unroll
            for (int s2 = 0; s2 < 2; ++s2) {
                const int r = 32 * st + 16 * s2 + 4 * hi + qq, col = 32 * dt + 16 * grp + 4 * pp;
                v_rd[dt][st][s2][0] = S::off8(r, col);
                v_rd[dt][st][s2][1] = S::off8(r + 8, col);
            }

    f32x16 o[D / 32];
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[dt][r] = 0.f;
    float l_i = 0.f, m_thr = -INFINITY, mc = 0.f;   // m_thr: the tile maximum that moves m; mc = m * c_log2
    const float thr_raw = WIN_RESCALE / c_log2;

    // keys j .. j+31 that a row at position `pos` (with the path `my_mask`) sees
    auto seen_by = [&](int pos, const uint64_t *my_mask, int j, uint32_t there) __attribute__((always_inline)) -> uint32_t {
        uint32_t m = seen_bits(j, pos, a.window, a.sinks) & bits_below(klen - j);
        if constexpr (TREE) {
            const int d = j - off;                            // first drafted token of the word, if not negative
            if (d + 32 > 0) {
                const int d0 = d > 0 ? d : 0, sh = d0 - d;    // sh: keys of the context at the word's start
                const int wd = d0 >> 6, bit = d0 & 63;
                uint64_t x = wd < a.tree_words ? my_mask[wd] >> bit : 0ull;
                if (bit && wd + 1 < a.tree_words) x |= my_mask[wd + 1] << (64 - bit);
                uint32_t dr = sh < 32 ? (uint32_t)x << sh : 0u;
                if (a.window < sq) {                          // else no path is longer than the window
                    for (int i = sh; i < 32; ++i) {
                        const int dd = d + i;
                        if (dd >= sq) break;
                        const int kp = off + depth_s[dd] - 1;
                        if (kp <= pos - a.window && kp >= a.sinks) dr &= ~(1u << i);
                    }
                }
                m = (m & bits_below(sh)) | (dr & bits_below(klen - j) & ~bits_below(sh));
            }
        }
        if constexpr (PAGED) m &= ((there & 1) ? 0xFFFFu : 0u) | ((there & 2) ? 0xFFFF0000u : 0u);
        return m;
    };
    auto seen = [&](int j, uint32_t there) __attribute__((always_inline)) -> uint32_t { return seen_by(pos, my_mask, j, there); };

    auto compute = [&](int j0, int buf, uint32_t there) __attribute__((always_inline)) {
        const char *kb = gsm + buf * C::TILE, *vb = gsm + (2 + buf) * C::TILE;
        f32x16 s[C::NS];
#pragma unroll
        for (int st = 0; st < C::NS; ++st) {
#pragma unroll
            for (int r = 0; r < 16; ++r) s[st][r] = 0.f;
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks)
                s[st] = T::mfma32(as_frag<T>(lds_read128(kb, k_rd[st][ks])), qf[ks], s[st]);
        }
        bool whole = j0 + BN - 1 <= pmin && (j0 > pmax - a.window || j0 + BN <= a.sinks) && j0 + BN <= klen;
        if (PAGED) whole = whole && there == (1u << NU) - 1;
        if (TREE) whole = whole && j0 + BN <= off;
        if (!__builtin_amdgcn_readfirstlane((int)whole)) {
#pragma unroll
            for (int st = 0; st < C::NS; ++st) {
                const uint32_t m = seen(j0 + 32 * st, there >> (2 * st)) >> (4 * hi);
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (!(m & (1u << crow(r, 0)))) s[st][r] = -INFINITY;
            }
        }
        // row maximum: registers, then the lane pair that shares the row
        float acc[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            float m = wmax3(s[0][4 * x], s[0][4 * x + 1], s[0][4 * x + 2]);
            if constexpr (C::NS == 2) {
                m = wmax3(m, s[0][4 * x + 3], s[C::NS - 1][4 * x]);
                m = wmax3(m, s[C::NS - 1][4 * x + 1], s[C::NS - 1][4 * x + 2]);
                acc[x] = wmax3(m, s[C::NS - 1][4 * x + 3], s[C::NS - 1][4 * x + 3]);
            } else {
                acc[x] = wmax3(m, s[0][4 * x + 3], s[0][4 * x + 3]);
            }
        }
        float mx = wmax3(wmax3(acc[0], acc[1], acc[2]), acc[3], acc[3]);
        {
            auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
            mx = wmax3(__uint_as_float(p[0]), __uint_as_float(p[1]), __uint_as_float(p[1]));
        }
        const bool grow = mx > m_thr;   // false for a row that has seen nothing yet (-inf)
        if (__builtin_amdgcn_ballot_w64(grow)) {
            const float mcx = mx * c_log2;
            const float alpha = grow ? (m_thr == -INFINITY ? 0.f : fast_exp2(mc - mcx)) : 1.f;
            if (grow) {
                m_thr = mx + thr_raw;
                mc = mcx;
            }
            l_i *= alpha;
#pragma unroll
            for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[dt][r] *= alpha;
        }
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
        typename T::frag pf[C::NS][2], pl[FINE ? C::NS : 1][2];
#pragma unroll
        for (int st = 0; st < C::NS; ++st) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[st][r] = fast_exp2(fmaf(s[st][r], c_log2, -mc));
                sum[r & 3] += s[st][r];
            }
#pragma unroll
            for (int s2 = 0; s2 < 2; ++s2) {
                u32x4 pk;
#pragma unroll
                for (int e = 0; e < 4; ++e) pk[e] = T::pack2(s[st][8 * s2 + 2 * e], s[st][8 * s2 + 2 * e + 1]);
                pf[st][s2] = as_frag<T>(pk);
                if constexpr (FINE) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        pk[e] = T::pack2(s[st][8 * s2 + 2 * e] - T::lo_float(pk[e]), s[st][8 * s2 + 2 * e + 1] - T::hi_float(pk[e]));
                    pl[st][s2] = as_frag<T>(pk);
                }
            }
        }
        l_i += (sum[0] + sum[1]) + (sum[2] + sum[3]);
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
            for (int st = 0; st < C::NS; ++st)
#pragma unroll
                for (int s2 = 0; s2 < 2; ++s2) {
                    const u32x2 lo = lds_read_tr(vb, v_rd[dt][st][s2][0]);
                    const u32x2 hv = lds_read_tr(vb, v_rd[dt][st][s2][1]);
                    const auto vt = as_frag<T>(u32x4{lo[0], lo[1], hv[0], hv[1]});
                    o[dt] = T::mfma32(vt, pf[st][s2], o[dt]);
                    if constexpr (FINE) o[dt] = T::mfma32(vt, pl[FINE ? st : 0][s2], o[dt]);
                }
    };

    // ---- the walk: wait for tile n, meet, stage tile n + 1 (over tile n - 1, which all have read), compute tile n
    auto step = [&](auto par, int n) __attribute__((always_inline)) {
        constexpr int P = decltype(par)::value;
        vmcnt0();
        if constexpr (NWR > 1) {
            __syncthreads();
        } else {
            // one wave to a group: its buffers are its own; its reads are done before it stages over them
            __builtin_amdgcn_s_waitcnt(0xC07F);   // lgkmcnt(0)
            asm volatile("" ::: "memory");
        }
        if (idx(n + 1) < i_end) there[1 - P] = stage(idx(n + 1), 1 - P);
        if (idx(n + 2) < i_end) load_entries(idx(n + 2));
        const int i = idx(n);
        if (i < i_end) {
            const int j0 = walk.tile(i) * BN;
            // a tile that none of the wave's rows sees adds nothing
            if (rw < R && j0 <= pmax && (j0 + BN - 1 > pmin - a.window || j0 < a.sinks)) compute(j0, P, there[P]);
        }
    };
    for (int n = 0; n < steps; n += 2) {
        step(std::integral_constant<int, 0>(), n);
        if (n + 1 < steps) step(std::integral_constant<int, 1>(), n + 1);
    }

    // ---- an infinity or NaN: this wave's rows again over its own tiles, key by key (fa_window_careful.h)
    if (!all_finite(o, l_i)) {
        LaneRow<D> qv, kv, vv, acc;
        for (int rr = 0; rr < 32 && rw + rr < R; ++rr) {
            const int tt = a.dgroup.div(rw + rr), gg = rw + rr - tt * G;
            qv.template load<T>(a.q + (int64_t)(q_start + tt) * a.q_rs + (int64_t)(kvh * G + gg) * a.q_hs, head_dim);
            acc.zero();
            const uint64_t *mask = nullptr;
            int p = off + tt;
            if constexpr (TREE) {
                mask = a.tree + (int64_t)(q_start + tt) * a.tree_words;
                p = off + depth_s[tt] - 1;
            }
            float m = -INFINITY, l = 0.f;
            for (int n = 0; n < steps; ++n) {
                if (idx(n) >= i_end) break;
                for (int j0 = walk.tile(idx(n)) * BN, st = 0; st < C::NS; ++st, j0 += 32) {
                    uint32_t bits = seen_by(p, mask, j0, 3u);
                    while (bits) {
                        const int j = j0 + __builtin_ctz(bits);
                        bits &= bits - 1;
                        int64_t ko = (int64_t)j * a.k_rs, vo = (int64_t)j * a.v_rs;
                        if constexpr (PAGED) {
                            const int e = tbl[j >> a.page_shift];
                            if ((uint32_t)e >= (uint32_t)a.num_pages) continue;
                            const int in = j & ((1 << a.page_shift) - 1);
                            ko = (int64_t)e * a.k_ps + (int64_t)in * a.k_rs;
                            vo = (int64_t)e * a.v_ps + (int64_t)in * a.v_rs;
                        }
                        kv.template load<T>(kbase + ko, head_dim);
                        vv.template load<T>(vbase + vo, head_dim);
                        const float s = qv.dot(kv) * a.scale * LOG2E;
                        const float top = fmaxf(m, s);
                        const float w0 = m == -INFINITY ? 0.f : fast_exp2(m - top), w1 = fast_exp2(s - top);
                        l = l * w0 + w1;
#pragma unroll
                        for (int e = 0; e < LaneRow<D>::E; ++e) acc.x[e] = (m == -INFINITY ? 0.f : acc.x[e] * w0) + w1 * vv.x[e];
                        m = top;
                    }
                }
            }
            acc.put(o, rr);
            if (l32 == rr) {
                m_thr = mc = m;
                l_i = hi ? 0.f : l;
            }
        }
    }

    zero_tail(a.o, a.o_rs, a.o_hs, a.nheads, a.head_dim, a.total_q, a.cu_q, a.batch);
    float l_tot = pair_sum(l_i);
    float mrow = m_thr == -INFINITY ? -INFINITY : mc;         // m * c_log2, -inf: nothing seen

    // ---- join the key groups: groups 1.. leave (O, l, m) in LDS, group 0 sums in their order
    if constexpr (KG > 1) {
        __syncthreads();
        constexpr int NR = 16 * (D / 32);
        float *xo = (float *)smem;                                     // [kg - 1][row wave][NR / 4][lane][4]
        float *xm = xo + (KG - 1) * NWR * NR * 64;                     // [kg - 1][row wave][lane][2]
        if (kg > 0) {
            const int base = (kg - 1) * NWR + wr;
#pragma unroll
            for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
                for (int q4 = 0; q4 < 4; ++q4)
                    *reinterpret_cast<f32x4 *>(xo + ((base * (NR / 4) + 4 * dt + q4) * 64 + lane) * 4) =
                        f32x4{o[dt][4 * q4], o[dt][4 * q4 + 1], o[dt][4 * q4 + 2], o[dt][4 * q4 + 3]};
            xm[(base * 64 + lane) * 2] = l_tot;
            xm[(base * 64 + lane) * 2 + 1] = mrow;
        }
        __syncthreads();
        if (kg > 0) return;
        float top = mrow;
#pragma unroll
        for (int x = 0; x < KG - 1; ++x) top = fmaxf(top, xm[((x * NWR + wr) * 64 + lane) * 2 + 1]);
        const float w0 = mrow == -INFINITY ? 0.f : fast_exp2(mrow - top);
        l_tot *= w0;
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[dt][r] *= w0;
#pragma unroll
        for (int x = 0; x < KG - 1; ++x) {
            const int base = x * NWR + wr;
            const float mx = xm[(base * 64 + lane) * 2 + 1];
            const float wx = mx == -INFINITY ? 0.f : fast_exp2(mx - top);
            l_tot += wx * xm[(base * 64 + lane) * 2];
#pragma unroll
            for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
                for (int q4 = 0; q4 < 4; ++q4) {
                    const f32x4 v = *reinterpret_cast<const f32x4 *>(xo + ((base * (NR / 4) + 4 * dt + q4) * 64 + lane) * 4);
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[dt][4 * q4 + e] += wx * v[e];
                }
        }
        mrow = top;
    }
    if (KG > 1 || a.nsplit > 1) {
        if (row >= R) return;
    }
    if (a.nsplit > 1) {
        const int64_t wrow = ((int64_t)split * a.total_q + q_start + t) * a.nheads + kvh * G + g;
        float *op = a.ws_o + wrow * D;
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4)
                *reinterpret_cast<f32x4 *>(op + 32 * dt + 8 * q4 + 4 * hi) =
                    f32x4{o[dt][4 * q4], o[dt][4 * q4 + 1], o[dt][4 * q4 + 2], o[dt][4 * q4 + 3]};
        if (hi == 0) {
            a.ws_ml[wrow * 2] = mrow;
            a.ws_ml[wrow * 2 + 1] = l_tot;
        }
        return;
    }

    // ---- epilogue: O / l in 16 bits
    const bool empty = mrow == -INFINITY && l_tot == 0.f;
    const float inv = empty ? 0.f : 1.f / l_tot;
    if constexpr (KG == 1) {
        __syncthreads();
        store_rows<D, T>(o, inv, smem + wave * 64 * D, head_dim, [&](int r) __attribute__((always_inline)) -> uint16_t * {
            if (rw + r >= R) return nullptr;
            const int tt = a.dgroup.div(rw + r), gg = rw + r - tt * G;
            return a.o + (int64_t)(q_start + tt) * a.o_rs + (int64_t)(kvh * G + gg) * a.o_hs;
        });
        if (row >= R) return;
    } else {
        // lanes l and l + 32 hold the halves of each group of 8 columns; one exchange gives each a 16-byte store
        uint16_t *op = a.o + (int64_t)(q_start + t) * a.o_rs + (int64_t)(kvh * G + g) * a.o_hs;
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
            for (int g4 = 0; g4 < 4; g4 += 2) {
                const uint32_t a0 = T::pack2(o[dt][4 * g4 + 0] * inv, o[dt][4 * g4 + 1] * inv);
                const uint32_t a1 = T::pack2(o[dt][4 * g4 + 2] * inv, o[dt][4 * g4 + 3] * inv);
                const uint32_t b0 = T::pack2(o[dt][4 * g4 + 4] * inv, o[dt][4 * g4 + 5] * inv);
                const uint32_t b1 = T::pack2(o[dt][4 * g4 + 6] * inv, o[dt][4 * g4 + 7] * inv);
                const auto s0 = __builtin_amdgcn_permlane32_swap(a0, b0, false, false);
                const auto s1 = __builtin_amdgcn_permlane32_swap(a1, b1, false, false);
                const int d = 32 * dt + 8 * (g4 + hi);
                if (d < head_dim) gstore128(op + d, u32x4{s0[0], s1[0], s0[1], s1[1]});
            }
    }
    if (hi == 0 && a.lse)
        a.lse[(int64_t)(b * a.nheads + kvh * G + g) * a.lse_stride + t] = empty ? -INFINITY : mrow * LN2 + __logf(l_tot);
}

// Joins the splits of a row: O = sum_s w_s O_s / sum_s w_s l_s with w_s = 2^(m_s - max m), in a fixed order. One wave to
// a row: its lanes take the splits' m and l (two each, 128 splits at most), then the columns, eight splits' loads in
// flight. Bound by launch and two loads one after the other: 2.9 us for one token of 12 heads (5.9 with a loop of single
// loads, 8 splits); 10.7 us for 16384 rows of 128 in 4 splits.
template <int D, typename T>
__global__ __launch_bounds__(256) void fa_window_join_kernel(const WinFwdArgs a) {
    constexpr float LN2 = 0.6931471805599453f;
    int q_start, sq;
    const int b = blockIdx.y;
    seq_bounds(a.cu_q, b, a.total_q, q_start, sq);
    sq = sq < a.max_q ? sq : a.max_q;
    const int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (i >= (int64_t)sq * a.nheads) return;
    const int64_t row = (int64_t)q_start * a.nheads + i, rows = a.total_q * a.nheads;
    constexpr int E = D >= 64 ? D / 64 : 1;
    typedef float vec __attribute__((ext_vector_type(E)));
    float m[2], w[2], top = -INFINITY, l = 0.f;
    float ls[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        const int s = lane + 64 * x;
        m[x] = s < a.nsplit ? a.ws_ml[(s * rows + row) * 2] : -INFINITY;
        ls[x] = s < a.nsplit ? a.ws_ml[(s * rows + row) * 2 + 1] : 0.f;
        top = fmaxf(top, m[x]);
    }
#pragma unroll
    for (int s = 32; s >= 1; s >>= 1) top = fmaxf(top, __shfl_xor(top, s));
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        w[x] = m[x] == -INFINITY ? 0.f : fast_exp2(m[x] - top);
        l += m[x] == -INFINITY ? ls[x] * 0.f : w[x] * ls[x];       // (a NaN stays one)
    }
    l = wave_sum(l);
    const int e0 = D >= 64 || lane < D ? E * lane : 0;
    const float *op = a.ws_o + row * D + e0;
    vec acc = {};
    for (int s0 = 0; s0 < a.nsplit; s0 += 8) {
        vec v[8];
#pragma unroll
        for (int x = 0; x < 8; ++x)
            if (s0 + x < a.nsplit) v[x] = *(const vec *)(op + (s0 + x) * rows * D);
#pragma unroll
        for (int x = 0; x < 8; ++x)
            if (s0 + x < a.nsplit) acc += v[x] * __shfl(s0 < 64 ? w[0] : w[1], (s0 + x) & 63);
    }
    const bool empty = top == -INFINITY && l == 0.f;
    const float inv = empty ? 0.f : 1.f / l;
    const int t = (int)(i / a.nheads), h = (int)(i - (int64_t)t * a.nheads);
    uint16_t *out = a.o + (int64_t)(q_start + t) * a.o_rs + (int64_t)h * a.o_hs + e0;
    if (e0 < a.head_dim && (D >= 64 || lane < D)) {
        if constexpr (E == 2)
            *(uint32_t *)out = T::pack2(acc[0] * inv, acc[1] * inv);
        else
            *out = T::from_float(acc[0] * inv);
    }
    if (lane == 0 && a.lse)
        a.lse[(int64_t)(b * a.nheads + h) * a.lse_stride + t] = empty ? -INFINITY : top * LN2 + __logf(l);
}

}  // namespace fa
