// fa_window_bwd_kernel.h — backward of the windowed attention (dense var-len, grouped heads).
//
// With P = exp(scale Q K^T - lse) on the entries a row sees and 0 elsewhere, delta = rowsum(dO * O):
//     dP = dO V^T,  dS = P (dP - delta),  dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO,
// dK and dV summed over the query heads of a group. dQ is computed by query rows (the forward's walk), dK and dV by
// keys, each written once, in one order, with no atomics. S and dP are computed in both: 7 matrix products of the
// forward's size against 5 with dQ by fp32 atomics, whose order changes the result and whose rate bounds it
// (1.3 TB/s measured for the dense backward).
//
// Row constants: ws_rows[i] = {lse log2(e), -delta} of packed row i of a sequence and key/value head, rows of a
// head one after the other, so that a tile's 32 pairs are 256 contiguous bytes (one LDS-DMA of 4 bytes a lane).
// The dQ kernel leaves them for the dK, dV kernel. delta comes from O in 16 bits, whose rounding is lost among many
// keys but shows where a row sees few; there it is summed from P and dP in fp32 first (WIN_EXACT_TILES).
#pragma once

#include "fa_window_careful.h"

namespace fa {

typedef float f32x2 __attribute__((ext_vector_type(2)));

struct WinBwdArgs {
    const uint16_t *q, *k, *v, *o, *dout;
    const float *lse;
    uint16_t *dq, *dk, *dv;
    f32x2 *ws_rows;               // [total_q * nheads]
    float *ws_part;               // [batch * nheads_k][sinks][slots][2][D]: dK, dV of the sinks by parts
    const int32_t *cu_q, *cu_k;
    int64_t q_rs, q_hs, k_rs, k_hs, v_rs, v_hs, o_rs, o_hs, do_rs, do_hs;
    int64_t dq_rs, dq_hs, dk_rs, dk_hs, dv_rs, dv_hs;
    int64_t total_q, total_k;
    int batch, nheads, nheads_k, head_dim, group;
    int max_q, lse_stride, window, sinks;
    // the sinks' rows behind the window, cut into `chunks` shares (0: walked with the rest): blocks of 32 keys,
    // partial sums a share leaves (one for each wave or pair), `slots` of them in all and the window's own
    int chunks, sink_blocks, per_chunk, slots;
    float scale;
    Div dgroup, dheads, dchunks, dsinkb;      // by group, nheads_k, chunks, sink_blocks
    BlockOrder order;
};

// first packed row (of the whole tensor's row constants) of a sequence and key/value head
__device__ __forceinline__ int64_t rows_base(const WinBwdArgs &a, int q_start, int len_q, int kvh) {
    return (int64_t)q_start * a.nheads + (int64_t)kvh * len_q * a.group;
}

// ---------------------------------------------------------------------------------------------- dQ
template <int D, int NW>
struct WinDqCfg {
    static constexpr int NT = 64 * NW;
    static constexpr int BM = 32 * NW;
    static constexpr int BN = 64;
    static constexpr int NC = D / 8;
    static constexpr int TILE = BN * D * 2;
    static constexpr int PIECES = TILE / 1024;
    static constexpr int PPW = (PIECES + NW - 1) / NW;
    static constexpr int RPP = 1024 / (2 * D);
    static constexpr int LDS = 4 * TILE;               // K[2], V[2]
};

// A wave owns 32 packed query rows (lane = row): S^T = K Q^T and dP^T = V dO^T with Q and dO rows in registers,
// dS^T packed in place is the B operand of dQ^T += K^T dS^T (K^T by transposed LDS reads). lse and delta are per
// lane, so no exchange between rows at all.
//
// A workgroup of few tiles walks them twice, first for delta = sum_j P_j dP_j: with the 16-bit O's delta the error of
// dQ and dK (rms, 60 to 400 keys from the sequence's start) measured 1.5 to 1.65 times that of a 32-bit backward
// rounded once, with this one 1.4 to 1.45 (what the rounding of dS leaves). 2 of 5 products more on those tiles.
//
// Measured: 8192 tokens, 16 heads of 128 on 4, window 1024: 120 us (matrix units 48 % busy, two waves a SIMD that wait for
// LDS between products); 8 x 2048 tokens, 12 heads of 64, window 256: 54 us (26 %).
constexpr int WIN_EXACT_TILES = 4;
//
// FINE (small calls, takes_fine in fa_window_api.cpp): dS, and P for dV, go to their products in two 16-bit parts, as
// in the forward: what their rounding leaves (1.4 and more of a single rounding, where outputs are few) goes to 1.0.
template <int D, typename T, int NW, bool FINE>
__global__ __launch_bounds__(64 * NW, 2) void fa_window_dq_kernel(const WinBwdArgs a) {
    using C = WinDqCfg<D, NW>;
    using S = Swz<D>;
    constexpr float LOG2E = 1.4426950408889634f;
    extern __shared__ __attribute__((aligned(16))) char smem[];

    int rb, w;
    a.order.get(blockIdx.x, rb, w);
    const int b = a.dheads.div(w);
    const int kvh = w - b * a.nheads_k;
    int q_start, len_q, k_start, klen;
    seq_bounds(a.cu_q, b, a.total_q, q_start, len_q);
    seq_bounds(a.cu_k, b, a.total_k, k_start, klen);
    const int off = klen - len_q, sq = len_q < a.max_q ? len_q : a.max_q;     // lse's rows end at max_q
    const int G = a.group, R = sq * G, r0 = rb * C::BM;
    if (r0 >= R) {
        zero_tail(a.dq, a.dq_rs, a.dq_hs, a.nheads, a.head_dim, a.total_q, a.cu_q, a.batch);
        return;
    }

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l32 = lane & 31, hi = lane >> 5;
    const int head_dim = a.head_dim;
    const int rw = r0 + 32 * wave, row = rw + l32;
    const int rc = row < R ? row : R - 1;
    const int t = a.dgroup.div(rc), g = rc - t * G, h = kvh * G + g;
    const int pos = off + t;
    int pmin = off + a.dgroup.div(rw), pmax = off + a.dgroup.div(rw + 31 < R ? rw + 31 : R - 1);
    if (rw >= R) pmin = pmax = pos;
    int k_end = off + a.dgroup.div(r0 + C::BM < R ? r0 + C::BM - 1 : R - 1) + 1;
    k_end = k_end < klen ? k_end : klen;
    const TileWalk walk = tile_walk(off + a.dgroup.div(r0), k_end, a.window, a.sinks, C::BN);

    const uint16_t *kbase = a.k + (int64_t)k_start * a.k_rs + (int64_t)kvh * a.k_hs;
    const uint16_t *vbase = a.v + (int64_t)k_start * a.v_rs + (int64_t)kvh * a.v_hs;
    int k_off[C::PPW], v_off[C::PPW];
#pragma unroll
    for (int i = 0; i < C::PPW; ++i) {
        const int r = C::RPP * (wave + NW * i) + lane / C::NC;
        const int c = (lane % C::NC) ^ S::x(r);
        const bool ok = c * 8 < head_dim;
        k_off[i] = ok ? (r * (int)a.k_rs + c * 8) * 2 : OOB;
        v_off[i] = ok ? (r * (int)a.v_rs + c * 8) * 2 : OOB;
    }
    auto stage = [&](int i, int buf) __attribute__((always_inline)) {
        const int j0 = walk.tile(i) * C::BN;
        int rows = klen - j0;
        rows = rows < 0 ? 0 : (rows > C::BN ? C::BN : rows);
        const i32x4 ks = make_srd(kbase + (int64_t)j0 * a.k_rs, rows * (int)a.k_rs * 2);
        const i32x4 vs = make_srd(vbase + (int64_t)j0 * a.v_rs, rows * (int)a.v_rs * 2);
#pragma unroll
        for (int n = 0; n < C::PPW; ++n) {
            const int p = wave + NW * n;
            if (C::PIECES % NW == 0 || p < C::PIECES) {
                dma16(ks, k_off[n], 0, lds_addr(smem + buf * C::TILE + 1024 * p));
                dma16(vs, v_off[n], 0, lds_addr(smem + (2 + buf) * C::TILE + 1024 * p));
            }
        }
    };

    // the first tile is on its way before the rows are read
    if (walk.n > 0) stage(0, 0);
    typename T::frag qf[D / 16], df[D / 16];
    float delta = 0.f;
    {
        const uint16_t *qp = a.q + (int64_t)(q_start + t) * a.q_rs + (int64_t)h * a.q_hs;
        const uint16_t *dp = a.dout + (int64_t)(q_start + t) * a.do_rs + (int64_t)h * a.do_hs;
        const uint16_t *op = a.o + (int64_t)(q_start + t) * a.o_rs + (int64_t)h * a.o_hs;
        u32x4 x[D / 16], y[D / 16], z[D / 16];
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
            const int c = 2 * ks + hi;
            x[ks] = y[ks] = z[ks] = u32x4{0u, 0u, 0u, 0u};
            if (c * 8 < head_dim) {
                x[ks] = gload128(qp + c * 8);
                y[ks] = gload128(dp + c * 8);
                z[ks] = gload128(op + c * 8);
            }
        }
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
            qf[ks] = as_frag<T>(x[ks]);
            df[ks] = as_frag<T>(y[ks]);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                delta += T::lo_float(y[ks][e]) * T::lo_float(z[ks][e]) + T::hi_float(y[ks][e]) * T::hi_float(z[ks][e]);
        }
        delta = pair_sum(delta);
    }
    const float lse2 = a.lse[(int64_t)(b * a.nheads + h) * a.lse_stride + t] * LOG2E;
    const float c_log2 = a.scale * LOG2E;

    const int grp = (lane >> 4) & 1, qq = (lane & 15) >> 2, pp = lane & 3;
    int k_rd[D / 16];                 // rows 32 further on are an immediate offset (the swizzle goes by row % 16)
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) k_rd[ks] = S::off(l32, 2 * ks + hi);
    int t_rd[D / 32][2];
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt) {
        const int r = 4 * hi + qq, col = 32 * dt + 16 * grp + 4 * pp;
        t_rd[dt][0] = S::off8(r, col);
        t_rd[dt][1] = S::off8(r + 8, col);
    }

    f32x16 dq[D / 32];
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) dq[dt][r] = 0.f;

    // one tile, 32 keys at a time; SUM: delta's terms alone
    float dsum = 0.f;
    auto compute = [&](auto sum_tag, int j0, int buf) __attribute__((always_inline)) {
        constexpr bool SUM = decltype(sum_tag)::value;
        const char *kb = smem + buf * C::TILE, *vb = smem + (2 + buf) * C::TILE;
        const bool whole = j0 + C::BN - 1 <= pmin && (j0 > pmax - a.window || j0 + C::BN <= a.sinks) && j0 + C::BN <= klen;
        const bool masked = !__builtin_amdgcn_readfirstlane((int)whole);
#pragma unroll
        for (int st = 0; st < 2; ++st) {
            const int ro = 32 * st * S::ROW_BYTES;
            f32x16 s, dp;
#pragma unroll
            for (int r = 0; r < 16; ++r) { s[r] = 0.f; dp[r] = SUM ? 0.f : -delta; }
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks) {
                s = T::mfma32(as_frag<T>(lds_read128(kb, k_rd[ks] + ro)), qf[ks], s);
                dp = T::mfma32(as_frag<T>(lds_read128(vb, k_rd[ks] + ro)), df[ks], dp);
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = fast_exp2(fmaf(s[r], c_log2, -lse2)) * dp[r];
            // by selection, so that an infinity in a masked place (the lse of a row that sees nothing) adds 0
            if (masked) {
                const int j = j0 + 32 * st;
                const uint32_t m = (seen_bits(j, pos, a.window, a.sinks) & bits_below(klen - j)) >> (4 * hi);
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = m & (1u << crow(r, 0)) ? s[r] : 0.f;
            }
            if constexpr (SUM) {
#pragma unroll
                for (int r = 0; r < 16; ++r) dsum += s[r];
                continue;
            }
            typename T::frag pf[2], pl[2];
#pragma unroll
            for (int s2 = 0; s2 < 2; ++s2) {
                u32x4 pk;
#pragma unroll
                for (int e = 0; e < 4; ++e) pk[e] = T::pack2(s[8 * s2 + 2 * e], s[8 * s2 + 2 * e + 1]);
                pf[s2] = as_frag<T>(pk);
                if constexpr (FINE) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        pk[e] = T::pack2(s[8 * s2 + 2 * e] - T::lo_float(pk[e]), s[8 * s2 + 2 * e + 1] - T::hi_float(pk[e]));
                    pl[s2] = as_frag<T>(pk);
                }
            }
#pragma unroll
            for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
                for (int dt = 0; dt < D / 32; ++dt) {
                    const int to = ro + 16 * s2 * S::ROW_BYTES;
                    const u32x2 lo = lds_read_tr(kb, t_rd[dt][0] + to);
                    const u32x2 hv = lds_read_tr(kb, t_rd[dt][1] + to);
                    const auto kt = as_frag<T>(u32x4{lo[0], lo[1], hv[0], hv[1]});
                    dq[dt] = T::mfma32(kt, pf[s2], dq[dt]);
                    if constexpr (FINE) dq[dt] = T::mfma32(kt, pl[s2], dq[dt]);
                }
        }
    };
    auto step = [&](auto sum_tag, auto par, int i) __attribute__((always_inline)) {
        constexpr int P = decltype(par)::value;
        if (i + 1 < walk.n) stage(i + 1, 1 - P);
        const int j0 = walk.tile(i) * C::BN;
        if (rw < R && j0 <= pmax && (j0 + C::BN - 1 > pmin - a.window || j0 < a.sinks)) compute(sum_tag, j0, P);
        vmcnt0();
        __syncthreads();
    };
    auto walk_all = [&](auto sum_tag) __attribute__((always_inline)) {
        vmcnt0();       // (the compiler's counters see it: the loop inherits no pending prologue load)
        __syncthreads();
        for (int i = 0; i < walk.n; i += 2) {
            step(sum_tag, std::integral_constant<int, 0>(), i);
            if (i + 1 < walk.n) step(sum_tag, std::integral_constant<int, 1>(), i + 1);
        }
    };
    if (walk.n <= WIN_EXACT_TILES) {
        walk_all(std::true_type{});
        delta = pair_sum(dsum);
        if (walk.n > 0) stage(0, 0);
    }
    if (hi == 0 && row < R) a.ws_rows[rows_base(a, q_start, len_q, kvh) + row] = f32x2{lse2, -delta};
    walk_all(std::false_type{});

    // an infinity or NaN: this wave's rows again, key by key (fa_window_careful.h)
    if (!all_finite(dq, 0.f)) {
        LaneRow<D> qv, dv, kv, vv, acc;
        for (int rr = 0; rr < 32 && rw + rr < R; ++rr) {
            const int tt = a.dgroup.div(rw + rr), hh = kvh * G + rw + rr - tt * G, p = off + tt;
            qv.template load<T>(a.q + (int64_t)(q_start + tt) * a.q_rs + (int64_t)hh * a.q_hs, head_dim);
            dv.template load<T>(a.dout + (int64_t)(q_start + tt) * a.do_rs + (int64_t)hh * a.do_hs, head_dim);
            const float l2 = __shfl(lse2, rr), del = __shfl(delta, rr);
            acc.zero();
            for (int n = 0; n < walk.n; ++n)
                for (int j0 = walk.tile(n) * C::BN, st = 0; st < 2; ++st, j0 += 32) {
                    uint32_t bits = seen_bits(j0, p, a.window, a.sinks) & bits_below(klen - j0);
                    while (bits) {
                        const int j = j0 + __builtin_ctz(bits);
                        bits &= bits - 1;
                        kv.template load<T>(kbase + (int64_t)j * a.k_rs, head_dim);
                        vv.template load<T>(vbase + (int64_t)j * a.v_rs, head_dim);
                        acc.add(fast_exp2(fmaf(qv.dot(kv), c_log2, -l2)) * (dv.dot(vv) - del), kv);
                    }
                }
            acc.put(dq, rr);
        }
    }
    zero_tail(a.dq, a.dq_rs, a.dq_hs, a.nheads, a.head_dim, a.total_q, a.cu_q, a.batch);
    store_rows<D, T>(dq, a.scale, smem + wave * 64 * D, head_dim, [&](int r) __attribute__((always_inline)) -> uint16_t * {
        if (rw + r >= R) return nullptr;
        const int tt = a.dgroup.div(rw + r), gg = rw + r - tt * G;
        return a.dq + (int64_t)(q_start + tt) * a.dq_rs + (int64_t)(kvh * G + gg) * a.dq_hs;
    });
}

// ------------------------------------------------------------------------------------------- dK, dV
// PAIR: two waves to a block of 32 keys (one computes S, P and dV, the other dP, dS and dK), else one.
template <int D, int NW, bool PAIR>
struct WinDkvCfg {
    static constexpr int NT = 64 * NW;
    static constexpr int NB = PAIR ? NW / 2 : NW;      // blocks of 32 keys
    static constexpr int BK = 32 * NB;                 // keys per workgroup
    static constexpr int BR = 32;                      // packed query rows per step
    static constexpr int NC = D / 8;
    static constexpr int TILE = BR * D * 2;
    static constexpr int PIECES = TILE / 1024;
    static constexpr int PPW = (PIECES + NW - 1) / NW;
    static constexpr int RPP = 1024 / (2 * D);
    static constexpr int STAGE = 2 * TILE + 256;       // Q, dO, row constants
    static constexpr int RING = PAIR ? 5 : 4;
    static constexpr int AHEAD = PAIR ? 2 : 3;         // stages in flight
    static constexpr int DMAS = 2 * PPW + 1;           // a wave's loads per stage
    static constexpr int OFF_P = RING * STAGE;         // PAIR: P of a step in fp32, two buffers for each pair
    static constexpr int LDS = OFF_P + (PAIR ? 2 * NB * 4096 : 0);
};

// 64 lanes x 4 bytes to LDS, as dma16
__device__ __forceinline__ void dma4(i32x4 srd, int voff, uint32_t lds) {
#if defined(__HIP_DEVICE_COMPILE__)
    uint32_t keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\t"
                 "buffer_load_dword %1, %2, 0 offen lds\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep)
                 : "v"(voff), "s"(srd), "s"(__builtin_amdgcn_readfirstlane(lds))
                 : "memory");
#endif
}

// A block of 32 keys (lane = key) keeps its K, V rows and dK^T, dV^T in registers and walks the packed query rows that
// see the workgroup's keys, all heads of the group: S = Q K^T, dP = dO V^T with Q and dO rows from LDS; P and dS in
// registers are the B operands of dV^T += dO^T P and dK^T += Q^T dS (transposed LDS reads).
//
// Tiles of 32 rows come by LDS-DMA into a ring of four stages, three ahead of the compute, so that a step (16 or 32
// matrix instructions a wave) does not wait for memory; one barrier a step.
//
// D = 128 needs 128 registers for dK^T and dV^T alone: there a pair of waves shares the block, each with one of the two
// accumulators. The P wave leaves P in LDS (fp32: dS takes P unrounded); the dS wave works one step behind it. Each
// starts a tile's first product a step before it uses it, so a stage is read in three steps, of a ring of five.
//
// A sink is seen by every later row, so its block would walk the whole sequence: its rows behind the window are cut
// into chunks of their own workgroups, in which every block of the workgroup holds the same 32 keys and takes every
// NB-th tile. Their sums, and the window's for the same keys, go to the workspace and are added in a fixed order
// by fa_window_sink_sum_kernel.
//
// Measured: 8192 tokens, 16 heads of 128 on 4, window 1024, 16 sinks: 210 us (matrix units 36 % busy, LDS 30 %: a step is a
// chain of two products, the exponentials between them and a barrier); 8 x 2048 tokens, 12 heads of 64, window 256: 69 us.
template <int D, typename T, int NW, bool PAIR, bool FINE>
__global__ __launch_bounds__(64 * NW, D <= 64 && !FINE ? 3 : 2) void fa_window_dkv_kernel(const WinBwdArgs a) {
    using C = WinDkvCfg<D, NW, PAIR>;
    using S = Swz<D>;
    constexpr float LOG2E = 1.4426950408889634f;
    extern __shared__ __attribute__((aligned(16))) char smem[];

    auto tails = [&]() __attribute__((always_inline)) {
        zero_tail(a.dk, a.dk_rs, a.dk_hs, a.nheads_k, a.head_dim, a.total_k, a.cu_k, a.batch);
        zero_tail(a.dv, a.dv_rs, a.dv_hs, a.nheads_k, a.head_dim, a.total_k, a.cu_k, a.batch);
    };
    // the sinks' short workgroups first, then the blocks of keys in an order by XCD
    const int nsink = a.chunks * a.sink_blocks * a.nheads_k * a.batch;
    const bool sink = (int)blockIdx.x < nsink;
    int kb, chunk = 0, w;
    if (sink) {
        const int x = a.dchunks.div(blockIdx.x);
        chunk = blockIdx.x - x * a.chunks;
        w = a.dsinkb.div(x);
        kb = x - w * a.sink_blocks;
    } else {
        // early keys are seen by the most rows
        a.order.get(blockIdx.x - nsink, kb, w);
        kb = a.order.nblk - 1 - kb;
    }
    const int b = a.dheads.div(w);
    const int kvh = w - b * a.nheads_k;
    int q_start, len_q, k_start, klen;
    seq_bounds(a.cu_q, b, a.total_q, q_start, len_q);
    seq_bounds(a.cu_k, b, a.total_k, k_start, klen);
    const int off = klen - len_q, sq = len_q < a.max_q ? len_q : a.max_q;     // lse's rows end at max_q
    const int G = a.group, k0 = kb * (sink ? 32 : C::BK);
    if (k0 >= klen) {              // (a sink that is not there leaves no sums: its dK, dV have no row)
        tails();
        return;
    }

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l32 = lane & 31, hi = lane >> 5;
    const int head_dim = a.head_dim;
    // block of 32 keys; a pair's waves are NB = 4 apart, on one SIMD: one's matrix work beside the other's exponentials
    const int blk = wave % C::NB;
    const bool dswave = PAIR && wave >= C::NB;         // the pair's second wave
    const int kw = k0 + (sink ? 0 : 32 * blk), key = kw + l32;

    // packed rows [r_beg, r_end): key j is seen from row (j - off) G on, up to row (j - off + window) G, a sink by
    // every row from there on
    int r_beg, r_end;
    const bool split = a.chunks > 0;
    if (sink) {
        const int64_t t64 = (int64_t)k0 - off + a.window;
        const int64_t r64 = t64 > 0 ? t64 * G : 0;
        const int lo = r64 < (int64_t)sq * G ? (int)r64 : sq * G;
        const int64_t beg = lo + (int64_t)chunk * a.per_chunk;
        r_beg = beg < (int64_t)sq * G ? (int)beg : sq * G;
        r_end = r_beg + a.per_chunk < sq * G ? r_beg + a.per_chunk : sq * G;
    } else {
        const int t_beg = k0 - off > 0 ? k0 - off : 0;
        const int64_t t64 = k0 < a.sinks && !split ? sq : (int64_t)k0 + C::BK - 1 + a.window - off;
        r_beg = t_beg * G;
        r_end = (t64 < 0 ? 0 : (t64 < sq ? (int)t64 : sq)) * G;
    }
    const int nt = r_end > r_beg ? (r_end - r_beg + C::BR - 1) / C::BR : 0;
    // The blocks of a head that run at once see mostly the same rows. Each starts its walk at a tile whose number is a
    // multiple of the walk's length and goes round, so that they read a tile at the same time, from the L2, instead
    // of one block's rows a block later, when it has left it.
    const int rot = sink || nt == 0 ? 0 : (nt - r_beg / C::BR % nt) % nt;
    auto row_of = [&](int n) __attribute__((always_inline)) -> int {      // first row of the n-th tile walked
        int u = n + rot;
        u -= u >= nt ? nt : 0;
        return r_beg + u * C::BR;
    };
    // this lane's rows [lo, up) relative to a tile's first: lane constants, the tile's row is taken off in the loop
    const int key_lo = (key - off) * G;                                        // first row that sees the key
    const int64_t key_w = ((int64_t)key - off + a.window) * G;                 // first row behind its window
    const int key_up = key_w < r_end && !(key < a.sinks && !split) ? (int)key_w : r_end;
    const int lane_beg = sink ? (key_w > r_end ? r_end : (int)key_w) : key_lo;
    const int lane_end = key >= klen || (sink && key >= a.sinks) ? lane_beg : (sink ? r_end : key_up);   // (none: empty)

    // ---- staging of tile n: row r is token r / G of head kvh G + r % G; rows behind the last land as zeros
    const uint16_t *qbase = a.q + (int64_t)q_start * a.q_rs + (int64_t)kvh * G * a.q_hs;
    const uint16_t *dbase = a.dout + (int64_t)q_start * a.do_rs + (int64_t)kvh * G * a.do_hs;
    const f32x2 *rows_g = a.ws_rows + rows_base(a, q_start, len_q, kvh);
    int q_off[C::PPW], do_off[C::PPW];                 // from the tile's first token
    auto lane_offsets = [&](int rt, int t0, int rows) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < C::PPW; ++i) {
            const int p = (wave + NW * i) % C::PIECES;     // fewer pieces than waves: some are staged twice, alike
            const int r = C::RPP * p + lane / C::NC, c = (lane % C::NC) ^ S::x(r);
            const int t = a.dgroup.div(rt + r), g = rt + r - t * G;
            const bool ok = r < rows && c * 8 < head_dim;
            q_off[i] = ok ? ((t - t0) * (int)a.q_rs + g * (int)a.q_hs + c * 8) * 2 : OOB;
            do_off[i] = ok ? ((t - t0) * (int)a.do_rs + g * (int)a.do_hs + c * 8) * 2 : OOB;
        }
    };
    // groups that divide 32 (r_beg and r_end are then whole tokens): a tile's lanes stand alike from its first token,
    // and rows behind the last are cut off by the descriptor
    const bool even = 32 % G == 0;
    if (even) lane_offsets(0, 0, C::BR);
    int st_buf = 0;                                    // the stage that is filled next
    auto next_buf = [&](int o) __attribute__((always_inline)) -> int {
        o += C::STAGE;
        return o == C::RING * C::STAGE ? 0 : o;
    };
    auto stage = [&](int n) __attribute__((always_inline)) {
        char *buf = smem + st_buf;
        st_buf = next_buf(st_buf);
        const int rt = row_of(n);
        const int t0 = a.dgroup.div(rt);               // the descriptors start at the tile's first token
        const int left = r_end - rt < C::BR ? r_end - rt : C::BR;
        int tokens = C::BR + 1;                        // (more than a tile's, within 32 bits: check_rows)
        if (even)
            tokens = a.dgroup.div(left);
        else
            lane_offsets(rt, t0, left);
        const i32x4 qs = make_srd(qbase + (int64_t)t0 * a.q_rs, tokens * (int)a.q_rs * 2);
        const i32x4 ds = make_srd(dbase + (int64_t)t0 * a.do_rs, tokens * (int)a.do_rs * 2);
#pragma unroll
        for (int i = 0; i < C::PPW; ++i) {
            const int p = (wave + NW * i) % C::PIECES;
            dma16(qs, q_off[i], 0, lds_addr(buf + 1024 * p));
            dma16(ds, do_off[i], 0, lds_addr(buf + C::TILE + 1024 * p));
        }
        // (every wave, the same 256 bytes: a stage is then the same number of loads for each)
        dma4(make_srd(rows_g + rt, left * 8), l32 * 8 + hi * 4, lds_addr(buf + 2 * C::TILE));
    };

    constexpr int AHEAD = C::AHEAD;
#pragma unroll
    for (int n = 0; n < AHEAD; ++n)
        if (n < nt) stage(n);

    typename T::frag kf[D / 16], vf[PAIR ? 1 : D / 16];   // PAIR: the wave's own operand, K or V, in kf
    {
        const int kc = key < klen ? key : klen - 1;
        const uint16_t *kp = a.k + (int64_t)(k_start + kc) * a.k_rs + (int64_t)kvh * a.k_hs;
        const uint16_t *vp = a.v + (int64_t)(k_start + kc) * a.v_rs + (int64_t)kvh * a.v_hs;
        if (dswave) kp = vp;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
            const int c = 2 * ks + hi;
            u32x4 x = {0u, 0u, 0u, 0u}, y = {0u, 0u, 0u, 0u};
            if (c * 8 < head_dim) {
                x = gload128(kp + c * 8);
                if constexpr (!PAIR) y = gload128(vp + c * 8);
            }
            kf[ks] = as_frag<T>(x);
            if constexpr (!PAIR) vf[ks] = as_frag<T>(y);
        }
    }
    f32x16 dk[D / 32], dv[PAIR ? 1 : D / 32];             // PAIR: the wave's own accumulator, dV or dK, in dk
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            dk[dt][r] = 0.f;
            if constexpr (!PAIR) dv[dt][r] = 0.f;
        }
    const float c_log2 = a.scale * LOG2E;

    const int grp = (lane >> 4) & 1, qq = (lane & 15) >> 2, pp = lane & 3;
    // The swizzles exclusive-or a chunk's number with bits of its row: k-step ks of a row read is the lane's address ^
    // 32 ks, column block dt of a transposed read ^ 64 dt, eight rows further on ^ 32 (images start at whole rows). One
    // register each instead of one for each read.
    static_assert(C::STAGE % S::ROW_BYTES == 0 && C::TILE % S::ROW_BYTES == 0, "images at whole rows");
    const int r_rd = S::off(l32, hi), t_rd = S::off8(4 * hi + qq, 16 * grp + 4 * pp);
    // X^T += A^T B over the tile's 32 rows: A rows in LDS (transposed reads), B packed in registers
    auto add_t = [&](f32x16 (&x)[D / 32], int rows, const u32x4 (&bv)[2]) __attribute__((always_inline)) {
        const int at = rows + t_rd;
        auto get = [&](int sg, int dt) __attribute__((always_inline)) -> u32x4 {
            const int ro = 16 * sg * S::ROW_BYTES;
            const u32x2 a0 = lds_read_tr(smem, (at ^ (dt << 6)) + ro);
            const u32x2 a1 = lds_read_tr(smem, (at ^ (dt << 6) ^ 32) + ro + 8 * S::ROW_BYTES);
            return u32x4{a0[0], a0[1], a1[0], a1[1]};
        };
        // A pair's waves have the registers to read ahead: half of the operands before the first product, the rest
        // beside it; single waves do not (75 us for 70).
        u32x4 ahead[PAIR ? D / 32 : 1];
        if constexpr (PAIR) {
#pragma unroll
            for (int dt = 0; dt < D / 32; ++dt) ahead[dt] = get(0, dt);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int sg = 0; sg < 2; ++sg) {
#pragma unroll
            for (int dt = 0; dt < D / 32; ++dt) {
                const u32x4 v = PAIR ? ahead[PAIR ? dt : 0] : get(sg, dt);
                if constexpr (PAIR)
                    if (sg == 0) ahead[dt] = get(1, dt);
                x[dt] = T::mfma32(as_frag<T>(v), as_frag<T>(bv[sg]), x[dt]);
            }
            if constexpr (PAIR)
                if (sg == 0) __builtin_amdgcn_sched_barrier(0);
        }
    };
    auto pack = [&](const f32x16 &x, u32x4 (&out)[2]) __attribute__((always_inline)) {
#pragma unroll
        for (int sg = 0; sg < 2; ++sg)
#pragma unroll
            for (int e = 0; e < 4; ++e) out[sg][e] = T::pack2(x[8 * sg + 2 * e], x[8 * sg + 2 * e + 1]);
    };
    // acc^T += rows^T b, b packed already; FINE: and what the packing left of it
    auto add_product = [&](f32x16 (&acc)[D / 32], int rows, const f32x16 &b, const u32x4 (&bv)[2]) __attribute__((always_inline)) {
        add_t(acc, rows, bv);
        if constexpr (FINE) {
            u32x4 rest[2];
#pragma unroll
            for (int sg = 0; sg < 2; ++sg)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    rest[sg][e] = T::pack2(b[8 * sg + 2 * e] - T::lo_float(bv[sg][e]), b[8 * sg + 2 * e + 1] - T::hi_float(bv[sg][e]));
            add_t(acc, rows, rest);
        }
    };
    // the tile's rows as A operands, all on their way before the first is used
    auto read_rows = [&](int rows, u32x4 (&x)[D / 16]) __attribute__((always_inline)) {
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) x[ks] = lds_read128(smem, (rows + r_rd) ^ (ks << 5));
        __builtin_amdgcn_sched_barrier(0);
    };
    // P of tile n: 0 (by selection: an infinity may stand there) in the rows that do not see this lane's key. Most
    // tiles are seen whole; the empty asm keeps the branch a branch.
    auto mask_p = [&](int n, f32x16 &p) __attribute__((always_inline)) {
        const int rt = row_of(n);
        uint32_t m = bits_below(lane_end - rt) & ~bits_below(lane_beg - rt);
        if (__builtin_amdgcn_ballot_w64(m != 0xFFFFFFFFu) == 0) return;
        asm volatile("");
        m >>= 4 * hi;
#pragma unroll
        for (int r = 0; r < 16; ++r) p[r] = m & (1u << crow(r, 0)) ? p[r] : 0.f;
    };
    // does the block take tile n?
    const int w_lo = (kw - off) * G;
    const int64_t w_up = kw < a.sinks && !split ? (int64_t)r_end : ((int64_t)kw + 31 - off + a.window) * G;
    auto takes = [&](int n) __attribute__((always_inline)) -> bool {
        const int rt = row_of(n);
        return sink ? n % C::NB == blk : (kw < klen && rt + C::BR > w_lo && rt < w_up);
    };
    // lse2 (WHICH 0) or -delta (1) of registers 4 q4 .. 4 q4 + 3, rows 8 q4 + 4 hi + e: they lie in LDS one after the
    // other, not in pairs, so that a read brings nothing that is not used (69 us for 76, 12 heads of 64)
    auto row_const = [&](int which, int buf, int q4) __attribute__((always_inline)) -> f32x4 {
        return *reinterpret_cast<const f32x4 *>(smem + buf + 2 * C::TILE + (32 * which + 8 * q4 + 4 * hi) * 4);
    };
    auto compute_one = [&](int n, int buf) __attribute__((always_inline)) {
        f32x16 s, dp;
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
            const f32x4 d = row_const(1, buf, q4);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                s[4 * q4 + e] = 0.f;
                dp[4 * q4 + e] = d[e];                 // dP starts at -delta
            }
        }
        // (operands read two k-steps at a time: all at once, as in a pair, took 81 us for 72, the registers short)
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
            s = T::mfma32(as_frag<T>(lds_read128(smem, (buf + r_rd) ^ (ks << 5))), kf[ks], s);
            dp = T::mfma32(as_frag<T>(lds_read128(smem, (buf + C::TILE + r_rd) ^ (ks << 5))), vf[PAIR ? 0 : ks], dp);
            if (ks % 2 == 1) __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
            const f32x4 l = row_const(0, buf, q4);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[4 * q4 + e] = fast_exp2(fmaf(s[4 * q4 + e], c_log2, -l[e]));
        }
        mask_p(n, s);
#pragma unroll
        for (int r = 0; r < 16; ++r) dp[r] *= s[r];
        u32x4 pk[2], sk[2];
        pack(s, pk);
        pack(dp, sk);
        if constexpr (!PAIR) {
            add_product(dv, buf + C::TILE, s, pk);
            add_product(dk, buf, dp, sk);
        }
    };
    // PAIR: S of a tile (P wave) or dP (dS wave), started one step before the rest of its work, so that the matrix
    // instructions of one tile run under the exponentials, LDS traffic and packing of the one before
    auto first_p = [&](int buf, f32x16 &s) __attribute__((always_inline)) {
        u32x4 x[D / 16];
        read_rows(buf, x);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) s = T::mfma32(as_frag<T>(x[ks]), kf[ks], s);
    };
    auto rest_p = [&](int n, int buf, f32x16 s) __attribute__((always_inline)) {
        char *img = smem + C::OFF_P + (2 * blk + (n & 1)) * 4096;
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
            const f32x4 l = row_const(0, buf, q4);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[4 * q4 + e] = fast_exp2(fmaf(s[4 * q4 + e], c_log2, -l[e]));
        }
        mask_p(n, s);
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4)
            *reinterpret_cast<f32x4 *>(img + (q4 * 64 + lane) * 16) = f32x4{s[4 * q4], s[4 * q4 + 1], s[4 * q4 + 2], s[4 * q4 + 3]};
        u32x4 pk[2];
        pack(s, pk);
        add_product(dk, buf + C::TILE, s, pk);         // dV^T
    };
    auto first_ds = [&](int buf, f32x16 &dp) __attribute__((always_inline)) {
        u32x4 y[D / 16];
        read_rows(buf + C::TILE, y);
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
            const f32x4 d = row_const(1, buf, q4);
#pragma unroll
            for (int e = 0; e < 4; ++e) dp[4 * q4 + e] = d[e];
        }
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) dp = T::mfma32(as_frag<T>(y[ks]), kf[ks], dp);
    };
    auto rest_ds = [&](int n, int buf, f32x16 dp) __attribute__((always_inline)) {
        const char *img = smem + C::OFF_P + (2 * blk + (n & 1)) * 4096;
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
            const f32x4 p = *reinterpret_cast<const f32x4 *>(img + (q4 * 64 + lane) * 16);
#pragma unroll
            for (int e = 0; e < 4; ++e) dp[4 * q4 + e] *= p[e];
        }
        u32x4 sk[2];
        pack(dp, sk);
        add_product(dk, buf, dp, sk);                  // dK^T
    };

    // ---- the walk
    vmcnt0();
    auto arrive = [&](int n) __attribute__((always_inline)) {
        // tile n has landed when at most the later stages' loads are out
        if (n + AHEAD - 1 < nt)
            vmcnt_n<C::DMAS *(AHEAD - 1)>();
        else if (AHEAD == 3 && n + 1 < nt)
            vmcnt_n<C::DMAS>();
        else
            vmcnt0();
        __syncthreads();
        if (n + AHEAD < nt) stage(n + AHEAD);
    };
    if constexpr (!PAIR) {
        int buf = 0;
        for (int n = 0; n < nt; ++n) {
            arrive(n);
            if (takes(n)) compute_one(n, buf);
            buf = next_buf(buf);
        }
    } else {
        // Step k of nt + 2: the P wave starts tile k and ends tile k - 1, the dS wave starts k - 1 and ends k - 2, whose
        // P the other left a step before. A loop for each (one loop with a branch moved the accumulators), with the
        // same barriers.
        auto walk = [&](auto lag_tag, auto &&first, auto &&rest) __attribute__((always_inline)) {
            constexpr int LAG = decltype(lag_tag)::value;
            f32x16 cur, next;
            for (int k = 0; k <= LAG; ++k) arrive(k);
            if (!sink) {
                // a tile that a block does not see goes through with P = 0: the barriers set the pace, and without
                // a branch the accumulators stay where they are
                first(0, cur);
                int buf = 0;
                for (int n = 1; n < nt; ++n) {
                    arrive(n + LAG);
                    const int at = next_buf(buf);
                    first(at, next);
                    rest(n - 1, buf, cur);
                    cur = next;
                    buf = at;
                }
                arrive(nt + LAG);
                rest(nt - 1, buf, cur);
            } else {
                int buf = 0;
                for (int n = 0; n < nt; ++n) {
                    if (takes(n)) first(buf, cur);
                    arrive(n + 1 + LAG);
                    if (takes(n)) rest(n, buf, cur);
                    buf = next_buf(buf);
                }
            }
            for (int k = nt + 1 + LAG; k < nt + 2; ++k) arrive(k);
        };
        if (nt > 0) {
            if (!dswave)
                walk(std::integral_constant<int, 0>(), first_p, rest_p);
            else
                walk(std::integral_constant<int, 1>(), first_ds, rest_ds);
        }
    }

    // an infinity or NaN: the wave's sums again, row by row (fa_window_careful.h). A sink's chunk takes the tiles that
    // its waves took.
    bool finite = all_finite(dk, 0.f);
    if constexpr (!PAIR) finite = finite && all_finite(dv, 0.f);
    if (!finite) {
        LaneRow<D> kv, vv, qv, dv_, gk, gv;
        for (int rr = 0; rr < 32 && kw + rr < klen; ++rr) {
            kv.template load<T>(a.k + (int64_t)(k_start + kw + rr) * a.k_rs + (int64_t)kvh * a.k_hs, head_dim);
            vv.template load<T>(a.v + (int64_t)(k_start + kw + rr) * a.v_rs + (int64_t)kvh * a.v_hs, head_dim);
            const int beg = __shfl(lane_beg, rr), end = __shfl(lane_end, rr);
            gk.zero();
            gv.zero();
            for (int n = 0; n < nt; ++n) {
                if (!takes(n)) continue;
                const int rt = row_of(n);
                for (int r = rt > beg ? rt : beg; r < end && r < rt + C::BR; ++r) {
                    const int tt = a.dgroup.div(r), hh = kvh * G + r - tt * G;
                    qv.template load<T>(a.q + (int64_t)(q_start + tt) * a.q_rs + (int64_t)hh * a.q_hs, head_dim);
                    dv_.template load<T>(a.dout + (int64_t)(q_start + tt) * a.do_rs + (int64_t)hh * a.do_hs, head_dim);
                    const f32x2 x = rows_g[r];
                    const float p = fast_exp2(fmaf(qv.dot(kv), c_log2, -x[0]));
                    gv.add(p, dv_);
                    gk.add(p * (dv_.dot(vv) + x[1]), qv);
                }
            }
            if constexpr (PAIR) {
                (dswave ? gk : gv).put(dk, rr);
            } else {
                gk.put(dk, rr);
                gv.put(dv, rr);
            }
        }
    }
    tails();
    __syncthreads();       // the ring is free: rows go out through it
    auto store = [&](const f32x16 (&x)[D / 32], bool is_v) __attribute__((always_inline)) {
        if (split && key < a.sinks && key < klen) {
            const int slot = sink ? chunk * C::NB + blk : a.slots - 1;
            float *pp_ = a.ws_part + ((((int64_t)(b * a.nheads_k + kvh) * a.sinks + key) * a.slots + slot) * 2 + (is_v ? 1 : 0)) * D;
#pragma unroll
            for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
                for (int q4 = 0; q4 < 4; ++q4)
                    *reinterpret_cast<f32x4 *>(pp_ + 32 * dt + 8 * q4 + 4 * hi) = f32x4{x[dt][4 * q4], x[dt][4 * q4 + 1], x[dt][4 * q4 + 2], x[dt][4 * q4 + 3]};
        }
        if (sink) return;
        const int64_t rs = is_v ? a.dv_rs : a.dk_rs, hs = is_v ? a.dv_hs : a.dk_hs;
        uint16_t *base = (is_v ? a.dv : a.dk) + (int64_t)(k_start + kw) * rs + (int64_t)kvh * hs;
        store_rows<D, T>(x, is_v ? 1.f : a.scale, smem + wave * 64 * D, head_dim, [&](int r) __attribute__((always_inline)) -> uint16_t * {
            return kw + r >= klen || (split && kw + r < a.sinks) ? nullptr : base + r * rs;
        });
    };
    if constexpr (PAIR) {
        store(dk, !dswave);
    } else {
        store(dv, true);
        store(dk, false);
    }
}

// The sinks' dK and dV: their parts in the parts' order, rounded once. A workgroup to a key and head; its quarters
// take a quarter of the parts each, eight loads in flight. 4 to 7 us: launch and those loads.
template <int D, typename T>
__global__ __launch_bounds__(8 * D) void fa_window_sink_sum_kernel(const WinBwdArgs a) {
    __shared__ float quarter[4][2 * D];
    const int key = blockIdx.x, bh = blockIdx.y, b = a.dheads.div(bh), kvh = bh - b * a.nheads_k;
    int k_start, klen;
    seq_bounds(a.cu_k, b, a.total_k, k_start, klen);
    if (key >= klen) return;
    const int x = threadIdx.x % (2 * D), part = threadIdx.x / (2 * D), is_v = x / D, d = x % D;
    const int per = (a.slots + 3) / 4, beg = part * per, end = beg + per < a.slots ? beg + per : a.slots;
    const float *p = a.ws_part + ((int64_t)bh * a.sinks + key) * a.slots * 2 * D + x;
    float sum = 0.f;
    for (int s = beg; s < end; s += 8) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = s + i < end ? p[(int64_t)(s + i) * 2 * D] : 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += v[i];
    }
    quarter[part][x] = sum;
    __syncthreads();
    if (part > 0 || d >= a.head_dim) return;
    sum = (quarter[0][x] + quarter[1][x]) + (quarter[2][x] + quarter[3][x]);
    if (is_v)
        a.dv[(int64_t)(k_start + key) * a.dv_rs + (int64_t)kvh * a.dv_hs + d] = T::from_float(sum);
    else
        a.dk[(int64_t)(k_start + key) * a.dk_rs + (int64_t)kvh * a.dk_hs + d] = T::from_float(sum * a.scale);
}

}  // namespace fa
