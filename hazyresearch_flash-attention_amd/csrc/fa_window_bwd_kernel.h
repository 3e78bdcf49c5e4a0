// fa_window_bwd_kernel.h — backward of the windowed attention (dense var-len, grouped heads).
//
// With P = exp(scale Q K^T - lse) on the entries a row sees and 0 elsewhere, delta = rowsum(dO * O):
//     dP = dO V^T,  dS = P (dP - delta),  dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO,
// dK and dV summed over the query heads of a group. Two kernels, each writing its outputs once, in one order, with
// no atomics: dQ by query rows (the forward's walk), dK and dV by keys. S and dP are computed in both: 7 matrix
// products of the forward's size against 5 with dQ by fp32 atomics, whose order changes the result and whose
// rate bounds it (1.3 TB/s measured for the dense backward).
#pragma once

#include "fa_window_common.h"

namespace fa {

struct WinBwdArgs {
    const uint16_t *q, *k, *v, *dout;
    const float *lse, *delta;
    uint16_t *dq, *dk, *dv;
    float *ws;
    const int32_t *cu_q, *cu_k;
    int64_t q_rs, q_hs, k_rs, k_hs, v_rs, v_hs, do_rs, do_hs;
    int64_t dq_rs, dq_hs, dk_rs, dk_hs, dv_rs, dv_hs;
    int64_t total_q, total_k;
    int batch, nheads, nheads_k, head_dim, group;
    int lse_stride, window, sinks, nblk;
    float scale;
};

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
template <int D, typename T, int NW>
__global__ __launch_bounds__(64 * NW, 2) void fa_window_dq_kernel(const WinBwdArgs a) {
    using C = WinDqCfg<D, NW>;
    using S = Swz<D>;
    constexpr float LOG2E = 1.4426950408889634f;
    extern __shared__ __attribute__((aligned(16))) char smem[];

    zero_tail(a.dq, a.dq_rs, a.dq_hs, a.nheads, a.head_dim, a.total_q, a.cu_q, a.batch);
    int w = xcd_contiguous(blockIdx.x, gridDim.x);
    const int rb = a.nblk - 1 - w % a.nblk;
    w /= a.nblk;
    const int kvh = w % a.nheads_k;
    const int b = w / a.nheads_k;
    int q_start, sq, k_start, klen;
    seq_bounds(a.cu_q, b, a.total_q, q_start, sq);
    seq_bounds(a.cu_k, b, a.total_k, k_start, klen);
    const int off = klen - sq;
    const int G = a.group, R = sq * G, r0 = rb * C::BM;
    if (r0 >= R) return;

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l32 = lane & 31, hi = lane >> 5;
    const int head_dim = a.head_dim;
    const int rw = r0 + 32 * wave, row = rw + l32;
    const int rc = row < R ? row : R - 1;
    const int t = rc / G, g = rc - t * G, h = kvh * G + g;
    const int pos = off + t;
    int pmin = off + rw / G, pmax = off + (rw + 31 < R ? rw + 31 : R - 1) / G;
    if (rw >= R) pmin = pmax = pos;
    int k_end = off + (r0 + C::BM < R ? r0 + C::BM - 1 : R - 1) / G + 1;
    k_end = k_end < klen ? k_end : klen;
    const TileWalk walk = tile_walk(off + r0 / G, k_end, a.window, a.sinks, C::BN);

    typename T::frag qf[D / 16], df[D / 16];
    {
        const uint16_t *qp = a.q + (int64_t)(q_start + t) * a.q_rs + (int64_t)h * a.q_hs;
        const uint16_t *dp = a.dout + (int64_t)(q_start + t) * a.do_rs + (int64_t)h * a.do_hs;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
            const int c = 2 * ks + hi;
            u32x4 x = {0u, 0u, 0u, 0u}, y = {0u, 0u, 0u, 0u};
            if (c * 8 < head_dim) {
                x = gload128(qp + c * 8);
                y = gload128(dp + c * 8);
            }
            qf[ks] = as_frag<T>(x);
            df[ks] = as_frag<T>(y);
        }
    }
    const int64_t li = (int64_t)(b * a.nheads + h) * a.lse_stride + t;
    const float lse2 = a.lse[li] * LOG2E, delta = a.delta[li];
    const float c_log2 = a.scale * LOG2E;

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

    const int grp = (lane >> 4) & 1, qq = (lane & 15) >> 2, pp = lane & 3;
    int k_rd[2][D / 16];
#pragma unroll
    for (int st = 0; st < 2; ++st)
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) k_rd[st][ks] = S::off(32 * st + l32, 2 * ks + hi);
    int t_rd[D / 32][2][2][2];
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
        for (int st = 0; st < 2; ++st)
#pragma unroll
            for (int s2 = 0; s2 < 2; ++s2) {
                const int r = 32 * st + 16 * s2 + 4 * hi + qq, col = 32 * dt + 16 * grp + 4 * pp;
                t_rd[dt][st][s2][0] = S::off8(r, col);
                t_rd[dt][st][s2][1] = S::off8(r + 8, col);
            }

    f32x16 dq[D / 32];
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) dq[dt][r] = 0.f;

    auto compute = [&](int j0, int buf) __attribute__((always_inline)) {
        const char *kb = smem + buf * C::TILE, *vb = smem + (2 + buf) * C::TILE;
        typename T::frag pf[2][2];
        // the mask runs in a copy of the sub-tile behind one wave-uniform branch: P and dS by selection, so that
        // an infinity in a masked place (lse of a row that sees nothing) adds 0
        auto sub = [&](auto masked_tag) __attribute__((always_inline)) {
            constexpr bool MASKED = decltype(masked_tag)::value;
#pragma unroll
            for (int st = 0; st < 2; ++st) {
                f32x16 s, dp;
#pragma unroll
                for (int r = 0; r < 16; ++r) { s[r] = 0.f; dp[r] = -delta; }
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks) {
                    s = T::mfma32(as_frag<T>(lds_read128(kb, k_rd[st][ks])), qf[ks], s);
                    dp = T::mfma32(as_frag<T>(lds_read128(vb, k_rd[st][ks])), df[ks], dp);
                }
                uint32_t m = 0;
                if constexpr (MASKED) {
                    const int j = j0 + 32 * st;
                    m = (seen_bits(j, pos, a.window, a.sinks) & bits_below(klen - j)) >> (4 * hi);
                }
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const float x = fast_exp2(fmaf(s[r], c_log2, -lse2)) * dp[r];
                    s[r] = MASKED && !(m & (1u << crow(r, 0))) ? 0.f : x;
                }
#pragma unroll
                for (int s2 = 0; s2 < 2; ++s2) {
                    u32x4 pk;
#pragma unroll
                    for (int e = 0; e < 4; ++e) pk[e] = T::pack2(s[8 * s2 + 2 * e], s[8 * s2 + 2 * e + 1]);
                    pf[st][s2] = as_frag<T>(pk);
                }
            }
        };
        const bool whole = j0 + C::BN - 1 <= pmin && (j0 > pmax - a.window || j0 + C::BN <= a.sinks) && j0 + C::BN <= klen;
        if (__builtin_amdgcn_readfirstlane((int)whole))
            sub(std::false_type{});
        else
            sub(std::true_type{});
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
            for (int st = 0; st < 2; ++st)
#pragma unroll
                for (int s2 = 0; s2 < 2; ++s2) {
                    const u32x2 lo = lds_read_tr(kb, t_rd[dt][st][s2][0]);
                    const u32x2 hv = lds_read_tr(kb, t_rd[dt][st][s2][1]);
                    dq[dt] = T::mfma32(as_frag<T>(u32x4{lo[0], lo[1], hv[0], hv[1]}), pf[st][s2], dq[dt]);
                }
    };
    auto step = [&](auto par, int i) __attribute__((always_inline)) {
        constexpr int P = decltype(par)::value;
        if (i + 1 < walk.n) stage(i + 1, 1 - P);
        const int j0 = walk.tile(i) * C::BN;
        if (rw < R && j0 <= pmax && (j0 + C::BN - 1 > pmin - a.window || j0 < a.sinks)) compute(j0, P);
        vmcnt0();
        __syncthreads();
    };
    if (walk.n > 0) stage(0, 0);
    vmcnt0();       // (the compiler's counters see it: the loop inherits no pending prologue load)
    __syncthreads();
    for (int i = 0; i < walk.n; i += 2) {
        step(std::integral_constant<int, 0>(), i);
        if (i + 1 < walk.n) step(std::integral_constant<int, 1>(), i + 1);
    }

    if (row >= R) return;
    uint16_t *op = a.dq + (int64_t)(q_start + t) * a.dq_rs + (int64_t)h * a.dq_hs;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
            const int d = 32 * dt + 8 * q4 + 4 * hi;
            if (d < head_dim)
                gstore64(op + d, u32x2{T::pack2(dq[dt][4 * q4] * a.scale, dq[dt][4 * q4 + 1] * a.scale),
                                       T::pack2(dq[dt][4 * q4 + 2] * a.scale, dq[dt][4 * q4 + 3] * a.scale)});
        }
}

// ------------------------------------------------------------------------------------------- dK, dV
template <int D, int NW>
struct WinDkvCfg {
    static constexpr int NT = 64 * NW;
    static constexpr int BK = 32 * NW;                 // keys per workgroup
    static constexpr int BR = 32;                      // packed query rows per step
    static constexpr int NC = D / 8;
    static constexpr int TILE = BR * D * 2;
    static constexpr int PIECES = TILE / 1024;
    static constexpr int PPW = (PIECES + NW - 1) / NW;
    static constexpr int RPP = 1024 / (2 * D);
    static constexpr int OFF_DO = 2 * TILE;
    static constexpr int OFF_ROW = 4 * TILE;           // lse[2][BR], delta[2][BR]
    static constexpr int LDS = OFF_ROW + 4 * BR * 4;
};

// A wave owns 32 keys (lane = key), whose K and V rows and dK^T, dV^T stay in registers, and walks the packed
// query rows that see the workgroup's keys, all heads of the group one after the other: S = Q K^T, dP = dO V^T with
// Q and dO rows from LDS; P and dS in registers are the B operands of dV^T += dO^T P and dK^T += Q^T dS.
template <int D, typename T, int NW>
__global__ __launch_bounds__(64 * NW, D <= 64 ? 2 : 1) void fa_window_dkv_kernel(const WinBwdArgs a) {
    using C = WinDkvCfg<D, NW>;
    using S = Swz<D>;
    constexpr float LOG2E = 1.4426950408889634f;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    float *row_s = (float *)(smem + C::OFF_ROW);

    zero_tail(a.dk, a.dk_rs, a.dk_hs, a.nheads_k, a.head_dim, a.total_k, a.cu_k, a.batch);
    zero_tail(a.dv, a.dv_rs, a.dv_hs, a.nheads_k, a.head_dim, a.total_k, a.cu_k, a.batch);
    int w = xcd_contiguous(blockIdx.x, gridDim.x);
    const int kb = w % a.nblk;
    w /= a.nblk;
    const int kvh = w % a.nheads_k;
    const int b = w / a.nheads_k;
    int q_start, sq, k_start, klen;
    seq_bounds(a.cu_q, b, a.total_q, q_start, sq);
    seq_bounds(a.cu_k, b, a.total_k, k_start, klen);
    const int off = klen - sq;
    const int G = a.group, k0 = kb * C::BK;
    if (k0 >= klen) return;

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l32 = lane & 31, hi = lane >> 5;
    const int head_dim = a.head_dim;
    const int kw = k0 + 32 * wave, key = kw + l32;

    // packed rows that see a key of the block: [r_beg, r_end). Key j is seen from row (j - off) G on, up to row
    // (j - off + window) G, a sink by every row from there on.
    const int t_beg = k0 - off > 0 ? k0 - off : 0;
    int64_t t_end64 = k0 < a.sinks ? sq : (int64_t)k0 + C::BK - 1 + a.window - off;
    const int t_end = t_end64 < 0 ? 0 : (t_end64 < sq ? (int)t_end64 : sq);
    const int r_beg = t_beg * G, r_end = t_end * G;
    const int nt = r_end > r_beg ? (r_end - r_beg + C::BR - 1) / C::BR : 0;

    typename T::frag kf[D / 16], vf[D / 16];
    {
        const int kc = key < klen ? key : klen - 1;
        const uint16_t *kp = a.k + (int64_t)(k_start + kc) * a.k_rs + (int64_t)kvh * a.k_hs;
        const uint16_t *vp = a.v + (int64_t)(k_start + kc) * a.v_rs + (int64_t)kvh * a.v_hs;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
            const int c = 2 * ks + hi;
            u32x4 x = {0u, 0u, 0u, 0u}, y = {0u, 0u, 0u, 0u};
            if (c * 8 < head_dim) {
                x = gload128(kp + c * 8);
                y = gload128(vp + c * 8);
            }
            kf[ks] = as_frag<T>(x);
            vf[ks] = as_frag<T>(y);
        }
    }
    f32x16 dk[D / 32], dv[D / 32];
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) { dk[dt][r] = 0.f; dv[dt][r] = 0.f; }
    const float c_log2 = a.scale * LOG2E;

    // ---- staging of one tile of packed rows: row r is token r / G of head kvh G + r % G; rows behind the last
    // one land as zeros
    const uint16_t *qbase = a.q + (int64_t)q_start * a.q_rs + (int64_t)kvh * G * a.q_hs;
    const uint16_t *dbase = a.dout + (int64_t)q_start * a.do_rs + (int64_t)kvh * G * a.do_hs;
    auto stage = [&](int i, int buf) __attribute__((always_inline)) {
        const int rt = r_beg + i * C::BR;
        const int t0 = rt / G;                         // the descriptor starts at the tile's first token
        const i32x4 qs = make_srd(qbase + (int64_t)t0 * a.q_rs, 0x7FFFFFFF);
        const i32x4 ds = make_srd(dbase + (int64_t)t0 * a.do_rs, 0x7FFFFFFF);
#pragma unroll
        for (int n = 0; n < C::PPW; ++n) {
            const int p = wave + NW * n;
            if (C::PIECES % NW == 0 || p < C::PIECES) {
                const int r = C::RPP * p + lane / C::NC;
                const int c = (lane % C::NC) ^ S::x(r);
                const int t = (rt + r) / G, g = rt + r - t * G;
                const bool ok = rt + r < r_end && c * 8 < head_dim;
                const int qo = ok ? ((t - t0) * (int)a.q_rs + g * (int)a.q_hs + c * 8) * 2 : OOB;
                const int dof = ok ? ((t - t0) * (int)a.do_rs + g * (int)a.do_hs + c * 8) * 2 : OOB;
                dma16(qs, qo, 0, lds_addr(smem + buf * C::TILE + 1024 * p));
                dma16(ds, dof, 0, lds_addr(smem + C::OFF_DO + buf * C::TILE + 1024 * p));
            }
        }
    };
    // lse and delta of the tile's rows: loaded by the first 32 lanes a step ahead, written at the step's end
    float lse_st = 0.f, del_st = 0.f;
    auto load_rows = [&](int i) __attribute__((always_inline)) {
        if (tid < C::BR) {
            int r = r_beg + i * C::BR + tid;
            r = r < r_end ? r : r_end - 1;
            const int t = r / G, g = r - t * G;
            const int64_t li = (int64_t)(b * a.nheads + kvh * G + g) * a.lse_stride + t;
            lse_st = a.lse[li] * LOG2E;
            del_st = -a.delta[li];
        }
    };
    auto store_rows = [&](int buf) __attribute__((always_inline)) {
        if (tid < C::BR) {
            row_s[buf * C::BR + tid] = lse_st;
            row_s[(2 + buf) * C::BR + tid] = del_st;
        }
    };

    const int grp = (lane >> 4) & 1, qq = (lane & 15) >> 2, pp = lane & 3;
    auto compute = [&](int i, int buf) __attribute__((always_inline)) {
        const char *qb = smem + buf * C::TILE, *db = smem + C::OFF_DO + buf * C::TILE;
        const float *lse_b = row_s + buf * C::BR, *del_b = row_s + (2 + buf) * C::BR;
        const int rt = r_beg + i * C::BR;
        f32x16 s, dp;
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
            const f32x4 d4 = *reinterpret_cast<const f32x4 *>(del_b + 8 * q4 + 4 * hi);
#pragma unroll
            for (int e = 0; e < 4; ++e) { s[4 * q4 + e] = 0.f; dp[4 * q4 + e] = d4[e]; }   // dP starts at -delta
        }
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
            const int ro = S::off(l32, 2 * ks + hi);
            s = T::mfma32(as_frag<T>(lds_read128(qb, ro)), kf[ks], s);
            dp = T::mfma32(as_frag<T>(lds_read128(db, ro)), vf[ks], dp);
        }
        // rows of the tile that see this lane's key, as bits
        const int lo = (key - off) * G - rt;
        const int64_t up64 = key < a.sinks ? (int64_t)r_end - rt : (int64_t)(key - off + (int64_t)a.window) * G - rt;
        const int up = (int)(up64 < 0 ? 0 : (up64 > 32 ? 32 : up64));
        uint32_t m = bits_below(up) & ~bits_below(lo) & bits_below(r_end - rt);
        if (key >= klen) m = 0;
        const bool whole = __builtin_amdgcn_ballot_w64(m != 0xFFFFFFFFu) == 0;
        m >>= 4 * hi;
        auto pds = [&](auto masked_tag) __attribute__((always_inline)) {
            constexpr bool MASKED = decltype(masked_tag)::value;
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4) {
                const f32x4 l4 = *reinterpret_cast<const f32x4 *>(lse_b + 8 * q4 + 4 * hi);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int r = 4 * q4 + e;
                    const bool dead = MASKED && !(m & (1u << crow(r, 0)));
                    const float p = fast_exp2(fmaf(s[r], c_log2, -l4[e]));
                    const float x = p * dp[r];
                    s[r] = dead ? 0.f : p;
                    dp[r] = dead ? 0.f : x;
                }
            }
        };
        if (whole)
            pds(std::false_type{});
        else
            pds(std::true_type{});
        u32x4 pk[2], sk[2];
#pragma unroll
        for (int sg = 0; sg < 2; ++sg)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                pk[sg][e] = T::pack2(s[8 * sg + 2 * e], s[8 * sg + 2 * e + 1]);
                sk[sg][e] = T::pack2(dp[8 * sg + 2 * e], dp[8 * sg + 2 * e + 1]);
            }
#pragma unroll
        for (int sg = 0; sg < 2; ++sg)
#pragma unroll
            for (int dt = 0; dt < D / 32; ++dt) {
                const int r = 16 * sg + 4 * hi + qq, col = 32 * dt + 16 * grp + 4 * pp;
                const int o0 = S::off8(r, col), o1 = S::off8(r + 8, col);
                const u32x2 a0 = lds_read_tr(db, o0), a1 = lds_read_tr(db, o1);
                dv[dt] = T::mfma32(as_frag<T>(u32x4{a0[0], a0[1], a1[0], a1[1]}), as_frag<T>(pk[sg]), dv[dt]);
                const u32x2 b0 = lds_read_tr(qb, o0), b1 = lds_read_tr(qb, o1);
                dk[dt] = T::mfma32(as_frag<T>(u32x4{b0[0], b0[1], b1[0], b1[1]}), as_frag<T>(sk[sg]), dk[dt]);
            }
    };
    // a wave skips a tile that sees none of its 32 keys
    const int w_lo = (kw - off) * G;
    const int64_t w_up = kw < a.sinks ? (int64_t)r_end : (int64_t)((int64_t)kw + 31 - off + a.window) * G;
    auto step = [&](auto par, int i) __attribute__((always_inline)) {
        constexpr int P = decltype(par)::value;
        if (i + 1 < nt) {
            stage(i + 1, 1 - P);
            load_rows(i + 1);
        }
        const int rt = r_beg + i * C::BR;
        if (kw < klen && rt + C::BR > w_lo && rt < w_up) compute(i, P);
        if (i + 1 < nt) store_rows(1 - P);
        vmcnt0();
        __syncthreads();
    };
    if (nt > 0) {
        stage(0, 0);
        load_rows(0);
        store_rows(0);
    }
    vmcnt0();
    __syncthreads();
    for (int i = 0; i < nt; i += 2) {
        step(std::integral_constant<int, 0>(), i);
        if (i + 1 < nt) step(std::integral_constant<int, 1>(), i + 1);
    }

    if (key >= klen) return;
    uint16_t *kp = a.dk + (int64_t)(k_start + key) * a.dk_rs + (int64_t)kvh * a.dk_hs;
    uint16_t *vp = a.dv + (int64_t)(k_start + key) * a.dv_rs + (int64_t)kvh * a.dv_hs;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
            const int d = 32 * dt + 8 * q4 + 4 * hi;
            if (d < head_dim) {
                gstore64(kp + d, u32x2{T::pack2(dk[dt][4 * q4] * a.scale, dk[dt][4 * q4 + 1] * a.scale),
                                       T::pack2(dk[dt][4 * q4 + 2] * a.scale, dk[dt][4 * q4 + 3] * a.scale)});
                gstore64(vp + d, u32x2{T::pack2(dv[dt][4 * q4], dv[dt][4 * q4 + 1]),
                                       T::pack2(dv[dt][4 * q4 + 2], dv[dt][4 * q4 + 3])});
            }
        }
}

}  // namespace fa
