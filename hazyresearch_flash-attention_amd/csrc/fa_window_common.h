// fa_window_common.h — what the windowed kernels share: the visibility rule as bit masks, the walk over the
// tiles that a block of rows sees, K/V staging into LDS.
//
// A query at position p sees key j when j <= p and (j > p - W or j < sinks). Rows of one sequence and one
// key/value head are packed: row r is token t = r / G of query head g = r % G of the head's group of G, so a
// tile of K/V staged once serves the whole group and a position's G rows lie side by side.
#pragma once

#include "fa_common.h"
#include "fa_launch.h"
#include "../../include/fa_window_hip.h"

namespace fa {

// bits 0 .. n-1 (n clamped to [0, 32])
__device__ __forceinline__ uint32_t bits_below(int n) {
    n = n < 0 ? 0 : (n > 32 ? 32 : n);
    return (uint32_t)((1ull << n) - 1ull);
}

// keys j0 .. j0+31 that position p sees, as bits
__device__ __forceinline__ uint32_t seen_bits(int j0, int p, int window, int sinks) {
    return bits_below(p + 1 - j0) & (~bits_below(p + 1 - window - j0) | bits_below(sinks - j0));
}

// The tiles of BN keys that positions pmin..pmax see, with keys below k_end: the sink tiles [0, ts) and the
// window's tiles, `gap` tiles further on; n in all.
struct TileWalk {
    int n, ts, gap;
    __device__ __forceinline__ int tile(int i) const { return i < ts ? i : i + gap; }
};
__device__ __forceinline__ TileWalk tile_walk(int pmin, int k_end, int window, int sinks, int bn) {
    TileWalk w;
    const int te = k_end > 0 ? (k_end + bn - 1) / bn : 0;
    const int w0 = pmin - window + 1;
    const int tw = w0 > 0 ? w0 / bn : 0;
    const int se = sinks < k_end ? sinks : (k_end > 0 ? k_end : 0);
    const int ts = (se + bn - 1) / bn;
    if (tw <= ts) {
        w.n = te; w.ts = te; w.gap = 0;
    } else {
        w.ts = ts; w.gap = tw - ts;
        w.n = ts + (te > tw ? te - tw : 0);
    }
    return w;
}

// n / d for 0 <= n < 2^31 by one 64-bit product: m = ceil(2^(31 + l) / d), l = ceil(log2 d). An integer division is
// some 40 instructions, and a workgroup's start has half a dozen of them.
struct Div {
    uint32_t m, sh;
    int d;
    __host__ static Div of(int d) {
        Div x;
        x.d = d < 1 ? 1 : d;
        uint32_t l = 0;
        while ((1ll << l) < x.d) ++l;
        x.sh = 31 + l;
        x.m = (uint32_t)(((1ull << x.sh) + (uint64_t)x.d - 1) / (uint64_t)x.d);
        return x;
    }
    __device__ __forceinline__ int div(int n) const { return (int)(((uint64_t)(uint32_t)n * m) >> sh); }
};

// Order of the workgroups L of a grid of nbh (sequence, head) pairs with nblk blocks each (late blocks first: they
// see the most keys while a window fills). The dispatcher hands workgroup L to XCD L & 7.
//   order > 0: pairs a multiple of 8. Each XCD takes nbh / 8 of them in groups of `order`, block by block with the
//              group's pairs side by side: the blocks that run at once are alike long, the rows of neighbouring
//              heads (which lie side by side in memory) are read together, a group's K/V fit the XCD's L2.
//   order = 0: each XCD a contiguous run of blocks, pair by pair (few pairs, equal blocks: a window's keys are
//              read by one XCD).
//   order < 0: all pairs' late blocks first, whatever the XCD (few pairs, unequal blocks).
struct BlockOrder {
    int nblk, nbh, order;
    Div blk, group, last, per, pairs;
    __host__ static BlockOrder of(int nblk, int nbh, int order) {
        const int nh = nbh / 8, rest = order > 0 && nh % order ? nh % order : order;
        return {nblk, nbh, order, Div::of(nblk), Div::of(order), Div::of(rest), Div::of(order > 0 ? order * nblk : 1), Div::of(nbh)};
    }
    __device__ __forceinline__ void get(int L, int &block, int &bh) const {
        int rank;
        if (order > 0) {
            const int nh = nbh >> 3, i = L >> 3;
            const int grp = per.div(i), w = i - grp * per.d;
            const bool full = nh - grp * order >= order;
            const Div &g = full ? group : last;
            rank = g.div(w);
            bh = (L & 7) * nh + grp * order + (w - rank * g.d);
        } else if (order == 0) {
            const int w = xcd_contiguous(L, nblk * nbh);
            bh = blk.div(w);
            rank = w - bh * nblk;
        } else {
            rank = pairs.div(L);
            bh = L - rank * nbh;
        }
        block = nblk - 1 - rank;
    }
};

// Wave-uniform 32-bit load through the scalar cache: block-table entries, one for a whole tile.
__device__ __forceinline__ int uniform_load(const int32_t *p) {
    typedef const int32_t __attribute__((address_space(4))) *cp;
    return *(cp)(uintptr_t)p;
}

// Sequence bounds from cu_seqlens, cut to the rows that there are.
__device__ __forceinline__ void seq_bounds(const int32_t *cu, int b, int64_t total, int &start, int &len) {
    const int tot = (int)total;
    int s = cu[b], e = cu[b + 1];
    s = s < 0 ? 0 : (s > tot ? tot : s);
    e = e > tot ? tot : e;
    start = s;
    len = e > s ? e - s : 0;
}

// A wave's 32 x D accumulators (X^T: lane = row l & 31, register r of block dt = column 32 dt + crow(r, lane / 32)) to
// global rows in 16 bits, through 64 D bytes of LDS of its own, so that a store instruction writes whole rows: from
// the registers it would be 8 bytes to each of 64 places. to(row) is where row 0..31 goes, or null.
template <int D, typename T, typename F>
__device__ __forceinline__ void store_rows(const f32x16 (&x)[D / 32], float mul, char *lds, int head_dim, F &&to) {
    using S = Swz<D>;
    const int lane = threadIdx.x & 63, l32 = lane & 31, hi = lane >> 5;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4)
            lds_write64(lds, S::off8(l32, 32 * dt + 8 * q4 + 4 * hi),
                        u32x2{T::pack2(x[dt][4 * q4] * mul, x[dt][4 * q4 + 1] * mul),
                              T::pack2(x[dt][4 * q4 + 2] * mul, x[dt][4 * q4 + 3] * mul)});
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    constexpr int NC = D / 8;
#pragma unroll
    for (int i = 0; i < NC / 2; ++i) {
        const int r = (lane + 64 * i) / NC, c = (lane + 64 * i) % NC;
        const u32x4 v = lds_read128(lds, S::off(r, c));
        uint16_t *p = to(r);
        if (p && c * 8 < head_dim) gstore128(p + c * 8, v);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Rows behind the last sequence belong to none: outputs are 0 there, whatever the allocation held. Every
// workgroup takes its share (usually there are none: one load).
__device__ __forceinline__ void zero_tail(uint16_t *p, int64_t rs, int64_t hs, int heads, int head_dim, int64_t total,
                                          const int32_t *cu, int batch) {
    int64_t end = cu[batch];
    end = end < 0 ? 0 : end;
    const int hc = head_dim / 8;
    for (int64_t r = end + blockIdx.x; r < total; r += gridDim.x)
        for (int x = threadIdx.x; x < heads * hc; x += blockDim.x)
            gstore128(p + r * rs + (int64_t)(x / hc) * hs + (x % hc) * 8, u32x4{0u, 0u, 0u, 0u});
}

}  // namespace fa
