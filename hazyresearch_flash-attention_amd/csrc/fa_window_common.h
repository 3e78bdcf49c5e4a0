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
