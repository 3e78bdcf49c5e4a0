// fa_window_careful.h — rows computed one key at a time, for results that came out infinite or NaN.
//
// The matrix instructions multiply a tile's values by weights of 0 where a row does not see a key, and 0 * inf is
// NaN: an infinity in a place that a row does not see (an unread page's leftovers, a token outside the window)
// would reach it through its tile. A wave whose sums are not all finite therefore computes them again here, taking
// only what each row sees; infinities that it does see come out as they should. One wave, one row or key at a time,
// lanes along head_dim: hundreds of times slower than the tiles, and never run on finite data.
#pragma once

#include "fa_window_common.h"

namespace fa {

// all of x finite? (wave-uniform)
template <int N>
__device__ __forceinline__ bool all_finite(const f32x16 (&x)[N], float more) {
    float t = more * 0.f;
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) t = fmaf(x[n][r], 0.f, t);
    return __builtin_amdgcn_ballot_w64(!(t == 0.f)) == 0;
}

__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
    for (int s = 32; s >= 1; s >>= 1) x += __shfl_xor(x, s);
    return x;
}

// A row of head_dim values over the lanes: E = D / 64 (at least 1) to a lane.
template <int D>
struct LaneRow {
    static constexpr int E = D >= 64 ? D / 64 : 1;
    float x[E];
    template <typename T>
    __device__ __forceinline__ void load(const uint16_t *p, int head_dim) {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = E * lane + e < head_dim ? T::to_float(p[E * lane + e]) : 0.f;
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = 0.f;
    }
    __device__ __forceinline__ float dot(const LaneRow &y) const {
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) s = fmaf(x[e], y.x[e], s);
        return wave_sum(s);
    }
    __device__ __forceinline__ void add(float w, const LaneRow &y) {
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = fmaf(w, y.x[e], x[e]);
    }
    // into lane rr's accumulators (column 32 dt + crow(r, lane / 32) in register r of block dt)
    __device__ __forceinline__ void put(f32x16 (&o)[D / 32], int rr) const {
        const int lane = threadIdx.x & 63, hi = lane >> 5;
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int d = 32 * dt + crow(r, hi);
                float v = __shfl(x[0], d / E);
                if constexpr (E == 2) {
                    const float w = __shfl(x[1], d / E);
                    v = d & 1 ? w : v;
                }
                if ((lane & 31) == rr) o[dt][r] = v;
            }
    }
};

}  // namespace fa
