// fa_window_kernels_impl.h — template launchers; included by fa_window_d{32,64,128}.hip.
#pragma once
#include "fa_window_launch.h"
#include "fa_window_fwd_kernel.h"
#include "fa_window_bwd_kernel.h"

namespace fa {

template <int D, typename T, int NWR, int KG, int BN, bool PAGED, bool TREE, bool FINE>
static hipError_t launch_window_fwd_k(const WinFwdArgs &a, hipStream_t s) {
    using C = WinFwdCfg<D, NWR, KG, BN>;
    auto kern = fa_window_fwd_kernel<D, T, NWR, KG, BN, PAGED, TREE, FINE>;
    const int lds = C::lds(TREE);
    FA_ENSURE_LDS(kern, lds);
    const int64_t wgs = (int64_t)a.nrb * a.nsplit * a.nheads_k * a.batch;
    hipLaunchKernelGGL(kern, dim3((uint32_t)wgs), dim3(C::NT), lds, s, a);
    return hipGetLastError();
}

template <int D, typename T>
static hipError_t launch_window_fwd_t(const WinFwdArgs &a, bool paged, WinShape shape, hipStream_t s) {
    if (!paged)
        return a.fine ? launch_window_fwd_k<D, T, WIN_FWD_WAVES, 1, WIN_FWD_KEYS, false, false, true>(a, s)
                      : launch_window_fwd_k<D, T, WIN_FWD_WAVES, 1, WIN_FWD_KEYS, false, false, false>(a, s);
    hipError_t e;
    const bool tree = a.tree != nullptr;
    switch (shape) {
        case WIN_4X1X64:
            e = tree ? launch_window_fwd_k<D, T, 4, 1, 64, true, true, false>(a, s)
                     : launch_window_fwd_k<D, T, 4, 1, 64, true, false, false>(a, s);
            break;
        case WIN_2X2X32:
            e = tree ? launch_window_fwd_k<D, T, 2, 2, 32, true, true, true>(a, s)
                     : launch_window_fwd_k<D, T, 2, 2, 32, true, false, true>(a, s);
            break;
        default:
            e = tree ? launch_window_fwd_k<D, T, 1, 4, 32, true, true, true>(a, s)
                     : launch_window_fwd_k<D, T, 1, 4, 32, true, false, true>(a, s);
    }
    if (e != hipSuccess || a.nsplit == 1) return e;
    // rows of the longest sequence that the forward's grid covers (nrb row blocks of the shape)
    const int64_t rows = (int64_t)a.nrb * win_shape_rows(shape) / a.group + 1;
    const dim3 grid((uint32_t)((rows * a.nheads + 3) / 4), a.batch);
    hipLaunchKernelGGL((fa_window_join_kernel<D, T>), grid, dim3(256), 0, s, a);
    return hipGetLastError();
}

template <int D>
hipError_t launch_window_fwd(const WinFwdArgs &a, int dtype, bool paged, WinShape shape, hipStream_t s) {
    return dtype == FA_DTYPE_BF16 ? launch_window_fwd_t<D, Bf16>(a, paged, shape, s)
                                  : launch_window_fwd_t<D, Fp16>(a, paged, shape, s);
}

template <int D, typename T, bool FINE>
static hipError_t launch_window_bwd_t(WinBwdArgs a, const WinBwdPlan &p, hipStream_t s) {
    hipError_t e = hipSuccess;
    if (p.max_rows > 0) {
        using C = WinDqCfg<D, WIN_DQ_WAVES>;
        auto kern = fa_window_dq_kernel<D, T, WIN_DQ_WAVES, FINE>;
        FA_ENSURE_LDS(kern, C::LDS);
        a.order = BlockOrder::of((p.max_rows + C::BM - 1) / C::BM, a.nheads_k * a.batch, p.order);
        hipLaunchKernelGGL(kern, dim3((uint32_t)((int64_t)a.order.nblk * a.order.nbh)), dim3(C::NT), C::LDS, s, a);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    if (p.max_k > 0) {
        using C = WinDkvCfg<D, win_dkv_waves(D), D == 128>;
        auto kern = fa_window_dkv_kernel<D, T, win_dkv_waves(D), D == 128, FINE>;
        FA_ENSURE_LDS(kern, C::LDS);
        static_assert(C::NB == WIN_DKV_BLOCKS, "the plan's blocks");
        a.order = BlockOrder::of((p.max_k + C::BK - 1) / C::BK, a.nheads_k * a.batch, p.order);
        const int64_t wgs = ((int64_t)a.order.nblk + (int64_t)a.chunks * a.sink_blocks) * a.order.nbh;
        hipLaunchKernelGGL(kern, dim3((uint32_t)wgs), dim3(C::NT), C::LDS, s, a);
        if ((e = hipGetLastError()) != hipSuccess) return e;
        if (a.chunks > 0) {
            hipLaunchKernelGGL((fa_window_sink_sum_kernel<D, T>), dim3(a.sinks, a.nheads_k * a.batch), dim3(8 * D), 0, s, a);
            e = hipGetLastError();
        }
    }
    return e;
}

template <int D, typename T>
static hipError_t launch_window_bwd_f(const WinBwdArgs &a, const WinBwdPlan &p, hipStream_t s) {
    return p.fine ? launch_window_bwd_t<D, T, true>(a, p, s) : launch_window_bwd_t<D, T, false>(a, p, s);
}

template <int D>
hipError_t launch_window_bwd(const WinBwdArgs &a, int dtype, const WinBwdPlan &p, hipStream_t s) {
    return dtype == FA_DTYPE_BF16 ? launch_window_bwd_f<D, Bf16>(a, p, s) : launch_window_bwd_f<D, Fp16>(a, p, s);
}

}  // namespace fa
