// fa_window_launch.h — launchers of the windowed and paged kernels, one translation unit per head-dim tile.
#pragma once
#include "fa_launch.h"
#include "../../include/fa_window_hip.h"

namespace fa {
struct WinFwdArgs;
struct WinBwdArgs;
// `shape` of a forward launch: row waves x key groups x keys per tile
enum WinShape { WIN_4X1X64, WIN_2X2X32, WIN_1X4X32 };
int win_shape_rows(WinShape s);      // packed rows per workgroup
int win_shape_groups(WinShape s);
int win_shape_keys(WinShape s);      // keys per tile
template <int D> hipError_t launch_window_fwd(const WinFwdArgs &a, int dtype, bool paged, WinShape shape, hipStream_t s);

// dense forward: waves of 32 packed rows to a workgroup, keys to a tile. At 8192 tokens, 16 heads of 128 on 4, window
// 1024: 4 x 64 92 us, 4 x 32 96, 2 x 64 167 (one workgroup's LDS for half the waves), 2 x 32 117, 8 x 64 98; at 8 x 2048
// tokens, 12 heads of 64, window 256: 39, 39, 49, 37, 45, and at window 1024 65, 70, 85, 72, 76.
constexpr int WIN_FWD_WAVES = 4, WIN_FWD_KEYS = 64;
// backward: waves of 32 packed rows (dQ), blocks of 32 keys and waves (dK, dV) to a workgroup
constexpr int WIN_DQ_WAVES = 4, WIN_DKV_BLOCKS = 4;
constexpr int win_dkv_waves(int D) { return D == 128 ? 2 * WIN_DKV_BLOCKS : WIN_DKV_BLOCKS; }
struct WinBwdPlan {
    int max_rows, max_k, order;
    bool fine;
};
template <int D> hipError_t launch_window_bwd(const WinBwdArgs &a, int dtype, const WinBwdPlan &p, hipStream_t s);
// the error text of the C ABI (fa_api.cpp)
int set_error(int code, const char *fmt, ...) __attribute__((format(printf, 2, 3)));
void clear_error();
}  // namespace fa
