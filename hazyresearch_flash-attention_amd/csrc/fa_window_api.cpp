// fa_window_api.cpp — the C ABI of include/fa_window_hip.h: argument checks, the choice of a launch shape and of
// the split, workspace sizes. Nothing here touches device memory; sizes that come from the device (cu_seqlens,
// context lengths, table entries) are checked by the kernels.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "fa_window_launch.h"
#include "fa_window_fwd_kernel.h"
#include "fa_window_bwd_kernel.h"

namespace fa {

int win_shape_rows(WinShape s) { return s == WIN_4X1X64 ? 128 : s == WIN_2X2X32 ? 64 : 32; }
int win_shape_groups(WinShape s) { return s == WIN_4X1X64 ? 1 : s == WIN_2X2X32 ? 2 : 4; }
int win_shape_keys(WinShape s) { return s == WIN_4X1X64 ? 64 : 32; }

namespace {

constexpr int NO_WINDOW = 0x3FFFFFFF;      // more than any position (lengths are below 2^30)
constexpr int64_t LEN_LIMIT = 1 << 30;

int tile_of(int head_dim) { return head_dim <= 32 ? 32 : head_dim <= 64 ? 64 : 128; }

// block_order's `order` (fa_window_common.h). A group's K/V (the keys in view of its heads) stay below 8 MiB, twice
// an XCD's L2: 8 x 2048 tokens, 12 heads of 64, no window: groups of 12 dkv 163 us, of 8 173, of 1 198.
int order_for(int64_t pairs, int64_t window, int64_t max_k, int head_dim) {
    const int64_t keys = window < max_k ? window : max_k;
    if (pairs % 8 == 0) {
        const int64_t one = (keys > 64 ? keys : 64) * tile_of(head_dim) * 4, g = ((int64_t)8 << 20) / one;
        return (int)(g < 1 ? 1 : (g > pairs / 8 ? pairs / 8 : g));
    }
    return 2 * keys <= max_k ? 0 : -1;
}
int cus() {
    const int n = device_cus();
    return n > 0 ? n : 256;
}

// Whether the products take P and dS in two 16-bit parts (fa_window_fwd_kernel.h, FINE): workgroups of `rows` packed rows
// that see few keys and all run at once, so that latency and not the matrix units bounds the call, and whose results are few,
// so that their roundings do not average out. 5 sequences up to 701, 6 heads of 80 on 2, window 100: kernels 77 us for 66,
// the call 80 either way (the host's); 8 x 2048 tokens, 12 heads of 64, window 100, 1536 workgroups: 175 for 141.
bool takes_fine(const FaWindowArgs *a, int64_t window, int rows) {
    const int group = a->nheads / a->nheads_k;
    const int64_t seen = window + rows / group + 1 + a->num_sinks;
    const int64_t wgs = ((int64_t)a->max_seqlen_q * group + rows - 1) / rows * a->nheads_k * a->batch;
    return (seen < a->max_seqlen_k ? seen : a->max_seqlen_k) <= 256 && wgs <= 2 * cus();
}
bool al16(const void *p) { return ((uintptr_t)p & 15) == 0; }

// what both entry families ask of the sizes
int check_sizes(const char *fn, int batch, int nheads, int nheads_k, int head_dim, int max_q, int window, int sinks,
                float scale, int dtype) {
    if (dtype != FA_DTYPE_FP16 && dtype != FA_DTYPE_BF16)
        return set_error(FA_ERR_INVALID_ARGUMENT, "%s: dtype must be fp16 or bf16", fn);
    if (batch <= 0 || batch > 65535) return set_error(FA_ERR_INVALID_ARGUMENT, "%s: batch_size must be in [1, 65535]", fn);
    if (nheads <= 0 || nheads_k <= 0 || nheads % nheads_k != 0)
        return set_error(FA_ERR_INVALID_ARGUMENT, "%s: nheads must be a positive multiple of nheads_k (got %d, %d)", fn, nheads, nheads_k);
    if (nheads > 65535) return set_error(FA_ERR_UNSUPPORTED, "%s: more than 65535 heads", fn);
    if (head_dim <= 0 || head_dim % 8 != 0 || head_dim > 128)
        return set_error(FA_ERR_UNSUPPORTED, "%s: head_size must be a multiple of 8 and <= 128 (got %d)", fn, head_dim);
    if (max_q < 0) return set_error(FA_ERR_INVALID_ARGUMENT, "%s: max_seqlen must be >= 0", fn);
    if (window < 0) return set_error(FA_ERR_INVALID_ARGUMENT, "%s: window must be >= 0 (0: none)", fn);
    if (sinks < 0) return set_error(FA_ERR_INVALID_ARGUMENT, "%s: num_sinks must be >= 0", fn);
    if (!std::isfinite(scale)) return set_error(FA_ERR_INVALID_ARGUMENT, "%s: softmax_scale must be finite", fn);
    return FA_OK;
}

// a (rows, heads, head_dim) tensor: 16-byte rows that do not overlap, a tile of rows within 32-bit offsets
int check_rows(const char *fn, const char *name, const void *p, int64_t rs, int64_t hs, int heads, int head_dim) {
    if (!p) return set_error(FA_ERR_INVALID_ARGUMENT, "%s: %s is NULL", fn, name);
    if (!al16(p) || rs % 8 || hs % 8)
        return set_error(FA_ERR_INVALID_ARGUMENT, "%s: %s must be 16-byte aligned with strides multiple of 8", fn, name);
    if (rs < 0 || hs < 0 || (heads > 1 && hs < head_dim) || rs < (int64_t)(heads - 1) * hs + head_dim)
        return set_error(FA_ERR_INVALID_ARGUMENT, "%s: rows of %s overlap", fn, name);
    if (rs >= (int64_t)1 << 23) return set_error(FA_ERR_UNSUPPORTED, "%s: row stride of %s is 2^23 elements or more", fn, name);
    return FA_OK;
}

int check_window(const FaWindowArgs *a, const char *fn, bool bwd) {
    if (!a) return set_error(FA_ERR_INVALID_ARGUMENT, "%s: args is NULL", fn);
    int rc = check_sizes(fn, a->batch, a->nheads, a->nheads_k, a->head_dim, a->max_seqlen_q, a->window, a->num_sinks,
                         a->softmax_scale, a->dtype);
    if (rc) return rc;
    if (a->reserved != 0) return set_error(FA_ERR_INVALID_ARGUMENT, "%s: reserved must be 0", fn);
    if (a->max_seqlen_k < 0 || a->total_q < 0 || a->total_k < 0)
        return set_error(FA_ERR_INVALID_ARGUMENT, "%s: negative length", fn);
    if (a->total_q >= LEN_LIMIT || a->total_k >= LEN_LIMIT || a->max_seqlen_k >= LEN_LIMIT ||
        (a->total_q + a->total_k + a->max_seqlen_q) * (a->nheads / a->nheads_k) >= LEN_LIMIT)
        return set_error(FA_ERR_UNSUPPORTED, "%s: 2^30 or more rows", fn);
    if (!a->cu_seqlens_q || !a->cu_seqlens_k) return set_error(FA_ERR_INVALID_ARGUMENT, "%s: cu_seqlens is NULL", fn);
    if (a->lse_stride < a->max_seqlen_q) return set_error(FA_ERR_INVALID_ARGUMENT, "%s: lse_stride < max_seqlen_q", fn);
    const int d = a->head_dim;
    const bool has_q = a->total_q > 0 && a->max_seqlen_q > 0, has_k = a->total_k > 0;
    if (has_q) {
        if (!a->softmax_lse) return set_error(FA_ERR_INVALID_ARGUMENT, "%s: softmax_lse is NULL", fn);
        if ((rc = check_rows(fn, "q", a->q, a->q_row_stride, a->q_head_stride, a->nheads, d))) return rc;
        if ((rc = check_rows(fn, "o", a->o, a->o_row_stride, a->o_head_stride, a->nheads, d))) return rc;
    }
    if (has_k && (has_q || bwd)) {
        if ((rc = check_rows(fn, "k", a->k, a->k_row_stride, a->k_head_stride, a->nheads_k, d))) return rc;
        if ((rc = check_rows(fn, "v", a->v, a->v_row_stride, a->v_head_stride, a->nheads_k, d))) return rc;
    }
    if (bwd && has_q) {
        if ((rc = check_rows(fn, "dout", a->dout, a->do_row_stride, a->do_head_stride, a->nheads, d))) return rc;
        if ((rc = check_rows(fn, "dq", a->dq, a->dq_row_stride, a->dq_head_stride, a->nheads, d))) return rc;
    }
    if (bwd && has_k) {
        if ((rc = check_rows(fn, "dk", a->dk, a->dk_row_stride, a->dk_head_stride, a->nheads_k, d))) return rc;
        if ((rc = check_rows(fn, "dv", a->dv, a->dv_row_stride, a->dv_head_stride, a->nheads_k, d))) return rc;
    }
    return FA_OK;
}

int grid_ok(const char *fn, int64_t wgs) {
    return wgs < (int64_t)1 << 31 ? FA_OK : set_error(FA_ERR_UNSUPPORTED, "%s: more than 2^31 workgroups", fn);
}

int hip_rc(hipError_t e, const char *fn) {
    return e == hipSuccess ? FA_OK : set_error(FA_ERR_LAUNCH, "%s: HIP error %d (%s)", fn, (int)e, hipGetErrorString(e));
}

int check_paged(const FaPagedArgs *a, const char *fn) {
    if (!a) return set_error(FA_ERR_INVALID_ARGUMENT, "%s: args is NULL", fn);
    int rc = check_sizes(fn, a->batch, a->nheads, a->nheads_k, a->head_dim, a->max_seqlen_q, a->window, a->num_sinks,
                         a->softmax_scale, a->dtype);
    if (rc) return rc;
    if (a->total_q < 0 || a->max_context_len < 0) return set_error(FA_ERR_INVALID_ARGUMENT, "%s: negative length", fn);
    if (a->page_size < 16 || (a->page_size & (a->page_size - 1)))
        return set_error(FA_ERR_UNSUPPORTED, "%s: page_size must be a power of two, 16 or more (got %d)", fn, a->page_size);
    if (a->num_pages < 0 || a->num_seqs < 0 || a->max_blocks < 0)
        return set_error(FA_ERR_INVALID_ARGUMENT, "%s: negative size", fn);
    if ((int64_t)a->max_blocks * a->page_size >= LEN_LIMIT || a->total_q >= LEN_LIMIT ||
        (a->total_q + a->max_seqlen_q) * (a->nheads / a->nheads_k) >= LEN_LIMIT)
        return set_error(FA_ERR_UNSUPPORTED, "%s: 2^30 or more rows or keys", fn);
    if (a->tree_mask && (a->tree_words < 1 || a->tree_words > 4 || a->max_seqlen_q > 64 * a->tree_words))
        return set_error(FA_ERR_UNSUPPORTED, "%s: tree_mask holds 1 to 4 words of 64 tokens, max_seqlen_q of them at least", fn);
    if (a->max_seqlen_q == 0 || a->total_q == 0) return FA_OK;
    if (!a->cu_seqlens_q) return set_error(FA_ERR_INVALID_ARGUMENT, "%s: cu_seqlens_q is NULL", fn);
    if (a->num_seqs > 0 && (!a->context_lens || (a->max_blocks > 0 && !a->block_table)))
        return set_error(FA_ERR_INVALID_ARGUMENT, "%s: block_table or context_lens is NULL", fn);
    if (a->table_stride < a->max_blocks) return set_error(FA_ERR_INVALID_ARGUMENT, "%s: table_stride < max_blocks", fn);
    if (!a->seq_ids && a->batch > a->num_seqs)
        return set_error(FA_ERR_INVALID_ARGUMENT, "%s: batch larger than the block table and no seq_ids", fn);
    if (a->softmax_lse && a->lse_stride < a->max_seqlen_q)
        return set_error(FA_ERR_INVALID_ARGUMENT, "%s: lse_stride < max_seqlen_q", fn);
    if ((rc = check_rows(fn, "q", a->q, a->q_row_stride, a->q_head_stride, a->nheads, a->head_dim))) return rc;
    if ((rc = check_rows(fn, "o", a->o, a->o_row_stride, a->o_head_stride, a->nheads, a->head_dim))) return rc;
    if (a->num_pages > 0) {
        if (!a->k_pages || !a->v_pages || !al16(a->k_pages) || !al16(a->v_pages) || (a->k_page_stride | a->k_row_stride |
            a->k_head_stride | a->v_page_stride | a->v_row_stride | a->v_head_stride) % 8)
            return set_error(FA_ERR_INVALID_ARGUMENT, "%s: k_pages and v_pages must be 16-byte aligned with strides multiple of 8", fn);
        // rows and heads of a page may lie in either order
        for (int64_t s : {a->k_page_stride, a->k_row_stride, a->k_head_stride, a->v_page_stride, a->v_row_stride, a->v_head_stride})
            if (s < 0) return set_error(FA_ERR_INVALID_ARGUMENT, "%s: negative page, row or head stride", fn);
        if (a->k_row_stride < a->head_dim || a->v_row_stride < a->head_dim)
            return set_error(FA_ERR_INVALID_ARGUMENT, "%s: rows of the pages overlap", fn);
        if (a->k_row_stride >= (int64_t)1 << 23 || a->v_row_stride >= (int64_t)1 << 23)
            return set_error(FA_ERR_UNSUPPORTED, "%s: row stride of the pages is 2^23 elements or more", fn);
    }
    return FA_OK;
}

// Shape and split of a paged call. 32 packed rows or fewer (single tokens, small groups): four waves of a
// workgroup take the same rows and every fourth tile; up to 64: two and two; more: 128 rows to a workgroup.
// (Eight waves on 256 rows, four tiles in flight, took 120 us for 64 drafts over 8 caches of 32000 keys where four waves,
// two workgroups to a CU, take 102: all eight wait at each barrier.) The keys are split where that makes the rounds of
// workgroups shorter: steps of a round and 4 more for its start and end, 2 for the join and an eighth for each part.
struct PagedPlan { WinShape shape; int nrb, nsplit; };
PagedPlan plan_paged(const FaPagedArgs *a) {
    PagedPlan p;
    const int64_t rows = (int64_t)a->max_seqlen_q * (a->nheads / a->nheads_k);
    p.shape = rows <= 32 ? WIN_1X4X32 : rows <= 64 ? WIN_2X2X32 : WIN_4X1X64;
    p.nrb = (int)((rows + win_shape_rows(p.shape) - 1) / win_shape_rows(p.shape));
    const int bn = win_shape_keys(p.shape), kg = win_shape_groups(p.shape);
    int64_t keys = (int64_t)a->max_context_len + a->max_seqlen_q;
    const int64_t room = (int64_t)a->max_blocks * a->page_size;
    keys = keys < room ? keys : room;
    if (a->window > 0) {
        const int64_t seen = (int64_t)a->window + a->max_seqlen_q + a->num_sinks + 2 * bn;
        keys = keys < seen ? keys : seen;
    }
    const int64_t tiles = (keys + bn - 1) / bn;
    const int64_t base = (int64_t)p.nrb * a->nheads_k * a->batch;
    // workgroups that a CU holds at once (LDS and registers of the shapes, by head-dim tile)
    const int per_cu = (p.shape == WIN_1X4X32 ? 1 : 2) * (tile_of(a->head_dim) == 128 ? 1 : 2);
    const int64_t slots = (int64_t)cus() * per_cu;
    int64_t want = 1, best = 0;
    for (int64_t n = 1; n <= 128 && (n == 1 || 2 * kg * n <= tiles); ++n) {
        const int64_t rounds = (base * n + slots - 1) / slots, steps = ((tiles + n - 1) / n + kg - 1) / kg;
        const int64_t cost = rounds * (steps + 4) + (n > 1 ? 2 : 0) + n / 8;
        if (n == 1 || cost < best) {
            best = cost;
            want = n;
        }
    }
    p.nsplit = (int)want;
    return p;
}

// The backward's shape, its workspace laid out behind `ws`, and the bytes it takes.
//
// The sinks' rows behind the window get workgroups of their own when a sequence may be longer than two windows:
// shares of 1024 rows (512 where a block of keys itself walks more than 4096 rows, so that they do not add a round of
// their own: 292 us against 311 at 8192 tokens, window 1024, 16 heads on 4; at 2048 tokens, window 256, 12 heads 1024
// rows take 71 us, 512 75), 64 to a head at most and no more than the partial sums' WIN_SINK_BYTES allow.
constexpr int64_t WIN_SINK_BYTES = (int64_t)64 << 20;
WinBwdPlan plan_bwd(const FaWindowArgs *a, WinBwdArgs &w, char *ws, int64_t &bytes) {
    WinBwdPlan p{};
    const int group = a->nheads / a->nheads_k;
    p.max_rows = a->total_q > 0 ? a->max_seqlen_q * group : 0;
    p.max_k = a->total_k > 0 ? a->max_seqlen_k : 0;
    const int64_t window = a->window > 0 && a->window < NO_WINDOW ? a->window : NO_WINDOW;
    w.window = (int)window;
    p.order = order_for((int64_t)a->nheads_k * a->batch, window, p.max_k, a->head_dim);
    w.sinks = a->num_sinks < p.max_k ? a->num_sinks : p.max_k;
    p.fine = takes_fine(a, window, 32 * WIN_DQ_WAVES);
    w.chunks = w.sink_blocks = w.per_chunk = w.slots = 0;
    bytes = a->total_q * a->nheads * (int64_t)sizeof(f32x2);
    bytes = (bytes + 255) / 256 * 256;
    w.ws_rows = (f32x2 *)ws;
    if (w.sinks > 0 && p.max_rows > 0 && p.max_k > 2 * window) {
        const int64_t part = (int64_t)a->batch * a->nheads_k * w.sinks * 2 * tile_of(a->head_dim) * (int64_t)sizeof(float);
        const int64_t share = (window + 32 * WIN_DKV_BLOCKS) * group > 4096 ? 512 : 1024;
        int64_t chunks = (p.max_rows + share - 1) / share;
        const int64_t fit = (WIN_SINK_BYTES / part - 1) / WIN_DKV_BLOCKS;
        chunks = chunks < fit ? chunks : fit;
        chunks = chunks < 1 ? 1 : (chunks > 64 ? 64 : chunks);
        const int64_t per = ((p.max_rows + chunks - 1) / chunks + 31) / 32 * 32;
        w.per_chunk = (int)per;
        w.chunks = (int)((p.max_rows + per - 1) / per);
        w.sink_blocks = (w.sinks + 31) / 32;
        w.slots = w.chunks * WIN_DKV_BLOCKS + 1;
        w.dchunks = Div::of(w.chunks);
        w.dsinkb = Div::of(w.sink_blocks);
        w.ws_part = (float *)(ws + bytes);
        bytes += part * w.slots;
    }
    return p;
}

int64_t paged_bytes(const FaPagedArgs *a, const PagedPlan &p) {
    if (p.nsplit == 1) return 0;
    const int64_t rows = (int64_t)p.nsplit * a->total_q * a->nheads;
    return rows * (tile_of(a->head_dim) + 2) * (int64_t)sizeof(float);
}

}  // namespace
}  // namespace fa

using namespace fa;

extern "C" {

int64_t fa_window_args_size(int what) { return what == 0 ? (int64_t)sizeof(FaWindowArgs) : what == 1 ? (int64_t)sizeof(FaPagedArgs) : -1; }

int fa_window_fwd(const FaWindowArgs *a, void *stream) {
    clear_error();
    int rc = check_window(a, "fa_window_fwd", false);
    if (rc) return rc;
    if (a->max_seqlen_q == 0 || a->total_q == 0) return FA_OK;
    WinFwdArgs w{};
    w.q = (const uint16_t *)a->q; w.k = (const uint16_t *)a->k; w.v = (const uint16_t *)a->v;
    w.o = (uint16_t *)a->o; w.lse = a->softmax_lse;
    w.cu_q = a->cu_seqlens_q; w.cu_k = a->cu_seqlens_k;
    w.q_rs = a->q_row_stride; w.q_hs = a->q_head_stride; w.o_rs = a->o_row_stride; w.o_hs = a->o_head_stride;
    w.k_rs = a->k_row_stride; w.k_hs = a->k_head_stride; w.v_rs = a->v_row_stride; w.v_hs = a->v_head_stride;
    w.total_q = a->total_q; w.total_k = a->total_k;
    w.batch = a->batch; w.nheads = a->nheads; w.nheads_k = a->nheads_k; w.head_dim = a->head_dim;
    w.group = a->nheads / a->nheads_k;
    w.max_q = a->max_seqlen_q;
    w.lse_stride = a->lse_stride;
    w.window = a->window > 0 && a->window < NO_WINDOW ? a->window : NO_WINDOW;
    w.sinks = a->num_sinks;
    w.nrb = (int)(((int64_t)a->max_seqlen_q * w.group + 32 * WIN_FWD_WAVES - 1) / (32 * WIN_FWD_WAVES));
    w.nsplit = 1;
    w.dgroup = Div::of(w.group);
    w.dheads = Div::of(w.nheads_k);
    w.dsplit = Div::of(1);
    w.order = BlockOrder::of(w.nrb, w.nheads_k * w.batch, order_for((int64_t)w.nheads_k * w.batch, w.window, a->max_seqlen_k, a->head_dim));
    w.scale = a->softmax_scale;
    w.fine = takes_fine(a, w.window, 32 * WIN_FWD_WAVES);
    if ((rc = grid_ok("fa_window_fwd", (int64_t)w.nrb * w.nheads_k * w.batch))) return rc;
    hipStream_t s = (hipStream_t)stream;
    hipError_t e;
    switch (tile_of(a->head_dim)) {
        case 32: e = launch_window_fwd<32>(w, a->dtype, false, WIN_4X1X64, s); break;
        case 64: e = launch_window_fwd<64>(w, a->dtype, false, WIN_4X1X64, s); break;
        default: e = launch_window_fwd<128>(w, a->dtype, false, WIN_4X1X64, s); break;
    }
    return hip_rc(e, "fa_window_fwd launch");
}

int64_t fa_window_bwd_workspace(const FaWindowArgs *a) {
    clear_error();
    if (!a) return -set_error(FA_ERR_INVALID_ARGUMENT, "fa_window_bwd_workspace: args is NULL");
    const int rc = check_sizes("fa_window_bwd_workspace", a->batch, a->nheads, a->nheads_k, a->head_dim, a->max_seqlen_q,
                               a->window, a->num_sinks, a->softmax_scale, a->dtype);
    if (rc) return -rc;
    if (a->total_q < 0 || a->total_k < 0 || a->max_seqlen_k < 0 || a->total_q >= LEN_LIMIT || a->total_k >= LEN_LIMIT ||
        (a->total_q + a->total_k + a->max_seqlen_q) * (a->nheads / a->nheads_k) >= LEN_LIMIT)
        return -set_error(FA_ERR_INVALID_ARGUMENT, "fa_window_bwd_workspace: lengths out of range");
    WinBwdArgs w{};
    int64_t bytes;
    plan_bwd(a, w, nullptr, bytes);
    return bytes;
}

int fa_window_bwd(const FaWindowArgs *a, void *stream) {
    clear_error();
    int rc = check_window(a, "fa_window_bwd", true);
    if (rc) return rc;
    WinBwdArgs w{};
    w.q = (const uint16_t *)a->q; w.k = (const uint16_t *)a->k; w.v = (const uint16_t *)a->v;
    w.o = (const uint16_t *)a->o; w.dout = (const uint16_t *)a->dout; w.lse = a->softmax_lse;
    w.dq = (uint16_t *)a->dq; w.dk = (uint16_t *)a->dk; w.dv = (uint16_t *)a->dv;
    w.cu_q = a->cu_seqlens_q; w.cu_k = a->cu_seqlens_k;
    w.q_rs = a->q_row_stride; w.q_hs = a->q_head_stride; w.k_rs = a->k_row_stride; w.k_hs = a->k_head_stride;
    w.v_rs = a->v_row_stride; w.v_hs = a->v_head_stride; w.o_rs = a->o_row_stride; w.o_hs = a->o_head_stride;
    w.do_rs = a->do_row_stride; w.do_hs = a->do_head_stride;
    w.dq_rs = a->dq_row_stride; w.dq_hs = a->dq_head_stride; w.dk_rs = a->dk_row_stride; w.dk_hs = a->dk_head_stride;
    w.dv_rs = a->dv_row_stride; w.dv_hs = a->dv_head_stride;
    w.total_q = a->total_q; w.total_k = a->total_k;
    w.batch = a->batch; w.nheads = a->nheads; w.nheads_k = a->nheads_k; w.head_dim = a->head_dim;
    w.group = a->nheads / a->nheads_k;
    w.dgroup = Div::of(w.group);
    w.dheads = Div::of(w.nheads_k);
    w.max_q = a->max_seqlen_q;
    w.lse_stride = a->lse_stride;
    w.scale = a->softmax_scale;
    int64_t bytes;
    const WinBwdPlan p = plan_bwd(a, w, (char *)a->workspace, bytes);
    if (bytes > 0 && (!a->workspace || !al16(a->workspace) || a->workspace_bytes < bytes))
        return set_error(FA_ERR_INVALID_ARGUMENT, "fa_window_bwd: workspace of %lld bytes needed", (long long)bytes);
    const int64_t most = (int64_t)(p.max_rows > p.max_k ? p.max_rows : p.max_k) / 32 + 1 + (int64_t)w.chunks * w.sink_blocks;
    if ((rc = grid_ok("fa_window_bwd", most * w.nheads_k * w.batch))) return rc;
    if (w.chunks > 0 && (int64_t)w.nheads_k * w.batch > 65535)
        return set_error(FA_ERR_UNSUPPORTED, "fa_window_bwd: batch * nheads_k above 65535");
    hipStream_t s = (hipStream_t)stream;
    hipError_t e;
    switch (tile_of(a->head_dim)) {
        case 32: e = launch_window_bwd<32>(w, a->dtype, p, s); break;
        case 64: e = launch_window_bwd<64>(w, a->dtype, p, s); break;
        default: e = launch_window_bwd<128>(w, a->dtype, p, s); break;
    }
    return hip_rc(e, "fa_window_bwd launch");
}

int64_t fa_paged_workspace(const FaPagedArgs *a) {
    clear_error();
    const int rc = check_paged(a, "fa_paged_workspace");
    if (rc) return -rc;
    if (a->max_seqlen_q == 0 || a->total_q == 0) return 0;
    return paged_bytes(a, plan_paged(a));
}

int fa_paged_fwd(const FaPagedArgs *a, void *stream) {
    clear_error();
    int rc = check_paged(a, "fa_paged_fwd");
    if (rc) return rc;
    if (a->max_seqlen_q == 0 || a->total_q == 0) return FA_OK;
    const PagedPlan p = plan_paged(a);
    const int64_t bytes = paged_bytes(a, p);
    if (bytes > 0 && (!a->workspace || !al16(a->workspace) || a->workspace_bytes < bytes))
        return set_error(FA_ERR_INVALID_ARGUMENT, "fa_paged_fwd: workspace of %lld bytes needed", (long long)bytes);
    WinFwdArgs w{};
    w.q = (const uint16_t *)a->q; w.k = (const uint16_t *)a->k_pages; w.v = (const uint16_t *)a->v_pages;
    w.o = (uint16_t *)a->o; w.lse = a->softmax_lse;
    w.cu_q = a->cu_seqlens_q;
    w.table = a->block_table; w.ctx = a->context_lens; w.seq_ids = a->seq_ids; w.tree = a->tree_mask;
    w.q_rs = a->q_row_stride; w.q_hs = a->q_head_stride; w.o_rs = a->o_row_stride; w.o_hs = a->o_head_stride;
    w.k_ps = a->k_page_stride; w.k_rs = a->k_row_stride; w.k_hs = a->k_head_stride;
    w.v_ps = a->v_page_stride; w.v_rs = a->v_row_stride; w.v_hs = a->v_head_stride;
    w.table_stride = a->table_stride; w.total_q = a->total_q;
    w.batch = a->batch; w.nheads = a->nheads; w.nheads_k = a->nheads_k; w.head_dim = a->head_dim;
    w.group = a->nheads / a->nheads_k;
    w.num_pages = a->num_pages; w.num_seqs = a->num_seqs; w.max_blocks = a->max_blocks;
    w.page_shift = __builtin_ctz(a->page_size);
    w.tree_words = a->tree_words; w.max_q = a->max_seqlen_q; w.lse_stride = a->lse_stride;
    w.window = a->window > 0 && a->window < NO_WINDOW ? a->window : NO_WINDOW;
    w.sinks = a->num_sinks;
    w.nrb = p.nrb; w.nsplit = p.nsplit;
    w.dgroup = Div::of(w.group);
    w.dheads = Div::of(w.nheads_k);
    w.dsplit = Div::of(w.nsplit);
    w.order.blk = Div::of(w.nrb);
    w.scale = a->softmax_scale;
    if (p.nsplit > 1) {
        w.ws_o = (float *)a->workspace;
        w.ws_ml = w.ws_o + (int64_t)p.nsplit * a->total_q * a->nheads * tile_of(a->head_dim);
    }
    if ((rc = grid_ok("fa_paged_fwd", (int64_t)w.nrb * w.nsplit * w.nheads_k * w.batch))) return rc;
    hipStream_t s = (hipStream_t)stream;
    hipError_t e;
    switch (tile_of(a->head_dim)) {
        case 32: e = launch_window_fwd<32>(w, a->dtype, true, p.shape, s); break;
        case 64: e = launch_window_fwd<64>(w, a->dtype, true, p.shape, s); break;
        default: e = launch_window_fwd<128>(w, a->dtype, true, p.shape, s); break;
    }
    return hip_rc(e, "fa_paged_fwd launch");
}

}  // extern "C"
