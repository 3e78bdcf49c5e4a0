// fa_torch_window.cpp — the windowed, paged and cache entry points of the compiled binding (module
// flash_attn._fa_C): tensor checks, outputs and workspaces from torch's allocator on the current stream, the call
// into the C ABI (include/fa_window_hip.h, include/fa_cache_hip.h), and the windowed attention's autograd function.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/utils/pybind.h>

#include <cmath>
#include <tuple>

#include "fa_cache_hip.h"
#include "fa_window_hip.h"

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

int dtype_of(const at::Tensor &t) {
    if (t.scalar_type() == at::kHalf) return FA_DTYPE_FP16;
    if (t.scalar_type() == at::kBFloat16) return FA_DTYPE_BF16;
    TORCH_CHECK(false, "FlashAttention only supports fp16 and bf16, got ", t.scalar_type());
}

// A (rows, heads, d) tensor as the kernels take it: 16-byte rows that do not overlap. Others (broadcast, overlapping
// or transposed rows, odd offsets) are copied.
at::Tensor rows(const at::Tensor &t) {
    const int64_t h = t.size(1), d = t.size(2);
    const bool ok = t.stride(2) == 1 && t.stride(0) >= (h - 1) * t.stride(1) + d && (h <= 1 || t.stride(1) >= d) &&
                    t.stride(0) % 8 == 0 && t.stride(1) % 8 == 0 && t.stride(0) < (1 << 23) &&
                    ((uintptr_t)t.data_ptr() & 15) == 0;
    return ok || t.numel() == 0 ? t : t.clone(at::MemoryFormat::Contiguous);
}

void check_i32(const at::Tensor &t, const char *name, const at::Tensor &like) {
    TORCH_CHECK(t.scalar_type() == at::kInt, name, " must be int32");
    TORCH_CHECK(t.device() == like.device(), name, " must be on the device ", like.device());
}

void check_cu(const at::Tensor &t, const char *name, const at::Tensor &like) {
    check_i32(t, name, like);
    TORCH_CHECK(t.dim() == 1 && t.is_contiguous(), name, " must be contiguous and 1-D");
}

void check_heads(int64_t nheads, int64_t nheads_k, int64_t d) {
    TORCH_CHECK(d > 0 && d % 8 == 0 && d <= 128, "head_size must be a multiple of 8 and <= 128");
    TORCH_CHECK(nheads > 0 && nheads_k > 0 && nheads % nheads_k == 0,
                "the heads of q must be a multiple of the heads of k and v (got ", nheads, " and ", nheads_k, ")");
}

void check_int(int64_t x, const char *name) {
    TORCH_CHECK(x >= 0 && x < (1ll << 31), name, " must be in [0, 2^31)");
}

hipStream_t stream_of(const at::Tensor &t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

void check_rc(int rc, const char *what) { TORCH_CHECK(rc == 0, what, " failed (code ", rc, "): ", fa_last_error()); }

int64_t round16(int64_t x) { return (x + 15) / 16 * 16; }

bool wants_grad(const at::Tensor &t) { return at::GradMode::is_enabled() && t.defined() && t.requires_grad(); }

// ------------------------------------------------------------------------------------ windowed attention
FaWindowArgs window_args(const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const at::Tensor &o,
                         const at::Tensor &lse, const at::Tensor &cu_q, const at::Tensor &cu_k, int64_t max_q,
                         int64_t max_k, int64_t window, int64_t sinks, double scale) {
    FaWindowArgs a{};
    a.q = q.data_ptr();
    a.k = k.data_ptr();
    a.v = v.data_ptr();
    a.o = o.data_ptr();
    a.softmax_lse = lse.data_ptr<float>();
    a.cu_seqlens_q = cu_q.data_ptr<int32_t>();
    a.cu_seqlens_k = cu_k.data_ptr<int32_t>();
    a.q_row_stride = q.stride(0); a.q_head_stride = q.stride(1);
    a.k_row_stride = k.stride(0); a.k_head_stride = k.stride(1);
    a.v_row_stride = v.stride(0); a.v_head_stride = v.stride(1);
    a.o_row_stride = o.stride(0); a.o_head_stride = o.stride(1);
    a.total_q = q.size(0);
    a.total_k = k.size(0);
    a.batch = (int32_t)(cu_q.numel() - 1);
    a.nheads = (int32_t)q.size(1);
    a.nheads_k = (int32_t)k.size(1);
    a.head_dim = (int32_t)q.size(2);
    a.max_seqlen_q = (int32_t)max_q;
    a.max_seqlen_k = (int32_t)max_k;
    a.lse_stride = (int32_t)lse.size(2);
    a.window = (int32_t)window;
    a.num_sinks = (int32_t)sinks;
    a.softmax_scale = (float)scale;
    a.dtype = dtype_of(q);
    return a;
}

void check_window(const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const at::Tensor &cu_q,
                  const at::Tensor &cu_k, int64_t max_q, int64_t max_k, int64_t window, int64_t sinks) {
    TORCH_CHECK(q.is_cuda(), "all tensors must be on the GPU");
    dtype_of(q);
    TORCH_CHECK(q.dim() == 3 && k.dim() == 3 && v.dim() == 3, "q, k, v must be (total, nheads, headdim)");
    TORCH_CHECK(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(), "q, k, v must have the same dtype");
    TORCH_CHECK(k.device() == q.device() && v.device() == q.device(), "q, k, v must be on the same device");
    check_cu(cu_q, "cu_seqlens_q", q);
    check_cu(cu_k, "cu_seqlens_k", q);
    TORCH_CHECK(cu_q.numel() >= 2, "batch_size must be positive");
    TORCH_CHECK(cu_k.numel() == cu_q.numel(), "cu_seqlens_k must have shape (batch_size + 1)");
    check_heads(q.size(1), k.size(1), q.size(2));
    TORCH_CHECK(k.size(2) == q.size(2) && v.sizes() == k.sizes(), "k, v must have shape (total_k, nheads_k, headdim)");
    check_int(max_q, "max_seqlen_q");
    check_int(max_k, "max_seqlen_k");
    check_int(window, "window_size");
    check_int(sinks, "num_sinks");
}

std::vector<at::Tensor> window_fwd(const at::Tensor &q_, const at::Tensor &k_, const at::Tensor &v_,
                                   const at::Tensor &cu_q, const at::Tensor &cu_k, int64_t max_q, int64_t max_k,
                                   int64_t window, int64_t sinks, double scale) {
    check_window(q_, k_, v_, cu_q, cu_k, max_q, max_k, window, sinks);
    c10::DeviceGuard guard(q_.device());
    const at::Tensor q = rows(q_), k = rows(k_), v = rows(v_);
    at::Tensor o = at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
    at::Tensor lse = at::empty({cu_q.numel() - 1, q.size(1), std::max<int64_t>(round16(max_q), 16)}, q.options().dtype(at::kFloat));
    if (max_q == 0) o.zero_();      // no row of any sequence: nothing is launched
    const FaWindowArgs a = window_args(q, k, v, o, lse, cu_q, cu_k, max_q, max_k, window, sinks, scale);
    check_rc(fa_window_fwd(&a, stream_of(q)), "fa_window_fwd");
    return {o, lse};
}

// Writes dq, dk, dv (whole tensors or views of a packed one).
void window_bwd(const at::Tensor &dout_, const at::Tensor &q_, const at::Tensor &k_, const at::Tensor &v_,
                const at::Tensor &o, const at::Tensor &lse, at::Tensor dq, at::Tensor dk, at::Tensor dv,
                const at::Tensor &cu_q, const at::Tensor &cu_k, int64_t max_q, int64_t max_k, int64_t window,
                int64_t sinks, double scale) {
    TORCH_CHECK(dout_.sizes() == q_.sizes() && dout_.scalar_type() == q_.scalar_type() && dout_.device() == q_.device(),
                "dout must have the shape, dtype and device of q");
    c10::DeviceGuard guard(q_.device());
    const at::Tensor q = rows(q_), k = rows(k_), v = rows(v_), dout = rows(dout_);
    if (max_q == 0) dq.zero_();
    if (max_k == 0) {
        dk.zero_();
        dv.zero_();
    }
    FaWindowArgs a = window_args(q, k, v, o, lse, cu_q, cu_k, max_q, max_k, window, sinks, scale);
    a.dout = dout.data_ptr();
    a.dq = dq.data_ptr();
    a.dk = dk.data_ptr();
    a.dv = dv.data_ptr();
    a.do_row_stride = dout.stride(0); a.do_head_stride = dout.stride(1);
    a.dq_row_stride = dq.stride(0); a.dq_head_stride = dq.stride(1);
    a.dk_row_stride = dk.stride(0); a.dk_head_stride = dk.stride(1);
    a.dv_row_stride = dv.stride(0); a.dv_head_stride = dv.stride(1);
    const int64_t bytes = fa_window_bwd_workspace(&a);
    check_rc(bytes < 0 ? (int)-bytes : 0, "fa_window_bwd_workspace");
    at::Tensor ws;
    if (bytes > 0) {
        ws = at::empty({bytes}, q.options().dtype(at::kByte));
        a.workspace = ws.data_ptr();
        a.workspace_bytes = bytes;
    }
    check_rc(fa_window_bwd(&a, stream_of(q)), "fa_window_bwd");
}

at::Tensor dense_like(const at::Tensor &t) { return at::empty(t.sizes(), t.options().memory_format(at::MemoryFormat::Contiguous)); }

struct WindowCfg {
    int64_t max_q, max_k, window, sinks;
    double scale;
    void save(AutogradContext *ctx) const {
        ctx->saved_data["mq"] = max_q;
        ctx->saved_data["mk"] = max_k;
        ctx->saved_data["w"] = window;
        ctx->saved_data["n"] = sinks;
        ctx->saved_data["sc"] = scale;
    }
    static WindowCfg load(AutogradContext *ctx) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "the windowed attention has no second derivative (create_graph=True)");
        return {ctx->saved_data["mq"].toInt(), ctx->saved_data["mk"].toInt(), ctx->saved_data["w"].toInt(),
                ctx->saved_data["n"].toInt(), ctx->saved_data["sc"].toDouble()};
    }
};

struct WindowAttnFn : public torch::autograd::Function<WindowAttnFn> {
    static variable_list forward(AutogradContext *ctx, const at::Tensor &q, const at::Tensor &k, const at::Tensor &v,
                                 const at::Tensor &cu_q, const at::Tensor &cu_k, int64_t max_q, int64_t max_k,
                                 int64_t window, int64_t sinks, double scale) {
        auto r = window_fwd(q, k, v, cu_q, cu_k, max_q, max_k, window, sinks, scale);
        ctx->save_for_backward({q, k, v, r[0], r[1], cu_q, cu_k});
        ctx->mark_non_differentiable({r[1]});
        WindowCfg{max_q, max_k, window, sinks, scale}.save(ctx);
        return {r[0], r[1]};
    }
    static variable_list backward(AutogradContext *ctx, variable_list g) {
        const WindowCfg c = WindowCfg::load(ctx);
        at::Tensor n;
        if (!g[0].defined()) return {n, n, n, n, n, n, n, n, n, n};
        auto t = ctx->get_saved_variables();
        c10::DeviceGuard guard(t[0].device());
        at::Tensor dq = dense_like(t[0]), dk = dense_like(t[1]), dv = dense_like(t[2]);
        window_bwd(g[0], t[0], t[1], t[2], t[3], t[4], dq, dk, dv, t[5], t[6], c.max_q, c.max_k, c.window, c.sinks, c.scale);
        return {dq, dk, dv, n, n, n, n, n, n, n};
    }
};

// kv (total_k, 2, nheads_k, headdim): dkv written whole
struct WindowAttnKVFn : public torch::autograd::Function<WindowAttnKVFn> {
    static variable_list forward(AutogradContext *ctx, const at::Tensor &q, const at::Tensor &kv, const at::Tensor &cu_q,
                                 const at::Tensor &cu_k, int64_t max_q, int64_t max_k, int64_t window, int64_t sinks,
                                 double scale) {
        auto r = window_fwd(q, kv.select(1, 0), kv.select(1, 1), cu_q, cu_k, max_q, max_k, window, sinks, scale);
        ctx->save_for_backward({q, kv, r[0], r[1], cu_q, cu_k});
        ctx->mark_non_differentiable({r[1]});
        WindowCfg{max_q, max_k, window, sinks, scale}.save(ctx);
        return {r[0], r[1]};
    }
    static variable_list backward(AutogradContext *ctx, variable_list g) {
        const WindowCfg c = WindowCfg::load(ctx);
        at::Tensor n;
        if (!g[0].defined()) return {n, n, n, n, n, n, n, n, n};
        auto t = ctx->get_saved_variables();
        c10::DeviceGuard guard(t[0].device());
        at::Tensor dq = dense_like(t[0]), dkv = dense_like(t[1]);
        window_bwd(g[0], t[0], t[1].select(1, 0), t[1].select(1, 1), t[2], t[3], dq, dkv.select(1, 0), dkv.select(1, 1),
                   t[4], t[5], c.max_q, c.max_k, c.window, c.sinks, c.scale);
        return {dq, dkv, n, n, n, n, n, n, n};
    }
};

// qkv (total, 3, nheads, headdim): dqkv written whole
struct WindowAttnQKVFn : public torch::autograd::Function<WindowAttnQKVFn> {
    static variable_list forward(AutogradContext *ctx, const at::Tensor &qkv, const at::Tensor &cu, int64_t max_s,
                                 int64_t window, int64_t sinks, double scale) {
        auto r = window_fwd(qkv.select(1, 0), qkv.select(1, 1), qkv.select(1, 2), cu, cu, max_s, max_s, window, sinks, scale);
        ctx->save_for_backward({qkv, r[0], r[1], cu});
        ctx->mark_non_differentiable({r[1]});
        WindowCfg{max_s, max_s, window, sinks, scale}.save(ctx);
        return {r[0], r[1]};
    }
    static variable_list backward(AutogradContext *ctx, variable_list g) {
        const WindowCfg c = WindowCfg::load(ctx);
        at::Tensor n;
        if (!g[0].defined()) return {n, n, n, n, n, n};
        auto t = ctx->get_saved_variables();
        c10::DeviceGuard guard(t[0].device());
        at::Tensor d = dense_like(t[0]);
        window_bwd(g[0], t[0].select(1, 0), t[0].select(1, 1), t[0].select(1, 2), t[1], t[2], d.select(1, 0), d.select(1, 1),
                   d.select(1, 2), t[3], t[3], c.max_q, c.max_k, c.window, c.sinks, c.scale);
        return {d, n, n, n, n, n};
    }
};

std::vector<at::Tensor> window_attn_kv(const at::Tensor &q, const at::Tensor &kv, const at::Tensor &cu_q, const at::Tensor &cu_k,
                                       int64_t max_q, int64_t max_k, int64_t window, int64_t sinks,
                                       c10::optional<double> scale_opt) {
    TORCH_CHECK(q.dim() == 3, "q must be (total_q, nheads, headdim)");
    TORCH_CHECK(kv.dim() == 4 && kv.size(1) == 2, "kv must be (total_k, 2, nheads, headdim)");
    const double scale = scale_opt ? *scale_opt : 1.0 / std::sqrt((double)q.size(2));
    if (!wants_grad(q) && !wants_grad(kv))
        return window_fwd(q, kv.select(1, 0), kv.select(1, 1), cu_q, cu_k, max_q, max_k, window, sinks, scale);
    return WindowAttnKVFn::apply(q, kv, cu_q, cu_k, max_q, max_k, window, sinks, scale);
}

std::vector<at::Tensor> window_attn_qkv(const at::Tensor &qkv, const at::Tensor &cu, int64_t max_s, int64_t window,
                                        int64_t sinks, c10::optional<double> scale_opt) {
    TORCH_CHECK(qkv.dim() == 4 && qkv.size(1) == 3, "qkv must be (total, 3, nheads, headdim)");
    const double scale = scale_opt ? *scale_opt : 1.0 / std::sqrt((double)qkv.size(3));
    if (!wants_grad(qkv))
        return window_fwd(qkv.select(1, 0), qkv.select(1, 1), qkv.select(1, 2), cu, cu, max_s, max_s, window, sinks, scale);
    return WindowAttnQKVFn::apply(qkv, cu, max_s, window, sinks, scale);
}

std::vector<at::Tensor> window_attn(const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const at::Tensor &cu_q,
                                    const at::Tensor &cu_k, int64_t max_q, int64_t max_k, int64_t window, int64_t sinks,
                                    c10::optional<double> scale_opt) {
    TORCH_CHECK(q.dim() == 3, "q, k, v must be (total, nheads, headdim)");
    const double scale = scale_opt ? *scale_opt : 1.0 / std::sqrt((double)q.size(2));
    if (!wants_grad(q) && !wants_grad(k) && !wants_grad(v))
        return window_fwd(q, k, v, cu_q, cu_k, max_q, max_k, window, sinks, scale);
    return WindowAttnFn::apply(q, k, v, cu_q, cu_k, max_q, max_k, window, sinks, scale);
}

// ------------------------------------------------------------------------------------ paged attention
std::vector<at::Tensor> paged_attn(const at::Tensor &q_, const at::Tensor &kp, const at::Tensor &vp,
                                   const at::Tensor &table, const at::Tensor &context, const at::Tensor &cu_q,
                                   int64_t max_q, c10::optional<int64_t> max_context, const c10::optional<at::Tensor> &tree,
                                   int64_t window, int64_t sinks, const c10::optional<at::Tensor> &seq_ids,
                                   c10::optional<double> scale_opt, bool want_lse) {
    TORCH_CHECK(q_.is_cuda(), "all tensors must be on the GPU");
    dtype_of(q_);
    TORCH_CHECK(q_.dim() == 3, "q must be (total_q, nheads, headdim)");
    TORCH_CHECK(kp.dim() == 4 && vp.dim() == 4, "k_pages, v_pages must be (num_pages, page_size, nheads_k, headdim)");
    TORCH_CHECK(kp.scalar_type() == q_.scalar_type() && vp.scalar_type() == q_.scalar_type(), "q and the pages must have the same dtype");
    TORCH_CHECK(kp.device() == q_.device() && vp.device() == q_.device(), "q and the pages must be on the same device");
    TORCH_CHECK(!wants_grad(q_) && !wants_grad(kp) && !wants_grad(vp),
                "flash_paged_attn_func has no backward: call it under torch.no_grad() or on detached tensors");
    check_heads(q_.size(1), kp.size(2), q_.size(2));
    TORCH_CHECK(kp.size(3) == q_.size(2) && vp.sizes() == kp.sizes(), "k_pages, v_pages must have shape (num_pages, page_size, nheads_k, headdim)");
    TORCH_CHECK(kp.stride(3) == 1 && vp.stride(3) == 1, "last dimension of the pages must be contiguous");
    check_i32(table, "block_table", q_);
    check_i32(context, "context_lens", q_);
    check_cu(cu_q, "cu_seqlens_q", q_);
    TORCH_CHECK(table.dim() == 2 && (table.size(1) <= 1 || table.stride(1) == 1), "block_table must be (num_seqs, max_blocks) with contiguous rows");
    TORCH_CHECK(context.dim() == 1 && context.is_contiguous() && context.size(0) == table.size(0), "context_lens must be (num_seqs), contiguous");
    TORCH_CHECK(cu_q.numel() >= 2, "batch_size must be positive");
    const int64_t batch = cu_q.numel() - 1, page = kp.size(1);
    if (seq_ids) {
        check_cu(*seq_ids, "seq_ids", q_);
        TORCH_CHECK(seq_ids->numel() == batch, "seq_ids must have shape (batch_size)");
    } else {
        TORCH_CHECK(table.size(0) == batch, "block_table must have batch_size rows unless seq_ids is given");
    }
    if (tree) {
        TORCH_CHECK(tree->scalar_type() == at::kLong && tree->device() == q_.device(), "tree_mask must be int64 on the device of q");
        TORCH_CHECK(tree->dim() == 2 && tree->is_contiguous() && tree->size(0) == q_.size(0), "tree_mask must be (total_q, words), contiguous");
        TORCH_CHECK(tree->size(1) >= 1 && tree->size(1) <= 4 && max_q <= 64 * tree->size(1),
                    "tree_mask holds 1 to 4 words of 64 tokens, max_seqlen_q of them at least");
    }
    check_int(max_q, "max_seqlen_q");
    check_int(window, "window_size");
    check_int(sinks, "num_sinks");
    check_int(kp.size(0), "num_pages");
    check_int(table.size(1) * page, "the block table's tokens");
    if (max_context) check_int(*max_context, "max_context_len");

    c10::DeviceGuard guard(q_.device());
    const at::Tensor q = rows(q_);
    at::Tensor o = at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
    at::Tensor lse;
    if (want_lse) lse = at::empty({batch, q.size(1), std::max<int64_t>(round16(max_q), 16)}, q.options().dtype(at::kFloat));
    if (max_q == 0) o.zero_();
    FaPagedArgs a{};
    a.q = q.data_ptr();
    a.o = o.data_ptr();
    a.softmax_lse = want_lse ? lse.data_ptr<float>() : nullptr;
    a.k_pages = kp.data_ptr();
    a.v_pages = vp.data_ptr();
    a.block_table = table.data_ptr<int32_t>();
    a.context_lens = context.data_ptr<int32_t>();
    a.seq_ids = seq_ids ? seq_ids->data_ptr<int32_t>() : nullptr;
    a.cu_seqlens_q = cu_q.data_ptr<int32_t>();
    a.tree_mask = tree ? reinterpret_cast<const uint64_t *>(tree->data_ptr<int64_t>()) : nullptr;
    a.q_row_stride = q.stride(0); a.q_head_stride = q.stride(1);
    a.o_row_stride = o.stride(0); a.o_head_stride = o.stride(1);
    a.k_page_stride = kp.stride(0); a.k_row_stride = kp.stride(1); a.k_head_stride = kp.stride(2);
    a.v_page_stride = vp.stride(0); a.v_row_stride = vp.stride(1); a.v_head_stride = vp.stride(2);
    a.table_stride = table.size(0) > 1 ? table.stride(0) : std::max<int64_t>(table.size(1), table.stride(0));
    a.total_q = q.size(0);
    a.batch = (int32_t)batch;
    a.nheads = (int32_t)q.size(1);
    a.nheads_k = (int32_t)kp.size(2);
    a.head_dim = (int32_t)q.size(2);
    a.num_pages = (int32_t)kp.size(0);
    a.page_size = (int32_t)page;
    a.num_seqs = (int32_t)table.size(0);
    a.max_blocks = (int32_t)table.size(1);
    a.max_seqlen_q = (int32_t)max_q;
    a.max_context_len = (int32_t)(max_context ? *max_context : table.size(1) * page);
    a.tree_words = tree ? (int32_t)tree->size(1) : 0;
    a.lse_stride = want_lse ? (int32_t)lse.size(2) : 0;
    a.window = (int32_t)window;
    a.num_sinks = (int32_t)sinks;
    a.softmax_scale = (float)(scale_opt ? *scale_opt : 1.0 / std::sqrt((double)q.size(2)));
    a.dtype = dtype_of(q);
    const int64_t bytes = fa_paged_workspace(&a);
    check_rc(bytes < 0 ? (int)-bytes : 0, "fa_paged_workspace");
    at::Tensor ws;
    if (bytes > 0) {
        ws = at::empty({bytes}, q.options().dtype(at::kByte));
        a.workspace = ws.data_ptr();
        a.workspace_bytes = bytes;
    }
    check_rc(fa_paged_fwd(&a, stream_of(q)), "fa_paged_fwd");
    if (want_lse) return {o, lse};
    return {o};
}

// ------------------------------------------------------------------------------------ the paged cache
// The cache's tensors, checked once when the Python object is made; the object keeps them alive.
struct Cache {
    at::Tensor k, v, table, seqlens, nblocks, refcount, status, scratch;
    FaCache c{};

    Cache(at::Tensor k_, at::Tensor v_, at::Tensor table_, at::Tensor seqlens_, at::Tensor nblocks_, at::Tensor refcount_,
          at::Tensor status_, int64_t window, int64_t sinks)
        : k(k_), v(v_), table(table_), seqlens(seqlens_), nblocks(nblocks_), refcount(refcount_), status(status_) {
        TORCH_CHECK(k.is_cuda(), "the cache must be on the GPU");
        dtype_of(k);
        TORCH_CHECK(k.dim() == 5 && k.is_contiguous() && v.is_contiguous() && v.sizes() == k.sizes() && v.dtype() == k.dtype() && v.device() == k.device(),
                    "k, v must be (layers, num_pages, page_size, nheads, headdim), contiguous");
        for (const at::Tensor *t : {&table, &seqlens, &nblocks, &refcount, &status}) {
            check_i32(*t, "the cache's tables", k);
            TORCH_CHECK(t->is_contiguous(), "the cache's tables must be contiguous");
        }
        for (int i = 0; i < 5; ++i) check_int(k.size(i), "a size of the cache");
        check_int(window, "window_size");
        check_int(sinks, "num_sinks");
        TORCH_CHECK(table.dim() == 2 && seqlens.numel() == table.size(0) && nblocks.numel() == table.size(0) &&
                        refcount.numel() == k.size(1) && status.numel() == 1, "the cache's tables do not fit each other");
        c10::DeviceGuard guard(k.device());
        scratch = at::empty({fa_cache_scratch_words((int32_t)k.size(1))}, table.options());
        c.k_pages = k.data_ptr();
        c.v_pages = v.data_ptr();
        c.block_table = table.data_ptr<int32_t>();
        c.seqlens = seqlens.data_ptr<int32_t>();
        c.nblocks = nblocks.data_ptr<int32_t>();
        c.refcount = refcount.data_ptr<int32_t>();
        c.status = status.data_ptr<int32_t>();
        c.scratch = scratch.data_ptr<int32_t>();
        c.layers = (int32_t)k.size(0);
        c.num_pages = (int32_t)k.size(1);
        c.page_size = (int32_t)k.size(2);
        c.nheads = (int32_t)k.size(3);
        c.head_dim = (int32_t)k.size(4);
        c.max_seqs = (int32_t)table.size(0);
        c.max_blocks = (int32_t)table.size(1);
        c.window = (int32_t)window;
        c.num_sinks = (int32_t)sinks;
        check_rc(fa_cache_truncate(&c, nullptr, 0, nullptr, nullptr), "the cache");   // no slots: the checks alone
    }

    const int32_t *ints(const at::Tensor &t, int64_t n, const char *name) const {
        check_i32(t, name, k);
        TORCH_CHECK(t.dim() == 1 && t.is_contiguous() && t.numel() == n, name, " must be a contiguous int32 vector, one entry for each slot");
        return t.data_ptr<int32_t>();
    }
    int32_t count_of(const at::Tensor &slots) const {
        TORCH_CHECK(slots.numel() <= FA_CACHE_MAX_SLOTS, "at most ", (int)FA_CACHE_MAX_SLOTS, " slots a call");
        return (int32_t)slots.numel();
    }

    void reserve(const at::Tensor &slots, int64_t count) {
        c10::DeviceGuard guard(k.device());
        check_int(count, "count");
        check_rc(fa_cache_reserve(&c, ints(slots, slots.numel(), "slots"), count_of(slots), nullptr, (int32_t)count, stream_of(k)), "fa_cache_reserve");
    }
    void reserve_each(const at::Tensor &slots, const at::Tensor &counts) {
        c10::DeviceGuard guard(k.device());
        check_rc(fa_cache_reserve(&c, ints(slots, slots.numel(), "slots"), count_of(slots), ints(counts, slots.numel(), "counts"), 0, stream_of(k)), "fa_cache_reserve");
    }
    void write(int64_t layer, const at::Tensor &slots, const at::Tensor &kn, const at::Tensor &vn, const at::Tensor &cu, int64_t max_seqlen) {
        c10::DeviceGuard guard(k.device());
        for (const at::Tensor *t : {&kn, &vn})
            TORCH_CHECK(t->dim() == 3 && t->scalar_type() == k.scalar_type() && t->device() == k.device() &&
                            t->size(1) == k.size(3) && t->size(2) == k.size(4),
                        "k, v must be (total, nheads, headdim) in the cache's dtype, heads and device");
        TORCH_CHECK(kn.size(0) == vn.size(0), "k and v must have the same number of rows");
        check_int(max_seqlen, "max_seqlen");
        check_int(layer, "layer");
        const at::Tensor kr = rows(kn), vr = rows(vn);
        check_rc(fa_cache_write(&c, (int32_t)layer, ints(slots, slots.numel(), "slots"), count_of(slots), kr.data_ptr(), kr.stride(0),
                                kr.stride(1), vr.data_ptr(), vr.stride(0), vr.stride(1), ints(cu, slots.numel() + 1, "cu_seqlens"),
                                kr.size(0), (int32_t)max_seqlen, stream_of(k)), "fa_cache_write");
    }
    void compact(const at::Tensor &slots, const at::Tensor &keep, const at::Tensor &counts) {
        c10::DeviceGuard guard(k.device());
        check_i32(keep, "keep", k);
        TORCH_CHECK(keep.dim() == 2 && keep.size(0) == slots.numel() && (keep.size(1) <= 1 || keep.stride(1) == 1), "keep must be (slots, max_keep) with contiguous rows");
        check_int(keep.size(1), "max_keep");
        check_rc(fa_cache_compact(&c, ints(slots, slots.numel(), "slots"), count_of(slots), keep.data_ptr<int32_t>(),
                                  std::max<int64_t>(keep.stride(0), keep.size(1)), (int32_t)keep.size(1),
                                  ints(counts, slots.numel(), "counts"), stream_of(k)), "fa_cache_compact");
    }
    void fork(const at::Tensor &parents, const at::Tensor &children) {
        c10::DeviceGuard guard(k.device());
        check_rc(fa_cache_fork(&c, ints(parents, parents.numel(), "parents"), ints(children, parents.numel(), "children"), count_of(parents), stream_of(k)), "fa_cache_fork");
    }
    void truncate(const at::Tensor &slots, const at::Tensor &lens) {
        c10::DeviceGuard guard(k.device());
        check_rc(fa_cache_truncate(&c, ints(slots, slots.numel(), "slots"), count_of(slots), ints(lens, slots.numel(), "lens"), stream_of(k)), "fa_cache_truncate");
    }
    void free(const at::Tensor &slots) {
        c10::DeviceGuard guard(k.device());
        check_rc(fa_cache_truncate(&c, ints(slots, slots.numel(), "slots"), count_of(slots), nullptr, stream_of(k)), "fa_cache_truncate");
    }
    void evict(const at::Tensor &slots) {
        c10::DeviceGuard guard(k.device());
        check_rc(fa_cache_evict(&c, ints(slots, slots.numel(), "slots"), count_of(slots), stream_of(k)), "fa_cache_evict");
    }
};

}  // namespace

void bind_window(pybind11::module &m) {
    m.def("window_attn", &window_attn);
    m.def("window_attn_kv", &window_attn_kv);
    m.def("window_attn_qkv", &window_attn_qkv);
    m.def("paged_attn", &paged_attn);
    pybind11::class_<Cache>(m, "PagedCache")
        .def(pybind11::init<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, int64_t, int64_t>())
        .def("reserve", &Cache::reserve)
        .def("reserve_each", &Cache::reserve_each)
        .def("write", &Cache::write)
        .def("compact", &Cache::compact)
        .def("fork", &Cache::fork)
        .def("truncate", &Cache::truncate)
        .def("free", &Cache::free)
        .def("evict", &Cache::evict);
}
