"""Causal attention with a sliding window and sinks, var-len, with grouped heads, forward and backward.

The windowed relative of `flash_attn_interface.flash_attn_unpadded_func`, same layouts and argument order. A query
row i of a sequence with sq rows and sk keys stands at position p = i + sk - sq (aligned to the end of the keys,
so a chunk of a prompt sees what is already there) and sees key j when

    j <= p   and   (j > p - window_size   or   j < num_sinks).

A row with p < 0 sees nothing: its output and its gradient are 0, its lse -inf. Rows of q, k and v behind the last
sequence belong to none: output and gradients are 0 there.

Scores, softmax statistics and sums are fp32; the probabilities are rounded to the input type for the product with
v (and dS for those with q and k), as they are in the other kernels; small calls with short windows take them in two such
parts, so that the output's own rounding is all that is left. Results do not depend on the order in which
workgroups run: there are no atomics, gradients of shared key/value heads included.
"""
from flash_attn import flash_attn_hip as _hip


def _binding():
    if _hip._C is None:
        raise ImportError("the windowed and paged operators need the compiled binding flash_attn/_fa_C.so: build it "
                          "with `python hazyresearch_flash-attention_amd/build.py` (and leave FA_HIP_LIB unset)")
    return _hip._C


def _window(window_size, num_sinks):
    """(window, sinks) as the C ABI takes them: 0 for no window."""
    if window_size is not None and window_size < 1:
        raise RuntimeError(f"window_size must be None or at least 1, got {window_size}")
    if num_sinks < 0:
        raise RuntimeError(f"num_sinks must be at least 0, got {num_sinks}")
    return 0 if window_size is None else min(int(window_size), 2 ** 30), min(int(num_sinks), 2 ** 30)


def flash_window_attn_unpadded_func(q, k, v, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k,
                                    window_size=None, num_sinks=0, softmax_scale=None, return_lse=False):
    """Windowed attention of q (total_q, nheads, headdim) over k, v (total_k, nheads_k, headdim), fp16 or bf16.

    nheads is a multiple of nheads_k; headdim a multiple of 8, at most 128. cu_seqlens_q / cu_seqlens_k: (batch + 1,)
    int32 on the device; max_seqlen_q / max_seqlen_k bound the sequences' lengths. window_size: keys that a query
    sees, its own among them (None: all up to its own). num_sinks: first keys that every later query sees.
    softmax_scale defaults to headdim**-0.5.

    Returns out (total_q, nheads, headdim), or (out, lse) with return_lse: lse (batch, nheads,
    round16(max_seqlen_q)) fp32, natural logarithm, without a gradient; entries past a sequence's end are unset.

    An infinity or NaN reaches the results of what sees it and nothing else, forward and backward (rows whose tiles
    hold one are computed again key by key, which is slow).
    """
    window, sinks = _window(window_size, num_sinks)
    out, lse = _binding().window_attn(q, k, v, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k, window, sinks,
                                      softmax_scale)
    return (out, lse) if return_lse else out


def flash_window_attn_unpadded_kvpacked_func(q, kv, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k,
                                             window_size=None, num_sinks=0, softmax_scale=None, return_lse=False):
    """`flash_window_attn_unpadded_func` of q (total_q, nheads, headdim) over packed kv (total_k, 2, nheads_k, headdim)."""
    window, sinks = _window(window_size, num_sinks)
    out, lse = _binding().window_attn_kv(q, kv, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k, window, sinks,
                                         softmax_scale)
    return (out, lse) if return_lse else out


def flash_window_attn_unpadded_qkvpacked_func(qkv, cu_seqlens, max_seqlen, window_size=None, num_sinks=0,
                                              softmax_scale=None, return_lse=False):
    """`flash_window_attn_unpadded_func` of packed qkv (total, 3, nheads, headdim)."""
    window, sinks = _window(window_size, num_sinks)
    out, lse = _binding().window_attn_qkv(qkv, cu_seqlens, max_seqlen, window, sinks, softmax_scale)
    return (out, lse) if return_lse else out
