"""Attention of new tokens over a key/value cache held in pages: one token a sequence, a chunk, or a tree of drafted
tokens, with the window and sinks of `flash_window_attn_interface`. Forward only.

Key j of a sequence lies in row j % page_size of page block_table[seq, j // page_size]. The new tokens' keys are in
the pages already (`paged_kv_cache.PagedKVCache.write`): the keys of a sequence with sq new tokens are 0 ..
context_len + sq - 1. Without a tree new token i stands at position context_len + i.

A tree is given as bits: row i of `tree_mask` names the new tokens of its sequence that token i sees, itself and its
ancestors (bit j % 64 of word j // 64 for token j); `pack_tree_mask` makes them from truth values and `tree_from_parents`
from each token's parent. A token's position is context_len + (its bits) - 1, and a new key stands at its own token's
position, so siblings share a position.
"""
import torch

from flash_attn.flash_window_attn_interface import _binding, _window


def pack_tree_mask(mask):
    """Truth values (total_q, n), n <= 256: whether a new token sees the n-th of its sequence -> (total_q,
    ceil(n / 64)) int64 for `flash_paged_attn_func`."""
    rows, n = mask.shape
    if n > 256:
        raise RuntimeError(f"a tree holds at most 256 tokens, got {n}")
    words = max(1, (n + 63) // 64)
    m = torch.zeros((rows, words * 64), dtype=torch.int64, device=mask.device)
    m[:, :n] = (mask != 0).to(torch.int64)
    shift = torch.arange(64, dtype=torch.int64, device=mask.device)
    return (m.view(rows, words, 64) << shift).sum(-1)     # each bit once: the sum is their union


def tree_from_parents(parents):
    """`tree_mask` of trees of one size: parents (batch, n) int, the index of each token's parent in its own tree
    (before the token itself) or -1 for a root. Each depth of the tree is one product of truth values."""
    batch, n = parents.shape
    idx = torch.arange(n, device=parents.device)
    step = (parents.unsqueeze(-1) == idx).float()                 # (batch, token, parent)
    seen = torch.eye(n, device=parents.device).expand(batch, n, n)
    reach = seen
    for _ in range(max(0, (n - 1).bit_length())):                 # paths of up to 1, 2, 4, ... steps
        reach = ((reach + torch.bmm(step, reach)) > 0).float()
        step = (torch.bmm(step, step) > 0).float()
    return pack_tree_mask((reach > 0).reshape(batch * n, n))


def flash_paged_attn_func(q, k_pages, v_pages, block_table, context_lens, cu_seqlens_q, max_seqlen_q,
                          max_context_len=None, tree_mask=None, window_size=None, num_sinks=0, seq_ids=None,
                          softmax_scale=None, return_lse=False):
    """Attention of q (total_q, nheads, headdim) over k_pages, v_pages (num_pages, page_size, nheads_k, headdim).

    fp16 or bf16; nheads a multiple of nheads_k; headdim a multiple of 8, at most 128; page_size a power of two, 16
    or more; the pages may be strided views with a contiguous last dimension. block_table (num_seqs, max_blocks) and
    context_lens (num_seqs,) int32: a sequence's pages and the keys before its first new token. cu_seqlens_q
    (batch + 1,) int32. seq_ids (batch,) int32 picks the sequences of this call out of the table; without it the
    table has batch rows. An id of -1 marks an unused entry, its output rows are 0.

    max_context_len bounds context_lens (default: what the table can hold). It only decides how the work is split;
    a capture for later lengths wants a bound on those. tree_mask (total_q, words) int64, 1 to 4 words, see above.
    window_size, num_sinks, softmax_scale and return_lse as in `flash_window_attn_unpadded_func`.

    A table entry outside [0, num_pages) is not read: nobody sees its keys. Rows of a page that no token sees may hold
    anything, infinities and NaN among them.
    """
    window, sinks = _window(window_size, num_sinks)
    r = _binding().paged_attn(q, k_pages, v_pages, block_table, context_lens, cu_seqlens_q, max_seqlen_q,
                              max_context_len, tree_mask, window, sinks, seq_ids, softmax_scale, return_lse)
    return (r[0], r[1]) if return_lse else r[0]
