"""A key/value cache in pages for `flash_paged_attn_interface`: room for tokens, beams that share pages, drafted
tokens kept or dropped, pages given back, all on the device.

    cache = PagedKVCache(layers, num_pages, page_size, nheads_k, headdim, max_seqs, max_blocks)
    cache.reserve(slots, n)                              # once a step
    for layer in range(layers):
        cache.write(layer, slots, k, v, cu_seqlens, n)   # the step's keys and values
        out = cache.attend(layer, q, slots, cu_seqlens, n, tree_mask=tree)
    cache.compact(slots, keep, counts)                   # the accepted tokens stay, the rest goes

No method reads a length on the host, so a step can be captured into a graph. What turns out on the device to be
impossible (no free page, an index out of range) is left undone and noted; `check()` raises it. Methods are ordered
like any work on the current stream; use of one cache on several streams needs events between them.
"""
import torch

from flash_attn.flash_paged_attn_interface import flash_paged_attn_func
from flash_attn.flash_window_attn_interface import _binding, _window

_ERRORS = {
    1: "not enough free pages",
    2: "a sequence passes max_blocks pages",
    4: "a slot is out of range or named twice",
    8: "a token has no page of its sequence's own (reserve comes first)",
    16: "indices to keep are not ascending, or their count is out of range",
    32: "a negative length, or one that the sequence cannot be cut to",
    64: "a fork into a slot that holds tokens",
}


class PagedKVCache:
    """num_pages pages of page_size tokens (a power of two, 16 or more) in each of num_layers layers, for up to
    max_seqs sequences (slots) of up to max_blocks pages. window_size and num_sinks are those of the attention over
    the cache: `attend` uses them, `evict` gives back what they leave behind.

    Attributes, all tensors on the device: k, v (num_layers, num_pages, page_size, nheads, headdim); block_table
    (max_seqs, max_blocks) int32, -1 where there is no page; seqlens, nblocks (max_seqs,) int32: tokens, and table
    entries in use; refcount (num_pages,) int32: sequences that hold a page, 0 for a free one; status (1,) int32.

    `slots` arguments are int32 vectors of up to 4096 sequence numbers, each named once; -1 is passed over."""

    def __init__(self, num_layers, num_pages, page_size, nheads, headdim, max_seqs, max_blocks, dtype=torch.bfloat16,
                 device="cuda", window_size=None, num_sinks=0):
        device = torch.device(device)
        self.window_size, self.num_sinks = window_size, num_sinks
        window, sinks = _window(window_size, num_sinks)
        i32 = {"dtype": torch.int32, "device": device}
        self.k = torch.empty((num_layers, num_pages, page_size, nheads, headdim), dtype=dtype, device=device)
        self.v = torch.empty_like(self.k)
        self.block_table = torch.full((max_seqs, max_blocks), -1, **i32)
        self.seqlens = torch.zeros(max_seqs, **i32)
        self.nblocks = torch.zeros(max_seqs, **i32)
        self.refcount = torch.zeros(num_pages, **i32)
        self.status = torch.zeros(1, **i32)
        self._cache = _binding().PagedCache(self.k, self.v, self.block_table, self.seqlens, self.nblocks, self.refcount,
                                            self.status, window, sinks)

    def reserve(self, slots, counts):
        """Pages for `counts` (an int, or an int32 vector) more tokens of each slot: the lowest free ones, in the
        order of the slots; all or none. A partly full last page that other sequences hold too is left to them and
        its rows are copied (the last of the call's slots that hold it keeps it when nobody else does)."""
        if isinstance(counts, torch.Tensor):
            self._cache.reserve_each(slots, counts)
        else:
            self._cache.reserve(slots, counts)

    def write(self, layer, slots, k, v, cu_seqlens, max_seqlen):
        """Stores k, v (total, nheads, headdim) of one layer behind the tokens of the slots: rows cu_seqlens[i] ..
        cu_seqlens[i + 1] - 1, at most max_seqlen of them, behind slots[i]. Lengths grow by `compact` only."""
        self._cache.write(layer, slots, k, v, cu_seqlens, max_seqlen)

    def attend(self, layer, q, slots, cu_seqlens_q, max_seqlen_q, max_context_len=None, tree_mask=None,
               softmax_scale=None, return_lse=False):
        """`flash_paged_attn_func` of q over one layer of the slots, whose new tokens are written."""
        return flash_paged_attn_func(q, self.k[layer], self.v[layer], self.block_table, self.seqlens, cu_seqlens_q,
                                     max_seqlen_q, max_context_len=max_context_len, tree_mask=tree_mask,
                                     window_size=self.window_size, num_sinks=self.num_sinks, seq_ids=slots,
                                     softmax_scale=softmax_scale, return_lse=return_lse)

    def compact(self, slots, keep, counts):
        """Keeps counts[i] of the tokens written behind slots[i]: those at keep[i, :counts[i]], ascending, counted
        from the slot's length. They are moved together in every layer and the length grows by counts[i]; pages
        behind the new end are given back."""
        self._cache.compact(slots, keep, counts)

    def fork(self, parents, children):
        """Each child, an empty slot, begins with its parent's tokens, in the parent's pages. (What the parent has
        written and not kept stays its own.)"""
        self._cache.fork(parents, children)

    def truncate(self, slots, lens):
        """Shortens the slots to lens (int32 vector) tokens and gives the pages behind back. A length whose window
        reaches into evicted pages is refused."""
        self._cache.truncate(slots, lens)

    def free(self, slots):
        """Empties the slots and gives their pages back."""
        self._cache.free(slots)

    def evict(self, slots):
        """Gives back the pages that no later token sees: past the sinks and wholly behind the window."""
        self._cache.evict(slots)

    def check(self):
        """Waits for the device and raises what could not be done since the last check."""
        bits = int(self.status.item())
        if bits:
            self.status.zero_()
            raise RuntimeError("PagedKVCache: " + "; ".join(t for b, t in _ERRORS.items() if bits & b))
