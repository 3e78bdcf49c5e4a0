"""Attention over a paged cache (flash_paged_attn_interface): single tokens, chunks and trees of drafted tokens against a
64-bit plain form within bounds that count the kernel's roundings; pages, masks, unused entries, refusals."""
import ctypes
import math

import pytest
import torch

from oracle import window_ref as ref

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _func():
    from flash_attn.flash_paged_attn_interface import flash_paged_attn_func
    return flash_paged_attn_func


# ---------------------------------------------------------------------------------------- CPU
def test_tree_masks():
    from flash_attn.flash_paged_attn_interface import pack_tree_mask, tree_from_parents
    m = tree_from_parents(torch.tensor([[-1, 0, 0, 2, -1], [-1, 0, 1, 2, 3]]))
    assert m.flatten().tolist() == [1, 3, 5, 13, 16, 1, 3, 7, 15, 31]
    t = torch.zeros(2, 200, dtype=torch.bool)
    t[0, [0, 63, 64, 199]] = True
    m = pack_tree_mask(t)
    assert m.shape == (2, 4) and m[0, 0].item() == 1 - 2 ** 63 and m[0, 1].item() == 1 and m[0, 3].item() == 1 << 7 and not m[1].any()
    chain = tree_from_parents(torch.arange(-1, 129).unsqueeze(0))
    assert [sum(bin(w & (2 ** 64 - 1)).count("1") for w in r) for r in chain.tolist()] == list(range(1, 131))
    with pytest.raises(RuntimeError, match="256"):
        pack_tree_mask(torch.zeros(1, 257, dtype=torch.bool))


def _abi():
    from flash_attn import flash_attn_hip as hip
    L = hip.lib()
    i64, i32, vp, f32 = ctypes.c_int64, ctypes.c_int32, ctypes.c_void_p, ctypes.c_float

    class Args(ctypes.Structure):
        _fields_ = [(n, vp) for n in "q o softmax_lse k_pages v_pages block_table context_lens seq_ids cu_seqlens_q tree_mask workspace".split()] + \
            [(n, i64) for n in ("workspace_bytes q_row_stride q_head_stride o_row_stride o_head_stride k_page_stride k_row_stride "
                                "k_head_stride v_page_stride v_row_stride v_head_stride table_stride total_q").split()] + \
            [(n, i32) for n in ("batch nheads nheads_k head_dim num_pages page_size num_seqs max_blocks max_seqlen_q max_context_len "
                                "tree_words lse_stride window num_sinks").split()] + [("softmax_scale", f32), ("dtype", i32)]
    L.fa_window_args_size.restype = i64
    L.fa_paged_workspace.restype = i64
    return L, Args


def _valid(Args):
    a = Args()
    for n in "q o softmax_lse k_pages v_pages block_table context_lens cu_seqlens_q".split():
        setattr(a, n, 4096)
    a.q_row_stride = a.o_row_stride = 128
    a.q_head_stride = a.o_head_stride = a.k_head_stride = a.v_head_stride = 64
    a.k_page_stride = a.v_page_stride = 2048
    a.k_row_stride = a.v_row_stride = 128
    a.table_stride = a.max_blocks = 64
    a.total_q, a.batch, a.nheads, a.nheads_k, a.head_dim = 1, 1, 2, 2, 64
    a.num_pages, a.page_size, a.num_seqs, a.max_seqlen_q, a.max_context_len, a.lse_stride = 9, 16, 1, 1, 1000, 1
    a.softmax_scale, a.dtype = 0.125, 1
    return a


@pytest.mark.parametrize("change, text", [
    ({"dtype": 2}, "dtype"), ({"batch": 0}, "batch_size"), ({"nheads": 3}, "multiple of nheads_k"), ({"head_dim": 12}, "head_size"),
    ({"page_size": 8}, "page_size"), ({"page_size": 48}, "page_size"), ({"max_blocks": 1 << 27}, "2^30"), ({"window": -1}, "window"),
    ({"num_sinks": -1}, "num_sinks"), ({"softmax_scale": math.nan}, "finite"), ({"q": 0}, "q is NULL"), ({"o": 4097}, "aligned"),
    ({"k_pages": 0}, "k_pages"), ({"v_row_stride": 132}, "multiple of 8"), ({"k_row_stride": 32}, "overlap"), ({"k_page_stride": -64}, "negative"),
    ({"context_lens": 0}, "context_lens"), ({"block_table": 0}, "block_table"), ({"table_stride": 3}, "table_stride"), ({"batch": 2}, "seq_ids"),
    ({"lse_stride": 0}, "lse_stride"), ({"tree_mask": 4096, "tree_words": 5}, "tree_mask"), ({"tree_mask": 4096, "tree_words": 1, "max_seqlen_q": 65}, "tree_mask"),
    ({"cu_seqlens_q": 0}, "cu_seqlens_q"), ({"max_context_len": -1}, "negative"),
])
def test_c_abi_refusals(change, text):
    L, Args = _abi()
    assert L.fa_window_args_size(1) == ctypes.sizeof(Args)
    a = _valid(Args)
    for n, x in change.items():
        setattr(a, n, x)
    assert L.fa_paged_fwd(ctypes.byref(a), None) != 0
    assert text in L.fa_last_error().decode(), L.fa_last_error()
    assert L.fa_paged_workspace(ctypes.byref(a)) < 0


def test_c_abi_workspace():
    L, Args = _abi()
    a = _valid(Args)
    need = L.fa_paged_workspace(ctypes.byref(a))
    assert need > 0 and need % (66 * 4 * 2) == 0            # the splits' O, m and l of two rows
    for ws, n in ((0, need), (4096, need - 4), (4100, need)):
        a.workspace, a.workspace_bytes = ws, n
        assert L.fa_paged_fwd(ctypes.byref(a), None) != 0 and "workspace" in L.fa_last_error().decode()
    assert L.fa_paged_fwd(None, None) != 0 and L.fa_paged_workspace(None) < 0
    a.max_seqlen_q = 0
    assert L.fa_paged_fwd(ctypes.byref(a), None) == 0 and L.fa_paged_workspace(ctypes.byref(a)) == 0


def test_refusals_before_any_launch():
    q = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    p = torch.zeros(2, 16, 2, 64, dtype=torch.bfloat16)
    t = torch.zeros(1, 1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="on the GPU"):
        _func()(q, p, p, t, t[0], torch.tensor([0, 1], dtype=torch.int32), 1)
    with pytest.raises(RuntimeError, match="window_size"):
        _func()(q, p, p, t, t[0], torch.tensor([0, 1], dtype=torch.int32), 1, window_size=0)


# ---------------------------------------------------------------------------------------- GPU
class Setup:
    """A cache of sequences with `ctx` keys and `new` tokens in shuffled pages; what no token sees holds NaN."""

    def __init__(self, dtype, d, hq, hk, page, ctx, new, seed=0, layout="rows", spare=2):
        from window_testutil import cu, randn
        dt = TYPES[dtype]
        self.ctx, self.new, self.page = ctx, new, page
        blocks = [-(-(c + n) // page) for c, n in zip(ctx, new)]
        pages = sum(blocks) + spare
        shape = (pages, page, hk, d)
        if layout == "heads":                # (pages, heads, rows, d) seen as (pages, rows, heads, d)
            make = lambda: torch.full((pages, hk, page, d), math.nan, dtype=dt, device="cuda").transpose(1, 2)
        elif layout == "packed":             # K and V of a row side by side
            both = torch.full((pages, page, hk, 2, d), math.nan, dtype=dt, device="cuda")
            parts = iter((both[..., 0, :], both[..., 1, :]))
            make = lambda: next(parts)
        else:
            make = lambda: torch.full(shape, math.nan, dtype=dt, device="cuda")
        self.k, self.v = make(), make()
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).int()
        self.table = torch.full((len(ctx), max(blocks) + 1), -1, dtype=torch.int32)
        self.keys = []
        at = 0
        for b, n in enumerate(blocks):
            self.table[b, :n] = order[at:at + n]
            at += n
            m = ctx[b] + new[b]
            kk, vv = randn(seed + 100 + b, (m, hk, d), dt), randn(seed + 200 + b, (m, hk, d), dt)
            j = torch.arange(m)
            p = self.table[b].long()[j // page].cuda()
            self.k[p, (j % page).cuda()], self.v[p, (j % page).cuda()] = kk, vv
            self.keys.append((kk, vv))
        self.table = self.table.cuda()
        self.context = torch.tensor(ctx, dtype=torch.int32, device="cuda")
        self.cu = cu(new)
        self.q = randn(seed + 1, (sum(new), hq, d), dt)
        self.dt, self.scale = dt, d ** -0.5

    def compare(self, got, window=None, sinks=0, tree=None, scale=None, skip=(), lse=None):
        """tree: truth values (total_q, n)."""
        from window_testutil import check
        scale = self.scale if scale is None else scale
        H, G = self.q.shape[1], self.q.shape[1] // self.k.shape[2]
        at = 0
        for b, (c, n) in enumerate(zip(self.ctx, self.new)):
            path = tree[at:at + n, :n].cuda() if tree is not None else torch.ones(n, n, device="cuda").tril().bool()
            pos = c + path.sum(1) - 1
            kpos = torch.cat([torch.arange(c, device="cuda"), pos])
            live = torch.cat([torch.ones(n, c, dtype=torch.bool, device="cuda"), path], 1)
            if window:
                live &= (kpos > pos[:, None] - window) | (kpos < sinks)
            for h in range(H):
                if b in skip:
                    assert not got[at:at + n, h].any()
                    continue
                a = (self.q[at:at + n, h], self.keys[b][0][:, h // G], self.keys[b][1][:, h // G], live, scale)
                out, ll, p = ref.attention(*a)
                e = ref.bounds(*a, p, out, dtype=self.dt) + torch.finfo(self.dt).tiny
                check(f"sequence {b} head {h}", got[at:at + n, h], out, e)
                if lse is not None:
                    x = lse[b, h, :n].double()
                    dead = torch.isinf(ll)
                    assert torch.equal(torch.isinf(x), dead)
                    assert ((x - ll).abs()[~dead] <= (2.0 ** -20 * (1 + ll.abs()) + 2.0 ** -24 * (self.q.shape[2] + 8) * 40)[~dead]).all()
            at += n

    def run(self, **kw):
        return _func()(self.q, self.k, self.v, self.table, self.context, self.cu, max(self.new), softmax_scale=kw.pop("scale", None), **kw)


def _random_tree(new, seed):
    g = torch.Generator().manual_seed(seed)
    n = max(new)
    mask = torch.zeros(sum(new), n, dtype=torch.bool)
    at = 0
    for m in new:
        for i in range(m):
            parent = int(torch.randint(-1, i, (1,), generator=g)) if i else -1
            if parent >= 0:
                mask[at + i] |= mask[at + parent]
            mask[at + i, i] = True
        at += m
    return mask


CASES = [
    # dtype, head_dim, heads, kv heads, page, contexts, new tokens, window, sinks, tree
    ("bf16", 64, 4, 4, 16, [0], [1], None, 0, False),
    ("bf16", 64, 8, 2, 16, [1, 16, 15, 500], [1, 1, 1, 1], None, 0, False),
    ("fp16", 128, 32, 4, 64, [1000, 63, 0], [1, 1, 1], None, 0, False),
    ("bf16", 128, 8, 1, 32, [777, 3], [1, 1], 100, 4, False),
    ("bf16", 32, 7, 7, 128, [260], [1], 33, 0, False),
    ("fp16", 80, 6, 2, 16, [300, 100], [5, 0], None, 0, False),            # a chunk; no new token
    ("bf16", 64, 4, 2, 64, [100, 0, 31], [70, 130, 1], 50, 3, False),      # a prompt's chunk
    ("bf16", 128, 16, 2, 16, [200, 17], [64, 9], None, 0, True),
    ("fp16", 64, 12, 12, 16, [130, 64, 1], [25, 25, 25], None, 0, True),
    ("bf16", 128, 14, 2, 64, [400], [40], 6, 2, True),                     # paths longer than the window
    ("bf16", 24, 4, 1, 16, [50], [200], None, 0, True),                    # masks of four words
    ("fp16", 64, 2, 2, 1024, [3000], [3], 1, 5, True),
    ("bf16", 64, 8, 8, 16, [0, 0], [33, 2], 4, 1, True),
    ("bf16", 96, 64, 1, 32, [90], [1], 1000, 0, False),
    ("bf16", 64, 40, 1, 16, [2000], [1], None, 0, False),
]


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["rows", "heads", "packed"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[0]}-d{c[1]}-h{c[2]}x{c[3]}-p{c[4]}-c{max(c[5])}-n{max(c[6])}-w{c[7]}-t{int(c[9])}")
def test_values(case, layout):
    from flash_attn.flash_paged_attn_interface import pack_tree_mask
    dt, d, hq, hk, page, ctx, new, w, s, tree = case
    x = Setup(dt, d, hq, hk, page, ctx, new, layout=layout)
    t = _random_tree(new, 3) if tree else None
    packed = pack_tree_mask(t).cuda() if tree else None
    for bound in (None, max(ctx), 0):        # how the work is split
        out, lse = x.run(max_context_len=bound, window_size=w, num_sinks=s, tree_mask=packed, return_lse=True)
        x.compare(out, w, s, t, lse=lse)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [-0.3, 0.0, 2.0])
def test_scales(scale):
    x = Setup("bf16", 64, 4, 2, 16, [400, 3], [3, 3])
    x.compare(x.run(scale=scale), scale=scale)


@pytest.mark.gpu
def test_sequences_picked_by_id_and_unused_entries():
    x = Setup("bf16", 128, 8, 2, 16, [100, 200, 50, 9], [2, 2, 2, 2])
    ids = torch.tensor([3, -1, 1, 7], dtype=torch.int32, device="cuda")
    got = x.run(seq_ids=ids)
    assert not got[2:4].any() and not got[6:8].any()
    pick = Setup("bf16", 128, 8, 2, 16, [100, 200, 50, 9], [2, 2, 2, 2])
    pick.ctx, pick.keys = [9, 0, 200, 0], [x.keys[3], x.keys[0], x.keys[1], x.keys[0]]
    pick.keys[1] = pick.keys[3] = (x.keys[3][0][:2], x.keys[3][1][:2])
    pick.compare(got, skip=(1, 3))


@pytest.mark.gpu
def test_masks_that_leave_a_row_empty():
    """A tree row without a bit, and no context: nothing is seen."""
    from flash_attn.flash_paged_attn_interface import pack_tree_mask
    x = Setup("bf16", 64, 4, 2, 16, [0, 40], [3, 3])
    t = torch.tensor([[1, 0, 0], [0, 0, 0], [1, 0, 1]] * 2).bool()
    out, lse = x.run(tree_mask=pack_tree_mask(t).cuda(), return_lse=True)
    assert not out[1].any() and torch.isinf(lse[0, :, 1]).all() and out[4].any()
    x.compare(out, tree=t, lse=lse)


@pytest.mark.gpu
@pytest.mark.parametrize("page", [16, 64])
def test_pages_that_are_not_there(page):
    """Entries behind the window evicted (-1); a table's wild entries (never read, seen by nobody)."""
    x = Setup("bf16", 128, 4, 1, page, [1000], [1])
    want = x.run(window_size=100, num_sinks=5)
    gone = x.table.clone()
    gone[0, -(-5 // page):900 // page] = -1
    keep, x.table = x.table, gone
    x.k[keep[0, 2].long()], x.v[keep[0, 2].long()] = math.nan, math.inf
    assert torch.equal(x.run(window_size=100, num_sinks=5), want)
    x.table = keep.clone()
    wild = 500 // page
    x.table[0, 2], x.table[0, wild] = -1, 1 << 30      # page 2 was spoilt above
    cols = torch.ones(1001, dtype=torch.bool)
    cols[2 * page:3 * page] = cols[wild * page:(wild + 1) * page] = False
    out = x.run()
    k, v = x.keys[0]
    for h in range(4):
        live = cols[None].cuda()
        a = (x.q[:, h], k[:, 0], v[:, 0], live, x.scale)
        r, _, p = ref.attention(*a)
        assert ((out[:, h].double() - r).abs() <= ref.bounds(*a, p, r)).all()


@pytest.mark.gpu
def test_infinities_reach_only_what_sees_them():
    """A drafted token's NaN stays with its descendants; a NaN in front of the window with nobody."""
    from flash_attn.flash_paged_attn_interface import pack_tree_mask
    x = Setup("bf16", 64, 4, 2, 16, [100], [4])
    t = torch.tensor([[1, 0, 0, 0], [1, 1, 0, 0], [1, 0, 1, 0], [1, 1, 0, 1]]).bool()
    for j in list(range(3, 50)) + [101]:
        p, r = int(x.table[0, j // 16]), j % 16
        x.k[p, r], x.v[p, r] = math.nan, math.nan
        x.keys[0][0][j], x.keys[0][1][j] = math.nan, math.nan
    out = x.run(tree_mask=pack_tree_mask(t).cuda(), window_size=40, num_sinks=3)
    assert torch.isfinite(out[[0, 2]]).all() and torch.isnan(out[[1, 3]]).all()
    keys = x.keys[0]
    keys[0][101], keys[1][101] = 0, 0
    want = torch.where(torch.isnan(out), 0, out)
    live = torch.cat([torch.ones(4, 100, dtype=torch.bool), t], 1).cuda()
    pos = torch.tensor([100, 101, 101, 102]).cuda()
    kpos = torch.cat([torch.arange(100).cuda(), pos])
    live &= (kpos > pos[:, None] - 40) | (kpos < 3)
    for h in range(4):
        a = (x.q[:, h], keys[0][:, h // 2], keys[1][:, h // 2], live, x.scale)
        r, _, p = ref.attention(*a)
        assert ((want[:, h].double() - r).abs() <= ref.bounds(*a, p, r))[[0, 2]].all()


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """Pages behind 2^32 bytes of a pool."""
    pages, page, hk, d = 5000, 1024, 8, 64            # 5.2 GB each
    k = torch.zeros(pages, page, hk, d, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    from window_testutil import cu, randn
    n = 3000
    kk, vv = randn(1, (n, hk, d), torch.bfloat16), randn(2, (n, hk, d), torch.bfloat16)
    ids = [4999, 4200, 4998]
    for i, p in enumerate(ids):
        m = min(page, n - i * page)
        k[p, :m], v[p, :m] = kk[i * page:i * page + m], vv[i * page:i * page + m]
    q = randn(3, (1, hk, d), torch.bfloat16)
    out = _func()(q, k, v, torch.tensor([ids], dtype=torch.int32, device="cuda"), torch.tensor([n - 1], dtype=torch.int32, device="cuda"), cu([1]), 1)
    for h in range(hk):
        a = (q[:, h], kk[:, h], vv[:, h], torch.ones(1, n, dtype=torch.bool, device="cuda"), d ** -0.5)
        r, _, p = ref.attention(*a)
        assert ((out[:, h].double() - r).abs() <= ref.bounds(*a, p, r)).all()


@pytest.mark.gpu
def test_graph_replays_with_growing_contexts():
    """Two graphs over one cache, captured once, replayed with other lengths and queries, eager calls between."""
    x = Setup("bf16", 128, 16, 2, 16, [900, 300], [1, 1])
    y = Setup("bf16", 128, 16, 2, 16, [900, 300], [1, 1], seed=5)
    run = lambda z: z.run(max_context_len=1000)
    run(x)
    graphs, outs = [], []
    for z in (x, y):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run(z))
        graphs.append(g)
    for ctx in ([900, 300], [17, 0], [500, 299]):
        for z in (x, y):
            z.context.copy_(torch.tensor(ctx, dtype=torch.int32))
            z.q.normal_()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for z, o in zip((x, y), outs):
            assert torch.equal(run(z), o)
            whole = z.keys
            z.ctx, z.keys = ctx, [(a[:c + 1], b[:c + 1]) for (a, b), c in zip(whole, ctx)]
            z.compare(o)
            z.keys = whole


@pytest.mark.gpu
def test_rows_behind_the_last_sequence_are_zero_and_streams():
    x = Setup("bf16", 64, 4, 2, 16, [100, 20], [2, 1])
    want = x.run()
    x.q = torch.cat([x.q, x.q.new_ones(50, 4, 64)])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = x.run()
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got[:3], want) and not got[3:].any()


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    x = Setup("bf16", 64, 4, 2, 16, [100], [2])
    with pytest.raises(RuntimeError, match="no backward"):
        _func()(x.q.requires_grad_(), x.k, x.v, x.table, x.context, x.cu, 2)
    x.q = x.q.detach()
    with pytest.raises(RuntimeError, match="batch_size rows"):
        _func()(x.q, x.k, x.v, x.table.expand(2, -1).contiguous(), x.context.expand(2).contiguous(), x.cu, 2)
    with pytest.raises(RuntimeError, match="tree_mask"):
        x.run(tree_mask=torch.zeros(2, 1, dtype=torch.int32, device="cuda"))
    with pytest.raises(RuntimeError, match="tree_mask"):
        x.run(tree_mask=torch.zeros(3, 1, dtype=torch.int64, device="cuda"))
    with pytest.raises(RuntimeError, match="int32"):
        _func()(x.q, x.k, x.v, x.table.long(), x.context, x.cu, 2)
    with pytest.raises(RuntimeError, match="power of two"):
        _func()(x.q, x.k[:, :12], x.v[:, :12], x.table, x.context, x.cu, 2)
    with pytest.raises(RuntimeError, match="same dtype"):
        _func()(x.q.half(), x.k, x.v, x.table, x.context, x.cu, 2)
