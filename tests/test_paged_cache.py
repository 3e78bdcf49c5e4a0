"""PagedKVCache: every call against a model of it on the host, whole states compared; what cannot be done is left
undone and noted; and a run of the operators together, as a long generation uses them."""
import ctypes
import math
import random

import pytest
import torch


# ---------------------------------------------------------------------------------------- CPU
def _abi():
    from flash_attn import flash_attn_hip as hip
    L = hip.lib()
    vp, i32 = ctypes.c_void_p, ctypes.c_int32

    class Cache(ctypes.Structure):
        _fields_ = [(n, vp) for n in "k_pages v_pages block_table seqlens nblocks refcount status scratch".split()] + \
            [(n, i32) for n in "layers num_pages page_size nheads head_dim max_seqs max_blocks window num_sinks".split()]
    for f in (L.fa_cache_struct_size, L.fa_cache_scratch_words):
        f.restype = ctypes.c_int64
    c = Cache(*[4096] * 8, 2, 10, 16, 2, 64, 4, 5, 0, 0)
    return L, c


@pytest.mark.parametrize("change, text", [
    ({"layers": 0}, "positive"), ({"num_pages": 0}, "positive"), ({"page_size": 24}, "page_size"), ({"page_size": 8}, "page_size"),
    ({"head_dim": 20}, "head_size"), ({"head_dim": 136}, "head_size"), ({"max_seqs": 70000}, "sequences"), ({"num_pages": 1 << 27}, "2^31"),
    ({"window": -1}, "window"), ({"status": 0}, "NULL"), ({"k_pages": 4100}, "aligned"),
])
def test_c_abi_refuses_a_cache(change, text):
    L, c = _abi()
    assert L.fa_cache_struct_size() == ctypes.sizeof(c)
    for n, x in change.items():
        setattr(c, n, x)
    i64, p = ctypes.c_int64, ctypes.byref(c)
    for rc in (L.fa_cache_reserve(p, 4096, 1, None, 1, None), L.fa_cache_truncate(p, 4096, 1, None, None),
               L.fa_cache_evict(p, 4096, 1, None), L.fa_cache_fork(p, 4096, 4096, 1, None),
               L.fa_cache_compact(p, 4096, 1, 4096, i64(4), 4, 4096, None),
               L.fa_cache_write(p, 0, 4096, 1, 4096, i64(128), i64(64), 4096, i64(128), i64(64), 4096, i64(1), 1, None)):
        assert rc != 0
        assert text in L.fa_last_error().decode()


def test_c_abi_refusals():
    L, c = _abi()
    i64, p = ctypes.c_int64, ctypes.byref(c)
    err = lambda: L.fa_last_error().decode()
    assert L.fa_cache_reserve(None, 4096, 1, None, 1, None) and "NULL" in err()
    assert L.fa_cache_reserve(p, 4096, 5000, None, 1, None) and "4096 slots" in err()
    assert L.fa_cache_reserve(p, None, 1, None, 1, None) and "slots" in err()
    assert L.fa_cache_reserve(p, 4096, 1, None, -1, None) and "count" in err()
    assert L.fa_cache_evict(p, 4096, 1, None) and "no window" in err()
    assert L.fa_cache_compact(p, 4096, 1, 4096, i64(9), 5000, 4096, None) and "4096 tokens" in err()
    assert L.fa_cache_compact(p, 4096, 1, 4096, i64(3), 4, 4096, None)
    assert L.fa_cache_write(p, 2, 4096, 1, 4096, i64(128), i64(64), 4096, i64(128), i64(64), 4096, i64(1), 1, None) and "layer" in err()
    assert L.fa_cache_write(p, 0, 4096, 1, 4104, i64(128), i64(64), 4096, i64(128), i64(64), 4096, i64(1), 1, None) and "aligned" in err()
    assert L.fa_cache_write(p, 0, 4096, 1, 4096, i64(132), i64(64), 4096, i64(128), i64(64), 4096, i64(1), 1, None) and "aligned" in err()
    assert L.fa_cache_truncate(p, None, 0, None, None) == 0      # no slots: nothing is launched


def test_the_cache_lives_on_the_gpu():
    from flash_attn.paged_kv_cache import PagedKVCache
    with pytest.raises(RuntimeError, match="on the GPU"):
        PagedKVCache(1, 4, 16, 2, 64, 2, 4, device="cpu")
    with pytest.raises(RuntimeError, match="window_size"):
        PagedKVCache(1, 4, 16, 2, 64, 2, 4, device="cpu", window_size=0)


# ---------------------------------------------------------------------------------------- the model
class Model:
    """The cache on the host, one entry at a time; pages hold a tag for each row of each layer."""

    def __init__(self, c):
        self.L, self.P, self.ps = c.k.shape[:3]
        self.S, self.B = c.block_table.shape
        self.window, self.sinks = c.window_size, c.num_sinks
        self.table = [[-1] * self.B for _ in range(self.S)]
        self.len, self.have, self.ref, self.status = [0] * self.S, [0] * self.S, [0] * self.P, 0
        self.k, self.v = c.k.clone(), c.v.clone()

    def blocks(self, n):
        return -(-n // self.ps)

    def slots_ok(self, slots):
        """Which may be worked on: in range, named once; -1 is passed over."""
        ok = []
        for i, s in enumerate(slots):
            if s == -1:
                continue
            if not 0 <= s < self.S or slots.count(s) > 1:
                self.status |= 4
            else:
                ok.append((i, s))
        return ok

    def reserve(self, slots, counts):
        err, cow, seen = 0, {}, set()
        for i, s in enumerate(slots):
            if s == -1:
                continue
            if not 0 <= s < self.S or s in seen:
                err |= 4
                continue
            seen.add(s)
            if counts[i] < 0:
                err |= 32
            elif counts[i] > 0:
                n = self.len[s]
                if self.blocks(n + counts[i]) > self.B:
                    err |= 2
                elif n % self.ps:
                    page = self.table[s][n // self.ps]
                    if page < 0:
                        err |= 8
                    elif self.ref[page] > 1:
                        cow[i] = page
        if err:
            self.status |= err
            return
        ref = list(self.ref)
        todo = []
        for i, s in enumerate(slots):
            if s == -1 or counts[i] <= 0:
                continue
            if i in cow and ref[cow[i]] > 1:
                ref[cow[i]] -= 1
                todo.append((s, self.len[s] // self.ps, cow[i]))
            for b in range(self.have[s], self.blocks(self.len[s] + counts[i])):
                todo.append((s, b, None))
        free = [p for p in range(self.P) if self.ref[p] == 0]
        if len(todo) > len(free):
            self.status |= 1
            return
        self.ref = ref
        for (s, b, old), p in zip(todo, free):
            self.table[s][b] = p
            self.ref[p] = 1
            if old is None:
                self.have[s] = b + 1
            else:
                n = self.len[s] % self.ps
                self.k[:, p, :n], self.v[:, p, :n] = self.k[:, old, :n], self.v[:, old, :n]

    def own(self, s, j):
        """(page, row) of token j if the sequence may write it."""
        b = j // self.ps
        p = self.table[s][b] if b < self.have[s] else -1
        return (p, j % self.ps) if p >= 0 and self.ref[p] == 1 else None

    def write(self, layer, slots, k, v, cu):
        for i, s in self.slots_ok(slots):
            for t in range(cu[i], cu[i + 1]):
                at = self.own(s, self.len[s] + t - cu[i])
                if at is None:
                    self.status |= 8
                else:
                    self.k[layer, at[0], at[1]], self.v[layer, at[0], at[1]] = k[t], v[t]

    def cut(self, s, n):
        need = self.blocks(n)
        for b in range(need, self.have[s]):
            if self.table[s][b] >= 0:
                self.ref[self.table[s][b]] -= 1
            self.table[s][b] = -1
        self.len[s], self.have[s] = n, min(need, self.have[s])

    def compact(self, slots, keep, counts):
        for i, s in self.slots_ok(slots):
            if not 0 <= counts[i] <= len(keep[i]):
                self.status |= 16
                continue
            row = keep[i][:counts[i]]
            if any(x < j or (j and row[j - 1] >= x) for j, x in enumerate(row)):
                self.status |= 16
                continue
            n = self.len[s]
            there = lambda j: j // self.ps < self.have[s] and self.table[s][j // self.ps] >= 0
            if any(not there(n + x) or self.own(s, n + j) is None for j, x in enumerate(row)):
                self.status |= 8
                continue
            for j, x in enumerate(row):
                a, b = (self.table[s][(n + x) // self.ps], (n + x) % self.ps), self.own(s, n + j)
                self.k[:, b[0], b[1]], self.v[:, b[0], b[1]] = self.k[:, a[0], a[1]].clone(), self.v[:, a[0], a[1]].clone()
            self.cut(s, n + len(row))

    def fork(self, parents, children):
        for i, (p, s) in enumerate(zip(parents, children)):
            if p == -1 and s == -1:
                continue
            if not 0 <= s < self.S or children.count(s) > 1 or not 0 <= p < self.S or s in parents:
                self.status |= 4
                continue
            if self.len[s] or self.have[s]:
                self.status |= 64
                continue
            n = self.blocks(self.len[p])
            for b in range(n):
                self.table[s][b] = self.table[p][b]
                if self.table[s][b] >= 0:
                    self.ref[self.table[s][b]] += 1
            self.len[s], self.have[s] = self.len[p], n

    def truncate(self, slots, lens):
        for i, s in self.slots_ok(slots):
            n = lens[i] if lens is not None else 0
            bad = n < 0 or n > self.len[s]
            if not bad and n > 0 and self.window:
                lo = max(0, n - self.window + 1)
                bad = lo < n and self.table[s][lo // self.ps] < 0
            if bad and lens is not None:
                self.status |= 32
                continue
            self.cut(s, n)

    def evict(self, slots):
        for _, s in self.slots_ok(slots):
            end = min(max(0, self.len[s] - self.window + 1) // self.ps, self.have[s])
            for b in range(self.blocks(self.sinks), end):
                if self.table[s][b] >= 0:
                    self.ref[self.table[s][b]] -= 1
                self.table[s][b] = -1

    def compare(self, c):
        assert c.block_table.tolist() == self.table
        assert c.seqlens.tolist() == self.len and c.nblocks.tolist() == self.have
        assert c.refcount.tolist() == self.ref
        assert c.status.item() == self.status, (c.status.item(), self.status)
        assert torch.equal(c.k, self.k) and torch.equal(c.v, self.v)


def _cache(*a, **kw):
    from flash_attn.paged_kv_cache import PagedKVCache
    c = PagedKVCache(*a, **kw)
    c.k.normal_()
    c.v.normal_()
    return c


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(12))
def test_random_calls_against_the_model(seed):
    """Calls of every kind, most of them possible, some not; the whole state is compared after each."""
    rng = random.Random(seed)
    window, sinks = ((None, 0), (40, 3), (16, 0), (1, 17))[seed % 4]
    heads, d = rng.choice([(2, 64), (1, 8), (3, 40), (8, 128)])
    c = _cache(2, rng.choice([12, 40]), rng.choice([16, 32]), heads, d, 6, 9, dtype=rng.choice([torch.bfloat16, torch.float16]),
               window_size=window, num_sinks=sinks)
    m = Model(c)
    wild = lambda s: s if rng.random() < 0.97 else rng.choice([-1, -1, -2, 6, 10 ** 6])
    for step in range(60):
        n = rng.randint(1, 5)
        slots = [wild(s) for s in (rng.sample(range(6), n) if rng.random() < 0.95 else [rng.randrange(6) for _ in range(n)])]
        op = rng.choice(["reserve", "reserve", "write", "write", "compact", "compact", "fork", "truncate", "evict", "free", "step", "step", "step"])
        if op in ("reserve", "step"):
            counts = [rng.choice([0, 1, 5, 20, -1 if rng.random() < 0.1 else 2]) for _ in slots]
            if rng.random() < 0.5:
                counts = [max(0, counts[0])] * n
                c.reserve(_i32(slots), counts[0])
            else:
                c.reserve(_i32(slots), _i32(counts))
            m.reserve(slots, counts)
        if op in ("write", "step"):
            lens = counts if op == "step" else [rng.randint(0, 6) for _ in slots]
            cu = [0]
            for x in lens:
                cu.append(cu[-1] + max(0, x))
            for layer in range(2):
                k, v = (torch.randn(cu[-1] + 2, heads, d, device="cuda").to(c.k.dtype) for _ in range(2))
                if len(set(slots)) == len(slots):
                    c.write(layer, _i32(slots), k, v, _i32(cu), max(1, max(lens)))
                    m.write(layer, slots, k, v, cu)
        if op in ("compact", "step"):
            most = max(1, max(counts) if op == "step" else 4)
            keep = [sorted(rng.sample(range(most + 2), min(most, 3))) + [0] * 3 for _ in slots]
            keep = [x[:3] for x in keep]
            if op == "step":
                keep = [list(range(counts[i]))[-3:] + [99] * (3 - min(3, max(0, counts[i]))) for i in range(n)]
                num = [min(3, max(0, x)) for x in counts]
            else:
                num = [rng.choice([0, 1, 2, 3, 4 if rng.random() < 0.1 else 1]) for _ in slots]
            c.compact(_i32(slots), _i32(keep), _i32(num))
            m.compact(slots, keep, num)
        if op == "fork":
            kids = [wild(s) for s in rng.sample(range(6), n)]
            c.fork(_i32(slots), _i32(kids))
            m.fork(slots, kids)
        if op == "truncate":
            lens = [rng.randint(0, max(0, m.len[s])) if 0 <= s < 6 and rng.random() < 0.9 else rng.choice([-1, 1000]) for s in slots]
            c.truncate(_i32(slots), _i32(lens))
            m.truncate(slots, lens)
        if op == "evict" and window:
            c.evict(_i32(slots))
            m.evict(slots)
        if op == "free":
            c.free(_i32(slots))
            m.truncate(slots, None)
        m.compare(c)
        held = sum(1 for row in m.table for p in row if p >= 0)
        assert held == sum(m.ref)
        if m.status and rng.random() < 0.7:
            with pytest.raises(RuntimeError, match="PagedKVCache"):
                c.check()
            m.status = 0
    c.status.zero_()
    c.check()


@pytest.mark.gpu
def test_many_slots_and_pages():
    """More slots than threads, more pages than one pass over them; a slot named twice far apart."""
    c = _cache(1, 9000, 16, 1, 8, 4096, 3)
    m = Model(c)
    slots = list(range(4096))
    random.Random(0).shuffle(slots)
    counts = [random.Random(1).choice([1, 16, 17]) for _ in slots]
    rng = random.Random(2)
    counts = [rng.choice([1, 16, 17]) for _ in slots]
    c.reserve(_i32(slots), _i32(counts))
    m.reserve(slots, counts)
    m.compare(c)
    keep = [[0]] * 4096
    c.compact(_i32(slots), _i32(keep), _i32([1] * 4096))
    m.compact(slots, keep, [1] * 4096)
    m.compare(c)
    twice = slots[:4000] + [slots[1]]
    c.reserve(_i32(twice), 30)
    m.reserve(twice, [30] * 4001)
    assert m.status == 4
    m.compare(c)
    c.free(_i32(slots[::2]))
    m.truncate(slots[::2], None)
    m.compare(c)
    with pytest.raises(RuntimeError, match="twice"):
        c.check()
    with pytest.raises(RuntimeError, match="4096 slots"):
        c.free(_i32(list(range(4096)) + [0]))


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """Layers and pages behind 2^32 bytes: a write, a copy of a shared page, a move."""
    from flash_attn.paged_kv_cache import PagedKVCache
    c = PagedKVCache(3, 4100, 64, 8, 128, 4, 3)            # 537 MB a layer and 4100 pages: 1.6 GB, rows past 2^31 elements
    big = PagedKVCache(9, 8192, 32, 8, 128, 4, 3)          # 537 MB a layer: 4.8 GB
    for cache in (c, big):
        cache.refcount[:-6] = 1                            # only the last pages are free
        s = _i32([0])
        cache.reserve(s, 40)
        k, v = (torch.randn(40, 8, 128, device="cuda").bfloat16() for _ in range(2))
        L = cache.k.shape[0]
        for layer in range(L):
            cache.write(layer, s, k + layer, v - layer, _i32([0, 40]), 40)
        cache.compact(s, _i32([list(range(10)) + [20, 39]]), _i32([12]))
        cache.fork(s, _i32([1]))
        cache.reserve(_i32([1]), 1)
        cache.check()
        pages = [int(cache.block_table[i, 0]) for i in (0, 1)]
        assert pages[0] >= cache.k.shape[1] - 6 and pages[0] != pages[1]
        rows = torch.tensor(list(range(10)) + [20, 39])
        for p in pages:
            for layer in range(L):
                assert torch.equal(cache.k[layer, p, :12], (k + layer)[rows]) and torch.equal(cache.v[layer, p, :12], (v - layer)[rows])


@pytest.mark.gpu
def test_a_write_names_a_slot_once():
    c = _cache(2, 8, 16, 2, 64, 3, 2)
    m = Model(c)
    c.reserve(_i32([0, 1, 2]), 20)
    m.reserve([0, 1, 2], [20] * 3)
    k, v = (torch.randn(60, 2, 64, device="cuda").bfloat16() for _ in range(2))
    cu = [0, 20, 40, 60]
    c.write(1, _i32([2, 0, 2]), k, v, _i32(cu), 20)
    m.write(1, [2, 0, 2], k, v, cu)
    m.compare(c)
    with pytest.raises(RuntimeError, match="twice"):
        c.check()


@pytest.mark.gpu
def test_a_need_of_2_to_the_32_pages():
    """65 sequences that ask for 2^32 + 1 pages together, of a cache of 8."""
    blocks = 2 ** 26 - 1
    c = _cache(1, 8, 16, 1, 8, 65, blocks)
    want = [blocks] * 64 + [2 ** 32 + 1 - 64 * blocks]
    assert sum(want) == 2 ** 32 + 1
    c.reserve(_i32(list(range(65))), _i32([16 * n for n in want]))
    assert c.status.item() == 1 and not c.nblocks.any() and not c.refcount.any()
    assert (c.block_table[:, ::997] == -1).all() and (c.block_table[:, :64] == -1).all()
    c.status.zero_()
    c.reserve(_i32([64, 3]), 64)
    c.check()
    assert c.block_table[64, :4].tolist() == [0, 1, 2, 3] and c.block_table[3, :4].tolist() == [4, 5, 6, 7]


@pytest.mark.gpu
def test_strided_new_rows_and_refusals():
    c = _cache(1, 8, 16, 2, 64, 2, 4)
    s = _i32([1])
    c.reserve(s, 20)
    qkv = torch.randn(20, 6, 64, device="cuda").bfloat16()
    c.write(0, s, qkv[:, 2:4], qkv[:, 4:], _i32([0, 20]), 20)
    c.compact(s, _i32([list(range(20))]), _i32([20]))
    c.check()
    rows = c.k[0][c.block_table[1, :2].long()].flatten(0, 1)[:20]
    assert torch.equal(rows, qkv[:, 2:4])
    with pytest.raises(RuntimeError, match="int32"):
        c.reserve(torch.tensor([0], device="cuda"), 1)
    with pytest.raises(RuntimeError, match="dtype, heads and device"):
        c.write(0, s, qkv[:, :3], qkv[:, :3], _i32([0, 20]), 20)
    with pytest.raises(RuntimeError, match="one entry for each slot"):
        c.truncate(s, _i32([1, 2]))
    with pytest.raises(RuntimeError, match="keep must be"):
        c.compact(s, _i32([0]), _i32([1]))
    with pytest.raises(RuntimeError, match="no window"):
        c.evict(s)
    with pytest.raises(RuntimeError, match="count must be"):
        c.reserve(s, -1)
    c.free(_i32([0, -1]))
    c.check()


@pytest.mark.gpu
@pytest.mark.parametrize("graphed", [False, True])
def test_a_long_generation(graphed):
    """Prompt by the windowed attention, written to pages; rounds of drafted trees over the cache, accepted paths kept,
    pages behind the window given back; a beam forked off; each output against the dense windowed attention of the
    sequence so far (two kernels: twice the bounds). Once with the rounds' calls captured and replayed."""
    from flash_attn.flash_paged_attn_interface import pack_tree_mask
    from flash_attn.flash_window_attn_interface import flash_window_attn_unpadded_func
    from oracle import window_ref as ref
    from window_testutil import cu
    L, H, HK, D, W, N, T = 2, 8, 2, 64, 48, 5, 6
    g = torch.Generator(device="cuda").manual_seed(3)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda").bfloat16()
    c = _cache(L, 40, 16, HK, D, 4, 40, window_size=W, num_sinks=N)
    prompts = [70, 33]
    slots, pc = _i32([2, 0]), cu(prompts)
    hist = [[(rand(n, HK, D), rand(n, HK, D)) for n in prompts] for _ in range(L)]      # by layer and sequence
    c.reserve(slots, _i32(prompts))
    for l in range(L):
        k, v = (torch.cat([hist[l][b][i] for b in range(2)]) for i in range(2))
        q = rand(sum(prompts), H, D)
        out = flash_window_attn_unpadded_func(q, k, v, pc, pc, 70, 70, W, N)
        c.write(l, slots, k, v, pc, 70)
        assert torch.isfinite(out).all()
    c.compact(slots, _i32([list(range(70))] * 2), _i32(prompts))
    parents = [-1, 0, 0, 1, 1, 3]
    path = torch.zeros(T, T, dtype=torch.bool)
    for i, p in enumerate(parents):
        if p >= 0:
            path[i] |= path[p]
        path[i, i] = True
    tree = pack_tree_mask(path.repeat(2, 1)).cuda()
    tc = cu([T, T])
    q, k, v = rand(L, 2 * T, H, D), rand(L, 2 * T, HK, D), rand(L, 2 * T, HK, D)
    keep, counts = _i32([[0, 1, 3], [0, 2, 0]]), _i32([3, 2])

    def round_():
        c.reserve(slots, T)
        outs = []
        for l in range(L):
            c.write(l, slots, k[l], v[l], tc, T)
            outs.append(c.attend(l, q[l], slots, tc, T, max_context_len=200, tree_mask=tree))
        c.compact(slots, keep, counts)
        c.evict(slots)
        return torch.stack(outs)
    graph = None
    for n in range(12):
        if graphed and n == 2:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                held = round_()
        q.copy_(rand(*q.shape)), k.copy_(rand(*k.shape)), v.copy_(rand(*v.shape))
        kept = [[0, 1, 3], [0, 2]] if n % 2 else [[0, 2], [0]]
        keep.copy_(_i32([x + [0] * (3 - len(x)) for x in kept]))
        counts.copy_(_i32([len(x) for x in kept]))
        if graph is not None:
            graph.replay()
            got = held
        else:
            got = round_()
        c.check()
        for l in range(L):
            for b in range(2):
                kk = torch.cat([hist[l][b][0], k[l, b * T:b * T + T]])
                vv = torch.cat([hist[l][b][1], v[l, b * T:b * T + T]])
                m = len(hist[l][b][0])
                pos = m + path.sum(1).cuda() - 1
                kpos = torch.cat([torch.arange(m, device="cuda"), pos])
                live = torch.cat([torch.ones(T, m, dtype=torch.bool), path], 1).cuda()
                live &= (kpos > pos[:, None] - W) | (kpos < N)
                for h in range(H):
                    a = (q[l, b * T:b * T + T, h], kk[:, h // 4], vv[:, h // 4], live, D ** -0.5)
                    r, _, p = ref.attention(*a)
                    assert ((got[l, b * T:b * T + T, h].double() - r).abs() <= ref.bounds(*a, p, r)).all()
                rows = torch.tensor(kept[b], device="cuda") + b * T
                hist[l][b] = (torch.cat([hist[l][b][0], k[l][rows]]), torch.cat([hist[l][b][1], v[l][rows]]))
        assert c.seqlens[2].item() == len(hist[0][0][0]) and c.seqlens[0].item() == len(hist[0][1][0])
    held_pages = int((c.refcount > 0).sum())
    assert held_pages <= 2 * (-(-W // 16) + 1 + 1 + 1)      # the window's pages, the sinks', the last one
    # a beam off the first sequence: one token each, and the chain's answer by the windowed attention over all keys
    c.fork(_i32([2]), _i32([3]))
    both = _i32([2, 3])
    c.reserve(both, 1)
    k1, v1, q1 = rand(L, 2, HK, D), rand(L, 2, HK, D), rand(L, 2, H, D)
    m = len(hist[0][0][0])
    for l in range(L):
        c.write(l, both, k1[l], v1[l], cu([1, 1]), 1)
    for l in range(L):
        got = c.attend(l, q1[l], both, cu([1, 1]), 1)
        kk = torch.cat([torch.cat([hist[l][0][0], k1[l, b:b + 1]]) for b in range(2)])
        vv = torch.cat([torch.cat([hist[l][0][1], v1[l, b:b + 1]]) for b in range(2)])
        want = flash_window_attn_unpadded_func(q1[l], kk, vv, cu([1, 1]), cu([m + 1, m + 1]), 1, m + 1, W, N)
        for b in range(2):
            for h in range(H):
                s = slice(b * (m + 1), (b + 1) * (m + 1))
                live = ref.seen(torch.tensor([m], device="cuda"), torch.arange(m + 1, device="cuda"), W, N)
                a = (q1[l, b:b + 1, h], kk[s, h // 4], vv[s, h // 4], live, D ** -0.5)
                r, _, p = ref.attention(*a)
                e = ref.bounds(*a, p, r)
                assert ((got[b:b + 1, h].double() - want[b:b + 1, h].double()).abs() <= 2 * e).all()
    c.check()
    c.free(_i32([0, 2, 3]))
    assert not c.refcount.any() and (c.block_table == -1).all()
    c.check()


_FIRST_CALL_CAPTURED = """
import sys
sys.path[:0] = sys.argv[1:]
import torch
from flash_attn.flash_window_attn_interface import flash_window_attn_unpadded_func as window
from flash_attn.paged_kv_cache import PagedKVCache
i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
torch.manual_seed(0)
q, k, v, dout = (torch.randn(300, h, 64, device="cuda").bfloat16().requires_grad_() for h in (4, 2, 2, 4))
cu = i32([0, 100, 300])
cache = PagedKVCache(1, 64, 16, 2, 64, 4, 8, window_size=40, num_sinks=2)
slots, cu2, keep, counts = i32([2, 0]), i32([0, 50, 100]), i32([list(range(50))] * 2), i32([50, 50])
kn, vn, qn = (torch.randn(100, h, 64, device="cuda").bfloat16() for h in (2, 2, 4))

def step():
    out = window(q, k, v, cu, cu, 200, 200, 40, 2)
    grads = torch.autograd.grad(out, (q, k, v), dout)
    cache.truncate(slots, i32_zero)
    cache.reserve(slots, 50)
    cache.write(0, slots, kn, vn, cu2, 50)
    o = cache.attend(0, qn, slots, cu2, 50)
    cache.compact(slots, keep, counts)
    cache.evict(slots)
    return [out.detach(), *grads, o, cache.block_table.clone(), cache.seqlens.clone(), cache.refcount.clone()]

i32_zero = i32([0, 0])
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = step()
replays = []
for _ in range(3):
    graph.replay()
    replays.append([x.clone() for x in got])
    torch.cuda.synchronize()
want = step()
for r in replays:
    for x, y in zip(r, want):
        assert torch.equal(x, y)
cache.check()
print("ok")
"""


@pytest.mark.gpu
def test_first_calls_of_a_process_inside_a_capture():
    """A fresh process whose first windowed, paged and cache calls are captured: every replay gives the eager results."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", _FIRST_CALL_CAPTURED, os.path.join(root, "hazyresearch_flash-attention_amd")],
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.split()[-1] == "ok", r.stdout[-2000:] + r.stderr[-4000:]
