"""Workloads of the windowed-attention and paged-cache operators, with their plain forms.

Three operators that a long-generation user calls next to each other:

* window: causal attention of var-len sequences where a query sees the `window` newest keys up to its own
  position and the first `sinks` keys; a query's position is aligned to the end of its keys. Forward alone
  (a prompt) and forward with backward (training); query heads share key/value heads in groups.
* paged: attention of new tokens (one, or a tree of drafted ones) over a cache held in pages, the same window.
* fork / commit: a cache's own upkeep. fork frees beams, cuts their parents back to the prompt, lets the beams share
  the parents' pages and makes room for one more token each (which copies a shared page that is only partly full). commit makes room for drafted tokens,
  writes them in every layer, keeps the accepted ones, moved together, and takes the step back again, so that a
  pass leaves the lengths as they were.

`listed()` and `draw()` give cases, `prepare()` the tensors a program has in hand, `run()` one pass, in the plain
form (`own = False`) or through the package's entry points (`own = True`); `exact()` is the definition in 64 bits.
"""
import math
import os
import sys

import numpy as np
import torch

own = False
DEV = "cuda"
PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "hazyresearch_flash-attention_amd")
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _package():
    if PKG not in sys.path:
        sys.path.insert(0, PKG)
    from flash_attn import flash_paged_attn_interface, flash_window_attn_interface, paged_kv_cache
    return flash_window_attn_interface, flash_paged_attn_interface, paged_kv_cache


# ------------------------------------------------------------------------------------------ cases
def _window(name, dtype, batch, seqlen, ragged, past, heads, kv_heads, head_dim, window, sinks, train):
    return {"name": name, "op": "window", "dtype": dtype, "batch": batch, "seqlen": seqlen, "ragged": ragged,
            "past": past, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "window": window,
            "sinks": sinks, "train": train}


def _paged(name, dtype, batch, context, ragged, tokens, tree, heads, kv_heads, head_dim, page, window, sinks):
    return {"name": name, "op": "paged", "dtype": dtype, "batch": batch, "context": context, "ragged": ragged,
            "tokens": tokens, "tree": tree, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "page": page, "window": window, "sinks": sinks}


def _cache(name, op, dtype, batch, context, tokens, layers, kv_heads, head_dim, page):
    return {"name": name, "op": op, "dtype": dtype, "batch": batch, "context": context, "tokens": tokens,
            "layers": layers, "kv_heads": kv_heads, "head_dim": head_dim, "page": page}


def listed():
    return [
        # the benchmark's layer (8 x 2048 tokens, 12 heads of 64) trained with a local window
        _window("train_bench_layer", "bf16", 8, 2048, False, 0, 12, 12, 64, 256, 4, True),
        # a long document of a model with grouped heads
        _window("train_long_grouped", "bf16", 1, 8192, False, 0, 16, 4, 128, 1024, 16, True),
        # a ragged batch of short samples, an odd head count and head size
        _window("train_ragged_fp16", "fp16", 5, 701, True, 0, 6, 2, 80, 100, 3, True),
        # a long prompt read in one pass
        _window("prompt_32k", "bf16", 1, 32768, False, 0, 8, 2, 128, 4096, 64, False),
        # one user, one token: latency
        _paged("decode_one", "bf16", 1, 1023, False, 1, False, 12, 4, 64, 16, 0, 0),
        # a server's batch of single tokens over long caches
        _paged("decode_batch", "bf16", 64, 8191, True, 1, False, 32, 8, 128, 64, 0, 0),
        # trees of 64 drafted tokens over long caches, windowed
        _paged("tree_64", "bf16", 8, 32000, True, 64, True, 32, 8, 128, 64, 8192, 64),
        # a small odd tree, ungrouped heads
        _paged("tree_25_fp16", "fp16", 3, 2049, True, 25, True, 12, 12, 64, 16, 0, 0),
        # one prompt to four beams
        _cache("fork_small", "fork", "bf16", 4, 203, 1, 4, 4, 64, 16),
        # a server's beams over all layers of a model
        _cache("fork_large", "fork", "bf16", 64, 1080, 1, 12, 8, 128, 64),
        # trees of drafts verified, for a server's batch
        _cache("commit_large", "commit", "bf16", 32, 997, 64, 12, 8, 128, 64),
        # one user's drafts verified
        _cache("commit_small", "commit", "bf16", 1, 500, 16, 4, 4, 64, 16),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["window", "window", "paged", "paged", "fork", "commit"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    kv = rng.choice([1, 2, 4, 8])
    dim = rng.choice([32, 64, 64, 80, 128, 128])
    if op == "window":
        batch = _log(rng, 1, 8)
        case = _window("", dtype, batch, _log(rng, 1, 4096 // batch * 2), rng.random() < 0.6,
                       rng.choice([0, 0, _log(rng, 1, 2000)]), kv * rng.choice([1, 2, 3, 4]), kv, dim,
                       _log(rng, 1, 1500), rng.choice([0, 1, 4, 40, 100]), rng.random() < 0.6)
        case["heads"], case["kv_heads"] = min(case["heads"], 16), min(kv, 4)
        case["heads"] -= case["heads"] % case["kv_heads"]
    elif op == "paged":
        tokens = rng.choice([1, 1, _log(rng, 2, 64)])
        case = _paged("", dtype, _log(rng, 1, 16), _log(rng, 1, 16000), rng.random() < 0.7, tokens, tokens > 1,
                      kv * rng.choice([1, 2, 4, 7, 8]), kv, dim, rng.choice([16, 32, 64, 128]),
                      rng.choice([0, 0, _log(rng, 16, 9000)]), rng.choice([0, 4, 70]))
    else:
        case = _cache("", op, dtype, _log(rng, 1, 32), _log(rng, 2, 1000), 1 if op == "fork" else _log(rng, 1, 64),
                      _log(rng, 1, 16), min(kv, 4), dim, rng.choice([16, 32, 64]))
    del case["name"]
    return case


def _lens(batch, longest, ragged):
    """Lengths of a batch: `longest` first, then (ragged) spread over [1, longest] by the golden ratio."""
    if not ragged:
        return [longest] * batch
    return [longest if i == 0 else max(1, int(longest * ((i * 0.6180339887498949) % 1.0))) for i in range(batch)]


def _seen(pos, window, sinks):
    """How many keys a query at position `pos` sees."""
    lo = max(0, pos - window + 1) if window else 0
    return pos - lo + 1 + min(sinks, lo)


def work(case):
    """Bytes and operations of one pass: every input read once, every output written once."""
    if case["op"] == "window":
        d, hq, hk = case["head_dim"], case["heads"], case["kv_heads"]
        pairs = rows = keys = 0
        for n in _lens(case["batch"], case["seqlen"], case["ragged"]):
            rows, keys = rows + n, keys + n + case["past"]
            pairs += sum(_seen(i + case["past"], case["window"], case["sinks"]) for i in range(n))
        fwd = 2 * d * (2 * rows * hq + 2 * keys * hk)
        if not case["train"]:
            return {"bytes": fwd, "flops": 4 * pairs * hq * d}
        return {"bytes": fwd + 2 * d * (4 * rows * hq + 4 * keys * hk) - 2 * d * (rows * hq), "flops": 14 * pairs * hq * d}
    if case["op"] == "paged":
        d, hq, hk, t = case["head_dim"], case["heads"], case["kv_heads"], case["tokens"]
        pairs = keys = 0
        for n in _lens(case["batch"], case["context"], case["ragged"]):
            w = case["window"]
            keys += (min(n, w + case["sinks"]) if w else n) + t
            pairs += sum(_seen(n + i, w, case["sinks"]) for i in range(t))
        return {"bytes": 2 * d * (2 * case["batch"] * t * hq + 2 * keys * hk), "flops": 4 * pairs * hq * d}
    row = 2 * 2 * case["kv_heads"] * case["head_dim"] * case["layers"]     # one token's K and V in every layer
    if case["op"] == "fork":
        copied = 3 * case["batch"] * (case["context"] % case["page"])      # the last holder keeps the page
        held = 4 * case["batch"] * -(-case["context"] // case["page"])     # their entries, and the pages' counts
        return {"bytes": 2 * copied * row + 16 * held, "flops": 0}
    kept = max(1, case["tokens"] // 4)
    return {"bytes": 2 * case["batch"] * (case["tokens"] + kept) * row, "flops": 0}


# ------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed * 7919 + 17)


def _randn(g, shape, dtype):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32).to(dtype)


def _cu(lens):
    return torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device=DEV)


def _tree(seed, lens, tokens, tree):
    """Bit masks (rows, words) of each drafted token's path: itself and its ancestors, parents drawn at random."""
    words = (tokens + 63) // 64
    rs = np.random.RandomState((seed * 31 + 5) % 2 ** 32)
    mask = np.zeros((len(lens) * tokens, words), dtype=np.uint64)
    for b in range(len(lens)):
        for i in range(tokens):
            row = mask[b * tokens + i]
            parent = (rs.randint(-1, i) if i else -1) if tree else i - 1
            if parent >= 0:
                row |= mask[b * tokens + parent]
            row[i // 64] |= np.uint64(1) << np.uint64(i % 64)
    return torch.from_numpy(mask.view(np.int64)).to(DEV)


def prepare(case, seed):
    g, dt = _gen(seed), TYPES[case["dtype"]]
    d, hk = case["head_dim"], case["kv_heads"]
    s = {"case": case, "scale": d ** -0.5}
    if case["op"] == "window":
        ql = _lens(case["batch"], case["seqlen"], case["ragged"])
        kl = [n + case["past"] for n in ql]
        s.update(ql=ql, kl=kl, cu_q=_cu(ql), cu_k=_cu(kl), q=_randn(g, (sum(ql), case["heads"], d), dt),
                 k=_randn(g, (sum(kl), hk, d), dt), v=_randn(g, (sum(kl), hk, d), dt))
        if case["train"]:
            s["dout"] = _randn(g, (sum(ql), case["heads"], d), dt)
            if own:
                for n in "qkv":
                    s[n].requires_grad_()
        return s
    batch, page, t = case["batch"], case["page"], case["tokens"]
    if case["op"] == "paged":
        ctx = _lens(batch, case["context"], case["ragged"])
        blocks = [-(-(n + t) // page) for n in ctx]
        pages = sum(blocks) + 3
        order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
        table = torch.full((batch, max(blocks)), -1, dtype=torch.int32, device=DEV)
        at = 0
        for b, n in enumerate(blocks):
            table[b, :n] = order[at:at + n]
            at += n
        s.update(ctx=ctx, table=table, context=torch.tensor(ctx, dtype=torch.int32, device=DEV),
                 cu_q=_cu([t] * batch), k=_randn(g, (pages, page, hk, d), dt), v=_randn(g, (pages, page, hk, d), dt),
                 q=_randn(g, (batch * t, case["heads"], d), dt), max_context=case["context"],
                 tree=_tree(seed, ctx, t, True) if case["tree"] else None)
        return s
    # a cache: `batch` sequences hold pages; fork gives each of them three beams more
    seqs = 4 * batch if case["op"] == "fork" else batch
    ctx = case["context"]
    blocks = -(-ctx // page)
    width = -(-(ctx + t) // page) + 1
    pages = batch * blocks + seqs * (width - blocks + 1) + 5
    L = case["layers"]
    if own:
        cache = _package()[2].PagedKVCache(L, pages, page, hk, d, seqs, width, dtype=dt, device=DEV)
    else:
        class Plain:
            pass
        cache = Plain()
        cache.k = torch.empty((L, pages, page, hk, d), dtype=dt, device=DEV)
        cache.v = torch.empty_like(cache.k)
        cache.block_table = torch.empty((seqs, width), dtype=torch.int32, device=DEV)
        cache.seqlens = torch.empty(seqs, dtype=torch.int32, device=DEV)
        cache.nblocks = torch.empty(seqs, dtype=torch.int32, device=DEV)
        cache.refcount = torch.empty(pages, dtype=torch.int32, device=DEV)
    for l in range(L):
        cache.k[l].copy_(_randn(g, cache.k.shape[1:], dt))
        cache.v[l].copy_(_randn(g, cache.v.shape[1:], dt))
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)[:batch * blocks].view(batch, blocks)
    cache.block_table.fill_(-1)
    cache.block_table[:batch, :blocks] = order
    cache.seqlens.zero_()
    cache.seqlens[:batch] = ctx
    cache.nblocks.zero_()
    cache.nblocks[:batch] = blocks
    cache.refcount.zero_()
    cache.refcount[order.flatten().long()] = 1
    s["cache"] = cache
    s["slots"] = torch.arange(seqs, dtype=torch.int32, device=DEV)
    if case["op"] == "fork":
        s["parents"] = s["slots"][:batch].repeat_interleave(3)
        s["children"] = s["slots"][batch:].clone()
        s["roots"], s["prompt"] = s["slots"][:batch].clone(), cache.seqlens[:batch].clone()
        s["beams"] = torch.cat([s["children"], s["roots"]])         # a parent comes last and keeps its own page
    else:
        rs = np.random.RandomState((seed * 13 + 1) % 2 ** 32)
        most = max(1, t // 4)
        keep = np.stack([np.sort(rs.permutation(t)[:most]) for _ in range(batch)]).astype(np.int32)
        s.update(keep=torch.from_numpy(keep).to(DEV), cu=_cu([t] * batch), lens=cache.seqlens.clone(),
                 counts=torch.from_numpy(rs.randint(1, most + 1, batch).astype(np.int32)).to(DEV),
                 knew=_randn(g, (L, batch * t, hk, d), dt), vnew=_randn(g, (L, batch * t, hk, d), dt))
    return s


# ------------------------------------------------------------------------------------------ plain forms
CHUNK = 512    # query rows worked on at once


def _plain_window(s):
    c = s["case"]
    q, k, v, dt = s["q"], s["k"], s["v"], s["q"].dtype
    hk, d, G = c["kv_heads"], c["head_dim"], c["heads"] // c["kv_heads"]
    out = torch.empty_like(q)
    train = c["train"]
    if train:
        dq = torch.empty_like(q)
        dk = torch.zeros(k.shape, dtype=torch.float32, device=DEV)
        dv = torch.zeros_like(dk)
    q0 = k0 = 0
    for n, m in zip(s["ql"], s["kl"]):
        kf, vf = k[k0:k0 + m].float(), v[k0:k0 + m].float()
        for i in range(0, n, CHUNK):
            e = min(n, i + CHUNK)
            pos = torch.arange(i, e, device=DEV) + (m - n)
            lo, hi = max(0, i + m - n - c["window"] + 1), e + m - n
            cols = torch.cat([torch.arange(min(c["sinks"], lo), device=DEV), torch.arange(lo, hi, device=DEV)])
            kk = kf[cols].transpose(0, 1).contiguous()                      # (hk, keys, d)
            vv = vf[cols].transpose(0, 1).contiguous()
            grouped = lambda x: x[q0 + i:q0 + e].float().view(e - i, hk, G, d).permute(1, 2, 0, 3).reshape(hk, -1, d).contiguous()
            qq = grouped(q)                                                 # (hk, G rows, d)
            dead = (cols > pos[:, None]) | ((cols <= pos[:, None] - c["window"]) & (cols >= c["sinks"]))
            p = torch.matmul(qq, kk.transpose(1, 2).contiguous()).mul_(s["scale"]).view(hk, G, e - i, -1)
            p.masked_fill_(dead, -math.inf)
            p.sub_(p.amax(-1, keepdim=True)).exp_()
            p.div_(p.sum(-1, keepdim=True))
            p = p.view(hk, G * (e - i), -1)
            back = lambda x: x.view(hk, G, e - i, d).permute(2, 0, 1, 3).reshape(e - i, -1, d).to(dt)
            o = torch.matmul(p, vv)
            out[q0 + i:q0 + e] = back(o)
            if train:
                do = grouped(s["dout"])
                ds = torch.matmul(do, vv.transpose(1, 2).contiguous())
                ds.sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(s["scale"])
                dq[q0 + i:q0 + e] = back(torch.matmul(ds, kk))
                dk[k0 + cols] += torch.matmul(ds.transpose(1, 2).contiguous(), qq).transpose(0, 1)
                dv[k0 + cols] += torch.matmul(p.transpose(1, 2).contiguous(), do).transpose(0, 1)
        q0, k0 = q0 + n, k0 + m
    return {"out": out, "dq": dq, "dk": dk.to(dt), "dv": dv.to(dt)} if train else {"out": out}


def _bits(tree, t):
    """(rows, t) truth values of bit masks."""
    at = torch.arange(t, device=DEV)
    return (tree[:, at // 64] >> (at % 64)) & 1 != 0


def _plain_paged(s):
    c = s["case"]
    t, page, hk, d = c["tokens"], c["page"], c["kv_heads"], c["head_dim"]
    G, dt = c["heads"] // hk, s["q"].dtype
    w = c["window"] or 1 << 30
    out = torch.empty_like(s["q"])
    path = _bits(s["tree"], t) if c["tree"] else torch.ones(t, t, device=DEV).tril().bool().repeat(c["batch"], 1)
    depth = path.sum(1)
    for b, n in enumerate(s["ctx"]):
        lo = max(0, n - w + 1)
        cols = torch.cat([torch.arange(min(c["sinks"], lo), device=DEV), torch.arange(lo, n + t, device=DEV)])
        rows = s["table"][b].long()[cols // page] * page + cols % page
        kk = s["k"].view(-1, hk, d)[rows].float().transpose(0, 1).contiguous()
        vv = s["v"].view(-1, hk, d)[rows].float().transpose(0, 1).contiguous()
        mine = slice(b * t, b * t + t)
        at = n + depth[mine] - 1                                            # positions of the new tokens
        where = torch.cat([cols[:-t], at])                                  # positions of the keys
        live = torch.cat([torch.ones(t, len(cols) - t, dtype=torch.bool, device=DEV), path[mine]], 1)
        live &= (where > at[:, None] - w) | (where < c["sinks"])
        qq = s["q"][mine].float().view(t, hk, G, d).permute(1, 2, 0, 3).reshape(hk, G * t, d)
        p = torch.matmul(qq, kk.transpose(1, 2).contiguous()).mul_(s["scale"]).view(hk, G, t, -1)
        p = torch.softmax(p.masked_fill_(~live, -math.inf), -1).view(hk, G * t, -1)
        out[mine] = torch.matmul(p, vv).view(hk, G, t, d).permute(2, 0, 1, 3).reshape(t, -1, d).to(dt)
    return {"out": out}


def _plain_reserve(c, slots, count):
    """Room for `count` more tokens of each sequence: the lowest free pages, in the order of the sequences; a
    partly full page that others hold too is left to them and its rows copied."""
    page = c.k.shape[2]
    free = torch.nonzero(c.refcount == 0).flatten().tolist()
    lens, have, table, refs = c.seqlens.tolist(), c.nblocks.tolist(), c.block_table.tolist(), c.refcount.tolist()
    src, dst, part, put, at = [], [], [], [], 0
    for i in slots.tolist():
        n = lens[i]
        b = n // page
        if n % page and refs[table[i][b]] > 1:
            refs[table[i][b]] -= 1
            src.append(table[i][b]), dst.append(free[at]), part.append(n % page), put.append((i, b, free[at]))
            at += 1
        for b in range(have[i], -(-(n + count) // page)):
            put.append((i, b, free[at]))
            at += 1
        have[i] = max(have[i], -(-(n + count) // page))
    for _, _, p in put:
        refs[p] = 1
    if put:
        i, b, p = torch.tensor(put, device=DEV).unbind(1)
        c.block_table[i, b] = p.to(torch.int32)
    c.nblocks.copy_(torch.tensor(have, dtype=torch.int32))
    c.refcount.copy_(torch.tensor(refs, dtype=torch.int32))
    if src:
        src, dst, part = (torch.tensor(x, device=DEV) for x in (src, dst, part))
        rows = torch.arange(page, device=DEV)
        for x in (c.k, c.v):
            take = (rows < part[:, None])[None, :, :, None, None]
            x[:, dst] = torch.where(take, x[:, src], x[:, dst])


def _plain_cut(c, slots, lens):
    """Sequences shortened to `lens`; the pages behind are given back."""
    page = c.k.shape[2]
    need = -(-lens // page)
    col = torch.arange(c.block_table.shape[1], device=DEV)
    rows = c.block_table[slots.long()]
    gone = (col >= need[:, None]) & (rows >= 0)
    c.refcount.index_add_(0, rows[gone].long(), torch.full((int(gone.sum()),), -1, dtype=torch.int32, device=DEV))
    c.block_table[slots.long()] = torch.where(gone, -1, rows)
    c.nblocks[slots.long()] = torch.minimum(c.nblocks[slots.long()], need)
    c.seqlens[slots.long()] = lens


def _places(c, slots, first, offsets):
    """Rows of the pool (pages flattened) of tokens first + offsets of each sequence."""
    page = c.k.shape[2]
    at = first[:, None] + offsets
    return c.block_table[slots.long()[:, None], at // page].long() * page + at % page


def _state_of(c):
    return {"k": c.k, "v": c.v, "block_table": c.block_table, "seqlens": c.seqlens, "nblocks": c.nblocks,
            "refcount": c.refcount}


def _plain_fork(s):
    c = s["cache"]
    page = c.k.shape[2]
    par, kid = s["parents"].long(), s["children"].long()
    _plain_cut(c, s["children"], torch.zeros_like(s["children"]))
    _plain_cut(c, s["roots"], s["prompt"])
    need = -(-c.seqlens[par] // page)
    col = torch.arange(c.block_table.shape[1], device=DEV)
    rows = torch.where(col < need[:, None], c.block_table[par], -1)
    c.block_table[kid] = rows
    c.seqlens[kid] = c.seqlens[par]
    c.nblocks[kid] = need
    held = rows[rows >= 0].long()
    c.refcount.index_add_(0, held, torch.ones(len(held), dtype=torch.int32, device=DEV))
    _plain_reserve(c, s["beams"], 1)
    return _state_of(c)


def _plain_commit(s):
    c, t = s["cache"], s["case"]["tokens"]
    slots, L = s["slots"], s["case"]["layers"]
    _plain_reserve(c, slots, t)
    n = c.seqlens[slots.long()]
    rows = _places(c, slots, n, torch.arange(t, device=DEV)).flatten()
    for l in range(L):
        c.k[l].view(-1, *c.k.shape[3:])[rows] = s["knew"][l]
        c.v[l].view(-1, *c.v.shape[3:])[rows] = s["vnew"][l]
    live = torch.arange(s["keep"].shape[1], device=DEV) < s["counts"][:, None]
    src = _places(c, slots, n, s["keep"])[live]
    dst = _places(c, slots, n, torch.arange(s["keep"].shape[1], device=DEV).expand_as(s["keep"]))[live]
    for x in (c.k, c.v):
        flat = x.view(L, -1, *x.shape[3:])
        flat[:, dst] = flat[:, src]
    _plain_cut(c, slots, n + s["counts"])
    _plain_cut(c, slots, s["lens"])
    return _state_of(c)


# ------------------------------------------------------------------------------------------ one pass
def run(s):
    c = s["case"]
    if not own:
        return {"window": _plain_window, "paged": _plain_paged, "fork": _plain_fork, "commit": _plain_commit}[c["op"]](s)
    window, paged, _ = _package()
    if c["op"] == "window":
        out = window.flash_window_attn_unpadded_func(
            s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], c["seqlen"], c["seqlen"] + c["past"], c["window"], c["sinks"])
        if not c["train"]:
            return {"out": out}
        dq, dk, dv = torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["dout"])
        return {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv}
    if c["op"] == "paged":
        return {"out": paged.flash_paged_attn_func(
            s["q"], s["k"], s["v"], s["table"], s["context"], s["cu_q"], c["tokens"], max_context_len=s["max_context"],
            tree_mask=s["tree"], window_size=c["window"] or None, num_sinks=c["sinks"])}
    cache = s["cache"]
    if c["op"] == "fork":
        cache.free(s["children"])
        cache.truncate(s["roots"], s["prompt"])
        cache.fork(s["parents"], s["children"])
        cache.reserve(s["beams"], 1)
    else:
        cache.reserve(s["slots"], c["tokens"])
        for l in range(c["layers"]):
            cache.write(l, s["slots"], s["knew"][l], s["vnew"][l], s["cu"], c["tokens"])
        cache.compact(s["slots"], s["keep"], s["counts"])
        cache.truncate(s["slots"], s["lens"])
    return _state_of(cache)


# ------------------------------------------------------------------------------------------ the definition
def _exact_attention(q, k, v, live, scale):
    """softmax(scale q k^T) v with the dead entries taken out; rows without a live key are 0. (heads, rows, d)."""
    a = (q @ k.mT.contiguous()) * scale
    a = torch.where(live, a, torch.full_like(a, -math.inf))
    top = a.detach().amax(-1, keepdim=True)
    e = torch.where(live, torch.exp(a - torch.where(torch.isinf(top), 0.0, top)), 0.0)
    total = e.sum(-1, keepdim=True)
    return (e / torch.where(total == 0, 1.0, total)) @ v


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "window":
        G = case["heads"] // case["kv_heads"]
        x = [s[n].detach().double() for n in "qkv"]
        res = {"out": torch.zeros_like(x[0])}
        if case["train"]:
            res.update(dq=torch.zeros_like(x[0]), dk=torch.zeros_like(x[1]), dv=torch.zeros_like(x[2]))
        q0 = k0 = 0
        for n, m in zip(s["ql"], s["kl"]):
            for h in range(case["heads"]):
                for i in range(0, n, 2048):
                    sl = slice(q0 + i, q0 + min(n, i + 2048))
                    q = x[0][sl, h].contiguous().requires_grad_(case["train"])
                    k = x[1][k0:k0 + m, h // G].contiguous().requires_grad_(case["train"])
                    v = x[2][k0:k0 + m, h // G].contiguous().requires_grad_(case["train"])
                    back = (torch.arange(i, i + len(q), device=DEV) + m - n)[:, None] - torch.arange(m, device=DEV)
                    live = (back >= 0) & ((back < case["window"]) | (torch.arange(m, device=DEV) < case["sinks"]))
                    with torch.enable_grad():
                        o = _exact_attention(q, k, v, live, s["scale"])
                    res["out"][sl, h] = o.detach()
                    if case["train"]:
                        gq, gk, gv = torch.autograd.grad(o, (q, k, v), s["dout"][sl, h].double())
                        res["dq"][sl, h] = gq
                        res["dk"][k0:k0 + m, h // G] += gk
                        res["dv"][k0:k0 + m, h // G] += gv
            q0, k0 = q0 + n, k0 + m
        return res
    if case["op"] == "paged":
        t, page, G = case["tokens"], case["page"], case["heads"] // case["kv_heads"]
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
        masks = s["tree"].cpu().numpy().view(np.uint64) if case["tree"] else None
        for b, n in enumerate(s["ctx"]):
            pages = s["table"][b, :-(-(n + t) // page)].long()
            k = s["k"][pages].double().flatten(0, 1)[:n + t]
            v = s["v"][pages].double().flatten(0, 1)[:n + t]
            path = np.zeros((t, t), dtype=bool)
            for i in range(t):
                for j in range(t):
                    path[i, j] = (int(masks[b * t + i, j // 64]) >> (j % 64)) & 1 if case["tree"] else j <= i
            depth = path.sum(1) - 1
            kpos = np.concatenate([np.arange(n), n + depth])
            qpos = (n + depth)[:, None]
            live = np.concatenate([np.ones((t, n), dtype=bool), path], 1)
            if case["window"]:
                live &= (qpos - kpos < case["window"]) | (kpos < case["sinks"])
            live = torch.from_numpy(live).to(DEV)
            for h in range(case["heads"]):
                q = s["q"][b * t:b * t + t, h].double()
                out[b * t:b * t + t, h] = _exact_attention(q, k[:, h // G].contiguous(), v[:, h // G].contiguous(), live, s["scale"])
        return {"out": out}
    # the cache, one entry at a time on the host
    c, page, t = s["cache"], case["page"], case["tokens"]
    table, lens, have = c.block_table.tolist(), c.seqlens.tolist(), c.nblocks.tolist()
    refs = c.refcount.tolist()
    k, v = c.k.clone(), c.v.clone()

    def take():
        p = refs.index(0)
        refs[p] = 1
        return p

    def room(i, count):
        n = lens[i]
        fresh = []
        if n % page and refs[table[i][n // page]] > 1:
            fresh.append((i, n // page, table[i][n // page]))
            refs[table[i][n // page]] -= 1
        for b in range(have[i], (n + count + page - 1) // page):
            fresh.append((i, b, None))
            have[i] = b + 1
        return fresh

    if case["op"] == "fork":
        for p, i in zip(s["parents"].tolist(), s["children"].tolist()):
            lens[i], have[i] = lens[p], (lens[p] + page - 1) // page
            for b in range(have[i]):
                table[i][b] = table[p][b]
                refs[table[i][b]] += 1
    fresh = []
    for i in s["beams" if case["op"] == "fork" else "slots"].tolist():
        fresh += room(i, t)
    for i, b, old in fresh:
        table[i][b] = take()
        if old is not None:
            n = lens[i] % page
            k[:, table[i][b], :n] = k[:, old, :n]
            v[:, table[i][b], :n] = v[:, old, :n]
    if case["op"] == "commit":
        for i in s["slots"].tolist():
            at = [table[i][(lens[i] + j) // page] * page + (lens[i] + j) % page for j in range(t)]
            kept = s["keep"][i, :s["counts"][i]].tolist()
            for pool, new in ((k, s["knew"]), (v, s["vnew"])):
                flat, mine = pool.view(case["layers"], -1, *pool.shape[3:]), new[:, i * t:i * t + t]
                flat[:, at] = mine
                flat[:, at[:len(kept)]] = mine[:, kept]
            for b in range((lens[i] + page - 1) // page, have[i]):
                refs[table[i][b]] -= 1
                table[i][b] = -1
            have[i] = (lens[i] + page - 1) // page
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    return {"k": k.double(), "v": v.double(), "block_table": ints(table), "seqlens": ints(lens), "nblocks": ints(have),
            "refcount": ints(refs)}
