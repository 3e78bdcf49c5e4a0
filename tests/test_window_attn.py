"""Windowed attention with sinks (flash_window_attn_interface): values and gradients against a 64-bit plain form within
bounds that count the kernels' roundings, masks and lengths where it can go wrong, refusals."""
import ctypes
import math
import os

import pytest
import torch

from oracle import window_ref as ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _func():
    from flash_attn.flash_window_attn_interface import flash_window_attn_unpadded_func
    return flash_window_attn_unpadded_func


# ---------------------------------------------------------------------------------------- CPU
def test_reference_gradients_against_differences():
    """The plain form's gradient formulas against central differences of its outputs, in 64 bits."""
    g = torch.Generator().manual_seed(0)
    q, k, v, dout = (torch.randn(n, 5, generator=g, dtype=torch.float64) for n in (7, 9, 9, 7))
    live = ref.seen(torch.arange(7) + 2 - 4, torch.arange(9), 3, 2)     # the first rows see nothing
    assert not live[0].any() and live.any()
    loss = lambda a, b, c: (ref.attention(a, b, c, live, 0.4)[0] * dout).sum().item()
    out, _, p = ref.attention(q, k, v, live, 0.4)
    grads = ref.gradients(q, k, v, live, 0.4, p, out, dout)[:3]
    for i, x in enumerate((q, k, v)):
        for at in range(x.numel()):
            step = torch.zeros_like(x).view(-1)
            step[at] = 1e-5
            args = [[q, k, v], [q, k, v]]
            args[0][i], args[1][i] = x + step.view_as(x), x - step.view_as(x)
            diff = (loss(*args[0]) - loss(*args[1])) / 2e-5
            assert abs(diff - grads[i].view(-1)[at].item()) < 1e-8


def test_reference_ignores_what_a_row_does_not_see():
    q, k, v = (torch.randn(6, 4, dtype=torch.float64) for _ in range(3))
    live = ref.seen(torch.arange(6), torch.arange(6), 2, 0)
    want = ref.attention(q, k, v, live, 1.0)[0]
    k[0], v[0] = math.nan, math.inf
    got = ref.attention(q, k, v, live, 1.0)[0]
    assert torch.equal(got[2:], want[2:])


def _refused(match, **kw):
    q = torch.zeros(4, 4, 64, dtype=torch.bfloat16)
    c = torch.tensor([0, 4], dtype=torch.int32)
    a = dict(q=q, k=q, v=q, cu_seqlens_q=c, cu_seqlens_k=c, max_seqlen_q=4, max_seqlen_k=4, window_size=2)
    a.update(kw)
    with pytest.raises(RuntimeError, match=match):
        _func()(**a)


def test_refusals_before_any_launch():
    _refused("must be on the GPU")
    _refused("window_size must be None or at least 1", window_size=0)
    _refused("num_sinks must be at least 0", num_sinks=-1)


def _abi():
    from flash_attn import flash_attn_hip as hip
    L = hip.lib()
    i64, i32, vp, f32 = ctypes.c_int64, ctypes.c_int32, ctypes.c_void_p, ctypes.c_float

    class Args(ctypes.Structure):
        _fields_ = [(n, vp) for n in ("q k v o softmax_lse cu_seqlens_q cu_seqlens_k dout dq dk dv workspace").split()] + \
            [("workspace_bytes", i64)] + \
            [(f"{n}_{s}_stride", i64) for n in ("q", "k", "v", "o", "do", "dq", "dk", "dv") for s in ("row", "head")] + \
            [("total_q", i64), ("total_k", i64)] + \
            [(n, i32) for n in "batch nheads nheads_k head_dim max_seqlen_q max_seqlen_k lse_stride window num_sinks".split()] + \
            [("softmax_scale", f32), ("dtype", i32), ("reserved", i32)]
    L.fa_window_args_size.restype = i64
    L.fa_window_bwd_workspace.restype = i64
    return L, Args


def _valid(Args):
    a = Args()
    for n in "q k v o softmax_lse cu_seqlens_q cu_seqlens_k dout dq dk dv workspace".split():
        setattr(a, n, 4096)
    for n in ("q", "k", "v", "o", "do", "dq", "dk", "dv"):
        setattr(a, n + "_row_stride", 128)
        setattr(a, n + "_head_stride", 64)
    a.total_q = a.total_k = 8
    a.batch, a.nheads, a.nheads_k, a.head_dim = 1, 2, 2, 64
    a.max_seqlen_q = a.max_seqlen_k = a.lse_stride = 8
    a.window, a.softmax_scale, a.dtype = 4, 0.125, 1
    return a


@pytest.mark.parametrize("change, text", [
    ({"dtype": 2}, "dtype"), ({"batch": 0}, "batch_size"), ({"batch": 70000}, "batch_size"), ({"nheads": 3}, "multiple of nheads_k"),
    ({"nheads_k": 0}, "nheads_k"), ({"head_dim": 36}, "head_size"), ({"head_dim": 136}, "head_size"),
    ({"window": -1}, "window"), ({"num_sinks": -2}, "num_sinks"), ({"softmax_scale": math.inf}, "finite"),
    ({"softmax_scale": math.nan}, "finite"), ({"lse_stride": 4}, "lse_stride"), ({"q": 0}, "q is NULL"), ({"k": 0}, "k is NULL"),
    ({"q": 4104}, "aligned"), ({"v_row_stride": 132}, "multiple of 8"), ({"k_row_stride": 64}, "overlap"),
    ({"k_row_stride": 1 << 23}, "2\\^23"), ({"total_q": 1 << 30}, "2\\^30"), ({"max_seqlen_q": -1}, "max_seqlen"),
    ({"cu_seqlens_k": 0}, "cu_seqlens"), ({"softmax_lse": 0}, "softmax_lse"), ({"reserved": 1}, "reserved"),
])
def test_c_abi_refusals(change, text):
    L, Args = _abi()
    assert L.fa_window_args_size(0) == ctypes.sizeof(Args)
    for fn in (L.fa_window_fwd, L.fa_window_bwd):
        a = _valid(Args)
        for n, x in change.items():
            setattr(a, n, x)
        assert fn(ctypes.byref(a), None) != 0
        import re
        assert re.search(text, L.fa_last_error().decode()), L.fa_last_error()


@pytest.mark.parametrize("change, text", [({"dout": 0}, "dout is NULL"), ({"dq": 0}, "dq is NULL"), ({"dv_row_stride": 64}, "overlap"),
                                          ({"workspace": 0}, "workspace"), ({"workspace_bytes": 8}, "workspace")])
def test_c_abi_refusals_of_the_backward(change, text):
    L, Args = _abi()
    a = _valid(Args)
    a.workspace_bytes = L.fa_window_bwd_workspace(ctypes.byref(a))
    assert a.workspace_bytes > 0
    for n, x in change.items():
        setattr(a, n, x)
    assert L.fa_window_bwd(ctypes.byref(a), None) != 0
    assert text in L.fa_last_error().decode()


def test_c_abi_null_and_empty():
    L, Args = _abi()
    assert L.fa_window_fwd(None, None) != 0 and L.fa_window_bwd(None, None) != 0
    assert L.fa_window_bwd_workspace(None) < 0
    a = _valid(Args)
    a.total_q = a.max_seqlen_q = 0
    a.q = a.o = a.softmax_lse = 0
    assert L.fa_window_fwd(ctypes.byref(a), None) == 0      # no rows: nothing is launched


# ---------------------------------------------------------------------------------------- GPU
CASES = [
    # dtype, head_dim, heads, kv heads, query lengths, key lengths, window, sinks
    ("bf16", 64, 2, 2, [70], [70], None, 0),
    ("bf16", 64, 2, 2, [1], [1], 1, 0),
    ("bf16", 64, 4, 2, [130, 1, 0, 33], [130, 1, 5, 33], 7, 0),
    ("fp16", 64, 3, 1, [200, 65], [200, 65], 64, 3),
    ("bf16", 128, 4, 1, [257, 31], [300, 31], 50, 1),
    ("fp16", 128, 2, 2, [96], [96], 32, 40),
    ("bf16", 32, 6, 2, [129, 128, 127], [129, 128, 127], 33, 2),
    ("bf16", 8, 2, 1, [40], [77], 9, 4),
    ("fp16", 24, 2, 2, [64, 5], [64, 200], 17, 0),
    ("bf16", 80, 5, 1, [90], [90], 31, 31),
    ("fp16", 96, 2, 1, [150], [151], 150, 7),
    ("bf16", 64, 2, 1, [60, 20], [40, 0], 16, 2),           # more rows than keys; no keys at all
    ("bf16", 128, 2, 1, [40], [10], None, 5),
    ("bf16", 64, 7, 1, [45, 300], [45, 310], 20, 100),      # more sinks than keys; a group of 7
    ("fp16", 128, 16, 1, [70], [200], 3, 1),
    ("bf16", 64, 1, 1, [700], [700], 40, 5),                # sinks seen from far behind (their own workgroups)
    ("fp16", 128, 6, 2, [601, 40], [650, 300], 33, 33),
    ("bf16", 32, 3, 1, [500], [500], 1, 1),
    ("bf16", 64, 64, 1, [9], [40], 12, 2),                  # a group wider than a tile
    ("bf16", 64, 2, 2, [3] * 40, [5] * 40, 2, 1),
]
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _run(case, seed=0, scale=None, tail=0, grad=True, prepare=None):
    from window_testutil import cu, randn
    dt, d, hq, hk, ql, kl, w, s = case
    dt = TYPES[dt]
    q, dout = (randn(seed + i, (sum(ql) + tail, hq, d), dt) for i in (0, 3))
    k, v = (randn(seed + i, (sum(kl) + tail, hk, d), dt) for i in (1, 2))
    if prepare:
        prepare(q, k, v, dout)
    for x in (q, k, v):
        x.requires_grad_(grad)
    out, lse = _func()(q, k, v, cu(ql), cu(kl), max(ql), max(kl), w, s, softmax_scale=scale, return_lse=True)
    res = {"out": out.detach(), "lse": lse}
    if grad:
        res["dq"], res["dk"], res["dv"] = torch.autograd.grad(out, (q, k, v), dout)
    return q.detach(), k.detach(), v.detach(), dout, res


def _compare(case, q, k, v, dout, res, scale=None):
    from window_testutil import check, dense_reference
    dt, d, hq, hk, ql, kl, w, s = case
    scale = d ** -0.5 if scale is None else scale
    r, lses, e = dense_reference(q, k, v, ql, kl, w, s, scale, TYPES[dt], dout if "dq" in res else None)
    for n in ("out", "dq", "dk", "dv"):
        if n in res:
            check(n, res[n], r[n], e[n])
    for b, (n, lse) in enumerate(zip(ql, lses)):
        got = res["lse"][b, :, :n].double()
        dead = torch.isinf(lse)
        assert torch.equal(torch.isinf(got), dead)
        # scores' error (bounds()), log of the sum, its rounding
        tol = 2.0 ** -20 * (1 + lse.abs()) + 2.0 ** -24 * (d + 8) * 40
        assert ((got - lse).abs()[~dead] <= tol[~dead]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[0]}-d{c[1]}-h{c[2]}x{c[3]}-q{max(c[4])}-w{c[6]}-s{c[7]}")
def test_values_and_gradients(case):
    _compare(case, *_run(case))


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [-0.2, 0.0, 1.0, 1e-30])
@pytest.mark.parametrize("d", [64, 128])
def test_scales(scale, d):
    case = ("bf16", d, 2, 1, [100], [120], 30, 4)
    _compare(case, *_run(case, scale=scale), scale=scale)


@pytest.mark.gpu
def test_rows_behind_the_last_sequence_are_zero():
    case = ("bf16", 64, 4, 2, [50, 20], [60, 20], 16, 2)
    q, k, v, dout, res = _run(case, tail=300)
    assert not res["out"][70:].any() and not res["dq"][70:].any() and not res["dk"][80:].any() and not res["dv"][80:].any()
    _compare(case, q, k, v, dout, res)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_infinities_where_no_row_sees_them(bad, d):
    """Keys in front of every window, and a token whose own rows alone are spoilt."""
    case = ("bf16", d, 4, 2, [70], [150], 20, 0)

    def prepare(q, k, v, dout):
        k[:61], v[:61] = bad, bad            # the first row (position 80) sees keys 61 .. 80
    q, k, v, dout, res = _run(case, prepare=prepare)
    assert all(torch.isfinite(res[n]).all() for n in ("out", "dq", "dk", "dv"))
    _compare(case, q, k, v, dout, res)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
def test_an_infinity_reaches_the_rows_that_see_it_and_no_other(d):
    case = ("bf16", d, 2, 1, [200], [200], 16, 0)

    def prepare(q, k, v, dout):
        v[100] = math.inf
    q, k, v, dout, res = _run(case, prepare=prepare)
    sees = torch.zeros(200, dtype=torch.bool)
    sees[100:116] = True
    assert (torch.isfinite(res["out"]).all(-1).all(-1).cpu() == ~sees).all()
    assert torch.isfinite(res["dq"][~sees.cuda()]).all()
    clean = torch.ones(200, dtype=torch.bool)
    clean[85:116] = False                    # keys that share a row with key 100
    assert torch.isfinite(res["dk"][clean.cuda()]).all()
    assert torch.isfinite(res["dv"]).all()
    r, _, e = __import__("window_testutil").dense_reference(q, k, v.nan_to_num(posinf=0.0), [200], [200], 16, 0, d ** -0.5, torch.bfloat16, dout)
    ok = ~sees.cuda()
    assert ((res["out"][ok].double() - r["out"][ok]).abs() <= e["out"][ok]).all()
    assert ((res["dv"][clean.cuda()].double() - r["dv"][clean.cuda()]).abs() <= e["dv"][clean.cuda()]).all()


@pytest.mark.gpu
def test_packed_and_strided_inputs():
    """q, k, v as views of one packed tensor, of a transposed one, with broadcast gradients."""
    from window_testutil import cu, randn
    f = _func()
    qkv = randn(0, (90, 3, 4, 64), torch.bfloat16).requires_grad_()
    c = cu([90])
    want = None
    for make in (lambda x: x, lambda x: x.clone(), lambda x: x.transpose(0, 1).contiguous().transpose(0, 1)):
        q, k, v = (make(qkv[:, i]) for i in range(3))
        out = f(q, k, v, c, c, 90, 90, 20, 2)
        w = randn(9, (4, 64), torch.bfloat16)
        g, = torch.autograd.grad((out.sum(0) * w).sum(), (qkv,))
        if want is None:
            want = (out.detach(), g)
        assert torch.equal(out, want[0]) and torch.equal(g, want[1])
    odd = torch.empty(90 * 4 * 64 + 4, dtype=torch.bfloat16, device="cuda")[4:].view(90, 4, 64)
    odd.copy_(qkv[:, 0])
    assert torch.equal(f(odd, qkv[:, 1], qkv[:, 2], c, c, 90, 90, 20, 2), want[0])


@pytest.mark.gpu
def test_equal_to_the_dense_forward_without_a_window():
    """Within the two kernels' roundings, the causal dense attention of the framework."""
    from flash_attn.flash_attn_interface import flash_attn_unpadded_func
    case = ("bf16", 64, 2, 2, [300, 77], [300, 77], None, 0)
    q, k, v, dout, res = _run(case, grad=False)
    from window_testutil import cu, dense_reference
    c = cu([300, 77])
    dense = flash_attn_unpadded_func(q, k, v, c, c, 300, 300, 0.0, causal=True)
    _, _, e = dense_reference(q, k, v, [300, 77], [300, 77], None, 0, 64 ** -0.5, torch.bfloat16)
    assert ((dense.double() - res["out"].double()).abs() <= 2 * e["out"]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
def test_repeats_bit_for_bit_on_any_stream(d):
    case = ("bf16", d, 8, 2, [700, 130], [720, 130], 60, 9)
    a = _run(case)[4]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b = _run(case)[4]
    torch.cuda.current_stream().wait_stream(s)
    for n in ("out", "dq", "dk", "dv"):
        assert torch.equal(a[n], b[n]), n


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
def test_graph_replays(d):
    """Forward and backward captured; replays with new inputs, eager work of the same kind between them."""
    from window_testutil import cu, randn
    f, c = _func(), cu([200, 90])
    q, k, v, dout = (randn(i, (290, 4 if i in (0, 3) else 2, d), torch.bfloat16) for i in range(4))

    def step(q, k, v, dout):
        a, b, e = (x.detach().requires_grad_() for x in (q, k, v))
        out = f(a, b, e, c, c, 200, 200, 24, 3)
        return (out.detach(),) + torch.autograd.grad(out, (a, b, e), dout)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(q, k, v, dout)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(q, k, v, dout)
    for i in range(3):
        for x, n in ((q, 10), (k, 20), (v, 30), (dout, 40)):
            x.copy_(randn(n + i, x.shape, x.dtype))
        graph.replay()
        torch.cuda.synchronize()
        want = step(q, k, v, dout)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want)), i


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """Rows so far apart that their bytes pass 2^32."""
    from window_testutil import check, cu, dense_reference, randn
    n, d, stride = 600, 64, 1 << 22
    q, k, v, dout = (randn(i, (n, 1, d), torch.bfloat16) for i in range(4))
    big = torch.empty(n * stride + 1024, dtype=torch.bfloat16, device="cuda")      # 5 GB
    kk, vv = (torch.as_strided(big, (n, 1, d), (stride, d, 1), off) for off in (0, 512))
    kk.copy_(k)
    vv.copy_(v)
    c = cu([n])
    q, kk, vv = (x.requires_grad_() for x in (q, kk.detach(), vv.detach()))
    out = _func()(q, kk, vv, c, c, n, n, 70, 3)
    dq, dk, dv = torch.autograd.grad(out, (q, kk, vv), dout)
    r, _, e = dense_reference(q.detach(), k, v, [n], [n], 70, 3, d ** -0.5, torch.bfloat16, dout)
    for name, x in (("out", out.detach()), ("dq", dq), ("dk", dk), ("dv", dv)):
        check(name, x, r[name], e[name])


@pytest.mark.gpu
def test_gradients_against_differences():
    """Directional derivatives of the plain form by differences, against the kernels' gradients: the difference is at
    most the sum of the gradient's bounds along the direction."""
    from window_testutil import dense_reference
    case = ("bf16", 64, 4, 2, [50, 30], [60, 30], 12, 3)
    q, k, v, dout, res = _run(case)
    _, _, e = dense_reference(q, k, v, case[4], case[5], 12, 3, 64 ** -0.5, torch.bfloat16, dout)
    g = torch.Generator(device="cuda").manual_seed(1)
    loss = lambda a, b, c: (dense_reference(a, b, c, case[4], case[5], 12, 3, 64 ** -0.5, torch.bfloat16)[0]["out"] * dout.double()).sum().item()
    q, k, v = q.double(), k.double(), v.double()
    for i, n in enumerate(("dq", "dk", "dv")):
        x = [q, k, v]
        way = torch.randn(x[i].shape, generator=g, device="cuda", dtype=torch.float64)
        up, down = list(x), list(x)
        up[i], down[i] = x[i] + 1e-5 * way, x[i] - 1e-5 * way
        diff = (loss(*up) - loss(*down)) / 2e-5
        got = (res[n].double() * way).sum().item()
        assert abs(got - diff) <= (e[n] * way.abs()).sum().item() + 1e-6 * abs(diff)


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    from window_testutil import cu, randn
    f = _func()
    q, k = randn(0, (8, 4, 64), torch.bfloat16), randn(1, (8, 2, 64), torch.bfloat16)
    c = cu([8])
    with pytest.raises(RuntimeError, match="dtype"):
        f(q, k.half(), k, c, c, 8, 8, 4)
    with pytest.raises(RuntimeError, match="multiple of the heads"):
        f(q, k[:, :1].expand(8, 3, 64), k[:, :1].expand(8, 3, 64), c, c, 8, 8, 4)
    with pytest.raises(RuntimeError, match="int32"):
        f(q, k, k, c.long(), c, 8, 8, 4)
    with pytest.raises(RuntimeError, match="on the device"):
        f(q, k, k, c.cpu(), c, 8, 8, 4)
    with pytest.raises(RuntimeError, match="fp16 and bf16"):
        f(q.float(), k.float(), k.float(), c, c, 8, 8, 4)
    with pytest.raises(RuntimeError, match="multiple of 8"):
        f(q[..., :20], k[..., :20], k[..., :20], c, c, 8, 8, 4)
    a, b = q.clone().requires_grad_(), k.clone().requires_grad_()
    out = f(a, b, b, c, c, 8, 8, 4)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(out.sum(), a, create_graph=True)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_small_calls_round_once(dtype, d):
    """A small call with a short window takes P and dS in two parts: its errors (rms) are those of one rounding, half a
    step at most and uniform over it, against the 1.4 of a second rounding; the same rows in a batch too large for it
    keep the bounds that count both."""
    from window_testutil import check, cu, dense_reference, randn
    n, many = 200, 200
    q, k, v, dout = (randn(i, (n, 2, d), dtype) for i in range(4))
    r, _, e = dense_reference(q, k, v, [n], [n], 30, 2, d ** -0.5, dtype, dout)
    for copies in (1, many):
        x = [t.repeat(copies, 1, 1).requires_grad_() for t in (q, k, v)]
        c = cu([n] * copies)
        out = _func()(*x, c, c, n, n, 30, 2)
        grads = torch.autograd.grad(out, x, dout.repeat(copies, 1, 1))
        for name, got in zip(("out", "dq", "dk", "dv"), (out.detach(), *grads)):
            got = got[-n:]
            check(name, got, r[name], e[name])
            if copies == 1:
                rounded = r[name].to(dtype).double()
                rms = lambda a: (a - r[name]).pow(2).mean().sqrt()
                assert rms(got.double()) <= 1.1 * rms(rounded)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("most", [0, 1, 10, 40])
def test_rows_past_max_seqlen_are_left_alone(d, most):
    """Sequences longer than max_seqlen_q says (C ABI): what is asked for is right, nothing else is written, the rows
    that are not computed add nothing to dk and dv."""
    from window_testutil import DEV, cu, randn
    L, Args = _abi()
    H, n, m = 4, [150, 7], [170, 30]
    q, k, v, dout = (randn(i, (sum(n if i in (0, 3) else m), h, d), torch.bfloat16) for i, h in enumerate((H, 2, 2, H)))
    full = _func()(q, k, v, cu(n), cu(m), 150, 170, 20, 3, return_lse=True)
    o, lse = torch.full_like(q, 7), torch.full((2 * H * most + 512,), 7.0, device=DEV)
    a = _valid(Args)
    g = {x: torch.full_like(y, 7) for x, y in (("dq", q), ("dk", k), ("dv", v))}
    c = cu(n), cu(m)
    for name, t in dict(q=q, k=k, v=v, o=o, dout=dout, softmax_lse=lse, cu_seqlens_q=c[0], cu_seqlens_k=c[1], **g).items():
        setattr(a, name, t.data_ptr())
    for name, h in dict(q=H, k=2, v=2, o=H, do=H, dq=H, dk=2, dv=2).items():
        setattr(a, name + "_row_stride", h * d)
        setattr(a, name + "_head_stride", d)
    a.total_q, a.total_k, a.batch, a.nheads, a.nheads_k, a.head_dim = sum(n), sum(m), 2, H, 2, d
    a.max_seqlen_q, a.max_seqlen_k, a.lse_stride, a.window, a.num_sinks = most, 170, most, 20, 3
    a.softmax_scale = d ** -0.5
    a.workspace_bytes = L.fa_window_bwd_workspace(ctypes.byref(a))
    ws = torch.empty(a.workspace_bytes, dtype=torch.uint8, device=DEV)
    a.workspace = ws.data_ptr()
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert L.fa_window_fwd(ctypes.byref(a), stream) == 0 and L.fa_window_bwd(ctypes.byref(a), stream) == 0
    torch.cuda.synchronize()
    kept = torch.zeros(sum(n), dtype=torch.bool, device=DEV)
    for at, x in ((0, n[0]), (n[0], n[1])):
        kept[at:at + min(x, most)] = True
    assert (lse[2 * H * most:] == 7).all() and (o[~kept] == 7).all() and (g["dq"][~kept] == 7).all()
    assert torch.equal(o[kept], full[0][kept])
    for b in range(2):
        rows = min(n[b], most)
        assert torch.equal(lse[:2 * H * most].view(2, H, most)[b, :, :rows], full[1][b, :, :rows])
    # the same gradients with the other rows' dout at 0
    x = [t.clone().requires_grad_() for t in (q, k, v)]
    want = torch.autograd.grad(_func()(*x, *c, 150, 170, 20, 3), x, dout * kept[:, None, None])
    for name, w in zip(("dk", "dv"), want[1:]):
        # sums of one set of terms in two orders, each rounded once: a step of bf16 apart at most
        assert (g[name].double() - w.double()).abs().max() <= 2 ** -7 * w.double().abs().max()
    assert torch.equal(g["dq"][kept], want[0][kept])


@pytest.mark.gpu
@pytest.mark.parametrize("n", [0, 1])
def test_nothing_to_do(n):
    from window_testutil import cu
    f = _func()
    q = torch.zeros(n, 2, 64, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    k = torch.ones(3, 1, 64, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    c = cu([0])
    out = f(q, k, k, c, cu([3]), 0, 3, 4)
    assert out.shape == q.shape and not out.any()
    dq, dk = torch.autograd.grad(out, (q, k), torch.ones_like(out))
    assert not dq.any() and not dk.any()


@pytest.mark.gpu
def test_packed_forms():
    """kvpacked and qkvpacked: the separate form's outputs and gradients, bit for bit."""
    from flash_attn import flash_window_attn_interface as fw
    from window_testutil import cu, randn
    c = cu([90, 1, 40])
    qkv = randn(0, (150, 3, 4, 64), torch.bfloat16).requires_grad_()
    dout = randn(1, (150, 4, 64), torch.bfloat16)
    q, k, v = (qkv.detach()[:, i].clone().requires_grad_() for i in range(3))
    want = fw.flash_window_attn_unpadded_func(q, k, v, c, c, 90, 90, 20, 2)
    grads = torch.stack(torch.autograd.grad(want, (q, k, v), dout), 1)
    out, lse = fw.flash_window_attn_unpadded_qkvpacked_func(qkv, c, 90, 20, 2, return_lse=True)
    assert lse.shape == (3, 4, 96) and not lse.requires_grad
    assert torch.equal(out, want) and torch.equal(torch.autograd.grad(out, qkv, dout)[0], grads)
    kv = qkv.detach()[:, 1:].clone().requires_grad_()
    out = fw.flash_window_attn_unpadded_kvpacked_func(q, kv, c, c, 90, 90, 20, 2)
    dq, dkv = torch.autograd.grad(out, (q, kv), dout)
    assert torch.equal(out, want) and torch.equal(dq, grads[:, 0]) and torch.equal(dkv, grads[:, 1:])
    with pytest.raises(RuntimeError, match="qkv must be"):
        fw.flash_window_attn_unpadded_qkvpacked_func(kv, c, 90, 20)


def test_modules_refuse_a_window_without_its_mask():
    from flash_attn.flash_attention import FlashAttention, FlashMHA
    with pytest.raises(RuntimeError, match="dropout"):
        FlashAttention(attention_dropout=0.1, window_size=8)
    with pytest.raises(RuntimeError, match="causal"):
        FlashMHA(64, 2, window_size=8)


@pytest.mark.gpu
@pytest.mark.parametrize("rotary", [None, "1d"])
def test_modules(rotary):
    """FlashMHA with a window, padded and not, against its own unwindowed layers around the plain form; gradients run."""
    from flash_attn.flash_attention import FlashAttention, FlashMHA
    from oracle import window_ref as ref
    torch.manual_seed(0)
    m = FlashMHA(128, 2, causal=True, use_rotary_emb=rotary, window_size=9, num_sinks=2, device="cuda", dtype=torch.bfloat16)
    x = torch.randn(2, 50, 128, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    mask = torch.ones(2, 50, dtype=torch.bool, device="cuda")
    mask[1, 30:] = False
    full, _ = m(x)
    padded, _ = m(x, key_padding_mask=mask)
    assert torch.equal(full[0], padded[0]) and torch.equal(full[1, :30], padded[1, :30])
    full.float().square().sum().backward()
    assert torch.isfinite(x.grad).all() and x.grad.abs().sum() > 0
    inner = FlashAttention(window_size=9, num_sinks=2)
    qkv = torch.randn(1, 50, 3, 2, 64, device="cuda", dtype=torch.bfloat16)
    out, _ = inner(qkv, causal=True)
    live = ref.seen(torch.arange(50, device="cuda"), torch.arange(50, device="cuda"), 9, 2)
    for h in range(2):
        a = (*(qkv[0, :, i, h] for i in range(3)), live, 64 ** -0.5)
        r, _, p = ref.attention(*a)
        assert ((out[0, :, h].double() - r).abs() <= ref.bounds(*a, p, r)).all()
    with pytest.raises(RuntimeError, match="causal"):
        inner(qkv)
