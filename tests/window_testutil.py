"""Shared helpers of the windowed, paged and cache tests (test infrastructure)."""
import torch

from oracle import window_ref as ref

DEV = "cuda"


def cu(lens):
    return torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32, device=DEV)


def randn(seed, shape, dtype):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(dtype).to(DEV)


def dense_reference(q, k, v, ql, kl, window, sinks, scale, dtype, dout=None):
    """64-bit out, lse by sequence (list of (heads, rows)), gradients, and their bounds, for packed sequences. Rows
    behind the last sequence: 0. `exact_delta` is left to the looser bound: it covers both."""
    H, G = q.shape[1], q.shape[1] // k.shape[1]
    f = lambda x: torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    r = {"out": f(q), "dq": f(q), "dk": f(k), "dv": f(v)}
    e = {n: torch.zeros_like(x) for n, x in r.items()}
    lses = []
    q0 = k0 = 0
    u = torch.finfo(dtype).eps / 2
    for n, m in zip(ql, kl):
        live = ref.seen(torch.arange(n, device=DEV) + m - n, torch.arange(m, device=DEV), window, sinks)
        qs, ks = slice(q0, q0 + n), slice(k0, k0 + m)
        lse = torch.zeros((H, n), dtype=torch.float64, device=DEV)
        for h in range(H):
            a = (q[qs, h], k[ks, h // G], v[ks, h // G], live, scale)
            out, lse[h], p = ref.attention(*a)
            r["out"][qs, h] = out
            if dout is None:
                e["out"][qs, h] = ref.bounds(*a, p, out, dtype=dtype)
                continue
            dq, dk, dv, ds = ref.gradients(*a, p, out, dout[qs, h])
            r["dq"][qs, h] = dq
            r["dk"][ks, h // G] += dk
            r["dv"][ks, h // G] += dv
            b = ref.bounds(*a, p, out, dout[qs, h], ds, dtype=dtype)
            e["out"][qs, h] = b[0]
            e["dq"][qs, h] = b[1]
            e["dk"][ks, h // G] += b[2]
            e["dv"][ks, h // G] += b[3]
        lses.append(lse)
        q0, k0 = q0 + n, k0 + m
    for n in ("dq", "dk", "dv"):         # the outputs' own rounding, and 16-bit subnormals' step
        e[n] += u * (1 + u) * (r[n].abs() + e[n]) + torch.finfo(dtype).tiny * u
    e["out"] += torch.finfo(dtype).tiny * u
    return r, lses, e


def check(name, got, want, bound):
    got = got.double()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    bad = ~((got - want).abs() <= bound)
    if bad.any():
        i = tuple(bad.nonzero()[0].tolist())
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} off, first at {i}: {got[i].item()} for "
                             f"{want[i].item()} (bound {bound[i].item():.3g})")
