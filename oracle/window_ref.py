"""Plain 64-bit windowed attention, with gradients by formula, and bounds on what a 16-bit kernel may be off.

One sequence and head at a time, every quantity by selection: an entry that a row does not see takes part in nothing,
whatever stands there (infinities and NaN among them).
"""
import math

import torch

F32 = 2.0 ** -24          # half a step of fp32


def seen(qpos, kpos, window, sinks):
    """(rows, keys) truth values: position p sees key position j when j <= p and (j > p - window or j < sinks)."""
    q, k = qpos[:, None], kpos[None, :]
    m = k <= q
    return m & ((k > q - window) | (k < sinks)) if window else m


def attention(q, k, v, live, scale):
    """q (rows, d), k, v (keys, d), live (rows, keys) -> out, lse, P in 64 bits; rows without a key: 0, -inf, 0."""
    q, k, v = q.double(), k.double(), v.double()
    s = torch.where(live, _products(q, k, live) * scale, -math.inf)
    top = s.amax(-1, keepdim=True) if s.shape[1] else torch.full((len(q), 1), -math.inf, dtype=torch.float64, device=q.device)
    e = torch.where(live, torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top)), 0.0)
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total == 0, torch.ones_like(total), total)
    lse = torch.where(total[:, 0] == 0, -math.inf, top[:, 0] + torch.log(torch.where(total[:, 0] == 0, 1.0, total[:, 0])))
    return _weighted(p, v, live), lse, p


def _clean(x):
    return torch.where(torch.isfinite(x), x, torch.zeros_like(x))


def _products(a, b, live):
    """a b^T where live; entries that are not, 0."""
    return torch.where(live, _clean(a) @ _clean(b).mT, 0.0)


def _weighted(w, x, live):
    """sum over the live columns of w x (x's rows that no row sees may hold anything)."""
    return torch.where(live, w, 0.0) @ _clean(x)


def gradients(q, k, v, live, scale, p, out, dout):
    q, k, v, dout = q.double(), k.double(), v.double(), dout.double()
    dp = _products(dout, v, live)
    delta = (p * dp).sum(-1, keepdim=True)
    ds = torch.where(live, p * (dp - delta), 0.0)
    return scale * _weighted(ds, k, live), scale * _weighted(ds.mT, q, live.mT), _weighted(p.mT, dout, live.mT), ds


def bounds(q, k, v, live, scale, p, out, dout=None, ds=None, exact_delta=False, dtype=torch.bfloat16):
    """Largest error of each output element, from the kernels' roundings: u = half a step of the 16-bit type, once for
    each P (for P V and P^T dO), once for each dS, once for each output; 2^-24 for each fp32 product and sum.

    Scores: |err s| <= (d + 4) 2^-24 |q||k| scale (the sum's d roundings, the scale's and the maximum's); exp adds
    2^-22; so P is off by a factor of 1 +- c with c = 2 (max err s + 2^-22), the 2 for numerator and denominator, and
    sums over n keys add n 2^-24."""
    u = torch.finfo(dtype).eps / 2
    q, k, v = _clean(q.double()).abs(), _clean(k.double()).abs(), _clean(v.double()).abs()
    n, d = live.shape[1], q.shape[1]
    s = torch.where(live, q @ k.mT, 0.0) * abs(scale)
    c = 2 * ((d + 4) * F32 * (s.amax(-1, keepdim=True) if n else 0.0) + 2.0 ** -22) + (n + 16) * F32
    a = p @ v
    e_out = (u + c) * a + u * (1 + u) * (out.abs() + (u + c) * a) + 2.0 ** -140
    if dout is None:
        return e_out
    do = _clean(dout.double()).abs()
    dp = torch.where(live, do @ v.mT, 0.0)
    # delta: from the 16-bit output, or from P and dP in fp32
    e_delta = (c + (n + d) * F32) * (p * dp).sum(-1, keepdim=True) * 2
    if not exact_delta:
        e_delta = e_delta + (do * e_out).sum(-1, keepdim=True)
    e_ds = (u + c) * ds.abs() + (1 + u) * p * (e_delta + (d + 4) * F32 * dp + c * (dp + (p * dp).sum(-1, keepdim=True)))
    m = live.shape[0]
    e_dq = abs(scale) * (e_ds @ k + (n + 8) * F32 * (ds.abs() @ k))
    e_dk = abs(scale) * (e_ds.mT @ q + (m + 8) * F32 * (ds.abs().mT @ q))
    e_dv = ((u + c) * p).mT @ do + (m + 8) * F32 * (p.mT @ do)
    return e_out, e_dq, e_dk, e_dv
