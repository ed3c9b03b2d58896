"""64-bit definitions and error bounds of the attention-side operators, for tests.

Bounds, per element, from the kernels' arithmetic (u: half a step of the
16-bit type, eps / 2 of torch.finfo; every fp32 step errs by 2^-24):

* attention: scores are fp32 dot products of exact 16-bit inputs, off by at
  most (D + 8) 2^-24 A with A = scale sum |q_d k_d| (products are exact in
  fp32, D - 1 additions, the scaling by log2 e and its product), which is a relative error of the
  probability; ex2.approx adds 2^-22, a maximum that changes between
  steps 2^-23 a rescaling, of which there are at most one per 16 positions and
  warp, and sums over n positions n 2^-24; each probability is rounded to 16 bits (u, and for
  fp16 half a step of its subnormals, 2^-25) before the product with V; the
  output is rounded once (u, or 2^-25 below fp16's normal range), the gate's
  sigmoid in fp32 errs by 2^-20 (__expf's argument up to 32 in magnitude).
* rotary: cos and sin err by 2^-21, the norm by (D / 2 + 8) 2^-24 relative, then
  three fp32 operations; the output is rounded once.
"""
import math

import torch


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def gather(cache, table_row, n, P):
    """[n, heads, D] double: the first n positions of a request."""
    if n == 0:
        return cache.new_zeros((0, cache.shape[1], cache.shape[3])).double()
    pages = table_row[:-(-n // P)].long()
    return cache[pages].transpose(1, 2).reshape(-1, cache.shape[1], cache.shape[3])[:n].double()


def attention(q, kc, vc, table, lens, rows, scale=None, window=0, gate=None, keep=None):
    """(out, lse, out's bound, lse's bound) in fp64.  lens, rows: host lists;
    keep(b) (optional): a bool tensor over the positions that count."""
    T, Hq, D = q.shape
    Hkv, P = kc.shape[1], kc.shape[2]
    G = Hq // Hkv
    scale = D ** -0.5 if scale is None else scale
    u = half_step(q.dtype)
    sub = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    dev = q.device
    out = torch.zeros(T, Hq, D, dtype=torch.float64, device=dev)
    tol = torch.zeros_like(out)
    lse = torch.full((T, Hq), -math.inf, dtype=torch.float64, device=dev)
    ltol = torch.zeros_like(lse)
    t = 0
    for b, (n, r) in enumerate(zip(lens, rows)):
        if n and r:
            k, v = gather(kc, table[b], n, P), gather(vc, table[b], n, P)
            p = torch.arange(n - r, n, device=dev)[:, None]
            j = torch.arange(n, device=dev)[None]
            seen = j <= p
            if window:
                seen = seen & (j > p - window)
            if keep is not None:
                seen = seen & keep(b)[None]
                k, v = torch.where(keep(b)[:, None, None], k, 0.0), torch.where(keep(b)[:, None, None], v, 0.0)
            some = seen.any(1)
            for h in range(Hq):
                qh = q[t:t + r, h].double()
                kh, vh = k[:, h // G], v[:, h // G]
                s = torch.where(seen, qh @ kh.T * scale, -math.inf)
                A = torch.where(seen, qh.abs() @ kh.abs().T * scale, 0.0).amax(1)
                z = torch.logsumexp(s, 1)
                w = torch.where(some[:, None], torch.exp(s - z[:, None]), 0.0)
                o = w @ vh
                mag = w @ vh.abs()
                rel = 2 * (D + 8) * 2.0 ** -24 * A + 2.0 ** -21 + (n + n / 16) * 2.0 ** -23
                e = (u + rel)[:, None] * mag + sub * (seen.double() @ vh.abs())
                if gate is not None:
                    sg = torch.sigmoid(gate[t:t + r, h].double())
                    o, e = o * sg, e * sg + 2.0 ** -20 * mag
                out[t:t + r, h] = o
                tol[t:t + r, h] = 1.05 * (e + u * o.abs()) + sub + 1e-30
                lse[t:t + r, h] = torch.where(some, z, -math.inf)
                ltol[t:t + r, h] = 1.05 * (rel + 2.0 ** -22 * torch.where(some, z.abs() + 1, 0.0))
        t += r
    return out, lse, tol, ltol


def axis_of(n, sections, interleaved):
    axes = len(sections)
    ax = [0] * n
    for a in range(1, axes):
        for m in range(sections[a]):
            ax[a + axes * m if interleaved else sum(sections[:a]) + m] = a
    return ax


def rope(x, positions, inv_freq, sections, interleaved, w=None, eps=1e-6):
    """(rotated, bound) in fp64; positions [axes, T]."""
    T, H, D = x.shape
    n = inv_freq.numel()
    ax = torch.tensor(axis_of(n, sections, interleaved), device=x.device)
    ang = positions.double()[ax].T * inv_freq.double()[None]
    c, s = ang.cos()[:, None], ang.sin()[:, None]
    y = x.double()
    if w is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    a, b = y[..., :n], y[..., n:2 * n]
    out = torch.cat([a * c - b * s, b * c + a * s, y[..., 2 * n:]], -1)
    mag = torch.cat([a.abs() + b.abs(), a.abs() + b.abs(), y[..., 2 * n:].abs()], -1)
    rel = 2.0 ** -20 + (D / 2 + 8) * 2.0 ** -24
    sub = 2.0 ** -25 if x.dtype == torch.float16 else 0.0
    return out, 1.05 * (half_step(x.dtype) * out.abs() + rel * mag) + sub + 1e-30


def close(got, ref, tol, what=""):
    g = got.double()
    bad = ~((g - ref).abs() <= tol) & ~(g == ref)
    if bad.any():
        i = tuple(int(v) for v in bad.nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside the bound, first at {i}: "
                             f"{float(g[i])} against {float(ref[i])} +- {float(tol[i])}")
