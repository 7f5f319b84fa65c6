"""Plain 64-bit forms of the paged-cache operators, and the error their kernels may make.

U[t] is half a step of type t relative to the value: one rounding to t is off by at most
that. Errors of the 32-bit arithmetic between roundings are counted in units of 2^-24."""
import math

import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
F = 2.0 ** -24


def rotate(x, w, positions, base, eps):
    """Per-head norm (w None: none) and rotation of x [T, heads, hd] in 64 bits; and the
    magnitude each output's 32-bit errors are relative to."""
    x = x.double()
    hd = x.shape[-1]
    y = x
    if w is not None:
        y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w.double()
    i = torch.arange(hd // 2, dtype=torch.float64, device=x.device)
    ang = positions.double()[:, None] * torch.pow(torch.tensor(base, dtype=torch.float64, device=x.device),
                                                  -2.0 * i / hd)
    c, s = torch.cos(ang)[:, None], torch.sin(ang)[:, None]
    a, b = y[..., :hd // 2], y[..., hd // 2:]
    mag = (a.abs() + b.abs()).repeat(1, 1, 2)
    return torch.cat([a * c - b * s, a * s + b * c], -1), mag


def rotate_bound(ref, mag, t):
    """One rounding to t; before it, in 32 bits: the mean of squares (at most hd + 8 units,
    halved by the root), root, two products (8), the sine and cosine (8, and 13 for an angle
    rounded to 2^-25 of a turn), the two products and the sum (3)."""
    return U[t] * ref.abs() + (68 + 32) * F * mag + (2.0 ** -24 if t == torch.float16 else 0.0)


def quantized(x, gs, bits):
    """Codes (packed from the low bits up), scales and biases of rows x [..., hd] of a 16-bit
    type by the cache's rule, in 32-bit arithmetic on the CPU: a step = range * (1 / steps),
    the end of larger magnitude kept exactly."""
    t = x.dtype
    v = x.cpu().float().unflatten(-1, (-1, gs))
    hi, lo = v.amax(-1), v.amin(-1)
    steps = torch.tensor(float(2 ** bits - 1))
    neg = lo.abs() > hi.abs()
    s = ((hi - lo) * (1.0 / steps)).clamp_min(1e-7)
    s = torch.where(neg, s, -s)
    edge = torch.where(neg, lo, hi)
    q0 = torch.round(edge / s)
    s = torch.where(q0 != 0, edge / torch.where(q0 != 0, q0, 1.0), s)
    b = torch.where(q0 != 0, edge, 0.0)
    q = torch.round((v - b[..., None]) / s[..., None]).clamp(0, float(steps)).long().flatten(-2)
    per = 32 // bits
    words = (q.unflatten(-1, (-1, per)) << (torch.arange(per) * bits)).sum(-1)
    words = torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)
    return words, s.to(t), b.to(t)


def values(codes, scales, biases, gs, bits):
    """s * q + b of packed rows [..., words] in 64 bits."""
    per = 32 // bits
    w = codes.view(torch.int32).long() & 0xffffffff
    q = (w.unsqueeze(-1) >> (torch.arange(per, device=w.device) * bits)) & (2 ** bits - 1)
    q = q.flatten(-2).unflatten(-1, (-1, gs)).double()
    return (q * scales.double().unsqueeze(-1) + biases.double().unsqueeze(-1)).flatten(-2)


def half_step(x, t):
    """Half the distance between t's values next to x (64-bit)."""
    low = -14 if t == torch.float16 else -126
    x = x.abs().clamp_min(2.0 ** low)
    m, _ = torch.frexp(x)                        # x / m is a power of two, exactly
    return x / m / 2 * torch.finfo(t).eps / 2


def attention(q, cu, k, v, table, lens, scale, masks, t, bad=None):
    """Rows attention in 64 bits. q [total, Hq, hd]; k, v the pools' values [rows, Hkv, hd];
    table, lens, cu, masks host lists. Returns (out, bound) on q's device: the error from
    p rounded to t (U), from scores of 32-bit sums (delta: p off by a factor exp(2 delta)
    after normalising), from sums over the keys, and from the last rounding."""
    total, Hq, hd = q.shape
    Hkv = k.shape[1]
    G = Hq // Hkv
    page = table["page"]
    out = torch.zeros(total, Hq, hd, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    for b, L in enumerate(lens):
        lo, hi = cu[b], cu[b + 1]
        n = hi - lo
        if n == 0 or L == 0:
            continue
        pids = table["rows"][b]
        at, ok = [], []
        for j in range(L):
            pid = pids[j // page]
            good = 0 <= pid < table["pages"]
            ok.append(good)
            at.append(pid * page + j % page if good else 0)
        at = torch.tensor(at, device=q.device)
        ok = torch.tensor(ok, device=q.device)
        kb, vb = k[at], v[at]
        kb = torch.where(ok[:, None, None], kb, 0.0)
        vb = torch.where(ok[:, None, None], vb, 0.0)
        j = torch.arange(L, device=q.device) - (L - n)
        if masks is None:
            see = j[None] <= torch.arange(n, device=q.device)[:, None]
        else:
            m = torch.tensor(masks[lo:hi], device=q.device)
            see = (j[None] < 0) | (((m[:, None] >> j.clamp(0, 63)[None]) & 1) == 1)
        see = see & ok[None]
        for h in range(Hq):
            kh, vh, qh = kb[:, h // G], vb[:, h // G], q[lo:hi, h].double()
            s = (qh @ kh.T) * scale
            delta = 2 * (hd + 8) * F * ((qh.abs() @ kh.abs().T) * abs(scale)).amax(-1)
            s = s.masked_fill(~see, -math.inf)
            p = torch.exp(s - s.amax(-1, keepdim=True).clamp_min(-1e300))
            den = p.sum(-1, keepdim=True)
            p = torch.where(den > 0, p / den.clamp_min(1e-300), 0.0)
            o = p @ vh
            out[lo:hi, h] = o
            each = U[t] + 2 * delta + (L + 64) * F
            tol[lo:hi, h] = U[t] * o.abs() + each[:, None] * (p @ vh.abs()) * 1.01
            if t == torch.float16:   # probabilities below 2^-14 of the largest: half a subnormal step
                tol[lo:hi, h] += 2.0 ** -25 * vh.abs().sum(0)[None] + 2.0 ** -25
    return out, tol
