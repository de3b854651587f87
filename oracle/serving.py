"""Float64 definitions of the serving operators: rotary positions, the 4-bit cache,
attention over it, and eviction by weight.  Plain torch on any device, one
sequence and head at a time where that is clearest; nothing of the package is used.
"""
import math

import torch

GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
EXPONENTS = {torch.float16: (-23, 13), torch.bfloat16: (-125, 125)}


def _pow2(e):
    """2^e of whole numbers, exactly, in float64 (pow may be off by a unit)."""
    table = torch.tensor([2.0 ** k for k in range(-300, 301)], dtype=torch.float64, device=e.device)
    return table[e.long() + 300]


def rotary(x, positions, frequencies, amplitude, layout, inverse=False):
    """x [Z, H, N, D] turned; positions [N] or [Z, N]."""
    R = 2 * frequencies.numel()
    y = x.detach().double().clone()
    pos = positions if positions.dim() == 2 else positions[None]
    a = pos[:, None, :, None].double() * frequencies.to(x.device).double()
    if inverse:
        a = -a
    c, s = amplitude * torch.cos(a), amplitude * torch.sin(a)
    i = torch.arange(R // 2, device=x.device)
    lo, hi = (i, i + R // 2) if layout == "half" else (2 * i, 2 * i + 1)
    u, w = y[..., lo].clone(), y[..., hi].clone()
    y[..., lo] = u * c - w * s
    y[..., hi] = u * s + w * c
    return y


def quantise(x, dtype):
    """(codes, scale bytes) of rows x [..., D]: the packed form."""
    grid = GRID.to(x.device)
    b = x.double().reshape(x.shape[:-1] + (-1, 32))
    lo, hi = EXPONENTS[dtype]
    top = b.abs().amax(-1)
    finite = torch.isfinite(top)
    b = torch.where(finite[..., None], b, torch.zeros_like(b))
    top = torch.where(finite, top, torch.zeros_like(top))
    # the smallest e of lo .. hi with top <= 7 * 2^e (hi where there is none)
    e = torch.full(top.shape, hi, dtype=torch.int64, device=x.device)
    for k in range(hi - 1, lo - 1, -1):
        e = torch.where(top <= 7.0 * 2.0 ** k, torch.full_like(e, k), e)
    a = b.abs() * _pow2(-e)[..., None]
    d = (a[..., None] - grid).abs()
    near = d.amin(-1, keepdim=True)
    # the nearest index, of two the even one
    index = torch.arange(8, device=x.device)
    rank = torch.where(d == near, index % 2, torch.full_like(index, 2))
    m = rank.argmin(-1)
    code = (m + 8 * torch.signbit(b)).reshape(x.shape)
    scale = torch.where(finite, e + 127, torch.full_like(e, 255))
    code = torch.where(finite.repeat_interleave(32, -1), code, torch.zeros_like(code))
    return (code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8), scale.to(torch.uint8)


def values(codes, scales):
    """Float64 values of packed rows."""
    grid = torch.cat((GRID, -GRID)).to(codes.device)
    c = torch.stack((codes % 16, codes // 16), -1).reshape(codes.shape[:-1] + (-1,)).long()
    s = _pow2(scales.long() - 127)
    s = torch.where(scales == 255, torch.full_like(s, math.nan), s)
    return grid[c] * s.repeat_interleave(32, -1)


def attend(q, k, v, lengths, scale, positions=None, first=None, counts=None):
    """(o, lse, weights, total, reach): attention of q [Z, Hq, T, D] over the first
    lengths[z] rows of k, v [Z, H, C, D] (float64).  With ``positions`` [Z, H, C]
    token i sees those at most first[z] + i.  ``weights`` [Z, H, C]: summed
    softmax weights.  For error bounds: ``total``, the sum of softmax weights times
    |v|, and ``reach`` [Z, Hq, T], the largest scale * sum |q||k| of a visible key."""
    Z, Hq, T, D = q.shape
    H, C = k.shape[1], k.shape[2]
    g = Hq // H
    o = torch.zeros((Z, Hq, T, D), dtype=torch.float64, device=q.device)
    total = torch.zeros_like(o)
    lse = torch.full((Z, Hq, T), -math.inf, dtype=torch.float64, device=q.device)
    reach = torch.zeros((Z, Hq, T), dtype=torch.float64, device=q.device)
    weights = torch.zeros((Z, H, C), dtype=torch.float64, device=q.device)
    for z in range(Z):
        n = int(lengths[z])
        t = T if counts is None else max(0, min(T, int(counts[z])))
        if n <= 0 or t == 0:
            continue
        for h in range(H):
            kk, vv = k[z, h, :n].double(), v[z, h, :n].double()
            x = q[z, h * g:(h + 1) * g, :t].double()
            s = torch.matmul(x, kk.T) * scale
            r = torch.matmul(x.abs(), kk.abs().T) * abs(scale)
            if positions is not None:
                at = int(first[z]) + torch.arange(t, device=q.device)
                hidden = positions[z, h, :n][None, :] > at[:, None]
                s = s.masked_fill(hidden, -math.inf)
                r = r.masked_fill(hidden, 0.0)
            else:
                hidden = torch.zeros((t, n), dtype=torch.bool, device=q.device)
            m = torch.logsumexp(s, -1)
            p = torch.where(torch.isinf(m)[..., None] & (m < 0)[..., None], torch.zeros_like(s), torch.exp(s - m[..., None]))
            p = p.masked_fill(hidden, 0.0)
            # a hidden row's values never reach a query, whatever they are
            for i in range(t):
                seen = ~hidden[i]
                o[z, h * g:(h + 1) * g, i] = torch.matmul(p[:, i][:, seen], vv[seen])
                total[z, h * g:(h + 1) * g, i] = torch.matmul(p[:, i][:, seen], vv[seen].abs())
            lse[z, h * g:(h + 1) * g, :t] = m
            reach[z, h * g:(h + 1) * g, :t] = r.amax(-1)
            weights[z, h, :n] = p.sum((0, 1))
    return o, lse, weights, total, reach


def _order(weights, positions, n, recent, sinks):
    """Slots in use in the order they go, and how many of them are unprotected."""
    w, pos = weights[:n].tolist(), positions[:n].tolist()
    newest = max(pos) if pos else 0
    safe = [(recent > 0 and p > newest - recent) or p < sinks for p in pos]
    key = [(1 if s else 0, 0.0 if s else (math.inf if x != x else x), 1 if (not s and x != x) else 0, i)
           for i, (s, x) in enumerate(zip(safe, w))]
    return [k[3] for k in sorted(key)], safe.count(False)


def claim(weights, positions, lengths, n, budget, recent=0, sinks=0):
    """int32 [Z, H, n]."""
    Z, H, _ = weights.shape
    out = torch.full((Z, H, n), -1, dtype=torch.int32)
    for z in range(Z):
        for h in range(H):
            L = int(lengths[z])
            order, loose = _order(weights[z, h], positions[z, h], L, recent, sinks)
            slots = list(range(L, budget))[:n]
            slots += sorted(order[:min(loose, n - len(slots))])
            out[z, h, :len(slots)] = torch.tensor(slots, dtype=torch.int32)
    return out


def evict(weights, positions, lengths, budget, recent=0, sinks=0):
    """Per sequence and head, the list of slots that stay."""
    Z, H, _ = weights.shape
    kept = []
    for z in range(Z):
        L = int(lengths[z])
        kept.append([sorted(_order(weights[z, h], positions[z, h], L, recent, sinks)[0][max(0, L - budget):])
                     for h in range(H)])
    return kept
