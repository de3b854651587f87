"""Definitions of the operators on drafted tokens, in float64 and plain loops."""
import math

import torch


def depths(parents):
    """Number of each token's ancestors; parents: a list."""
    d = []
    for i, p in enumerate(parents):
        d.append(d[p] + 1 if 0 <= p < i else 0)
    return d


def seen(parents):
    """bool [T, T]: whether token i sees token j, itself or an ancestor."""
    T = len(parents)
    out = torch.zeros((T, T), dtype=torch.bool)
    for i in range(T):
        j = i
        while True:
            out[i, j] = True
            if not 0 <= parents[j] < j:
                break
            j = parents[j]
    return out


def pack(table):
    """int32 words [..., T, ceil(T / 32)] of a bool table [..., T, T]."""
    T = table.shape[-1]
    words = (T + 31) // 32
    t = torch.zeros(table.shape[:-1] + (32 * words,), dtype=torch.int64)
    t[..., :T] = table
    w = (t.unflatten(-1, (words, 32)) << torch.arange(32)).sum(-1)
    return torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32)


def visible(table, lengths, counts, capacity):
    """bool [Z, T, capacity]: whether drafted token i of sequence z sees a slot; table bool [Z, T, T]."""
    Z, T, _ = table.shape
    out = torch.zeros((Z, T, capacity), dtype=torch.bool)
    for z in range(Z):
        n = max(0, min(int(lengths[z]), capacity))
        t = T if counts is None else max(0, min(T, int(counts[z])))
        context = n - t
        for i in range(t):
            out[z, i, :max(0, context)] = True
            for j in range(t):
                if context + j >= 0:
                    out[z, i, context + j] = table[z, i, j]
    return out


def attend(q, k, v, see, scale):
    """(o, lse, total, reach): attention of q [Z, Hq, T, D] over the rows of k, v [Z, H, C, D] that
    ``see`` [Z, T, C] names.  Rows that see nothing, or only scores of -inf, give 0.  For error bounds:
    ``total``, the sum of softmax weights times |v|, and ``reach`` [Z, Hq, T], the largest scale * sum |q||k| of a seen row."""
    Z, Hq, T, D = q.shape
    g = Hq // k.shape[1]
    o = torch.zeros((Z, Hq, T, D), dtype=torch.float64, device=q.device)
    total, reach = torch.zeros_like(o), torch.zeros((Z, Hq, T), dtype=torch.float64, device=q.device)
    lse = torch.full((Z, Hq, T), -math.inf, dtype=torch.float64, device=q.device)
    for z in range(Z):
        for i in range(T):
            at = see[z, i].nonzero().flatten().to(q.device)
            if len(at) == 0:
                continue
            for h in range(Hq):
                kk, vv, x = k[z, h // g, at].double(), v[z, h // g, at].double(), q[z, h, i].double()
                s = kk @ x * scale
                reach[z, h, i] = (kk.abs() @ x.abs()).max() * abs(scale)
                m = torch.logsumexp(s, -1)
                lse[z, h, i] = m
                if m == -math.inf:
                    continue
                p = torch.exp(s - m)
                o[z, h, i] = p @ vv
                total[z, h, i] = p @ vv.abs()
    return o, lse, total, reach


def keep(buffer, tokens, lengths, counts, value=None):
    """A cache buffer [Z, H, C, ...] after the accepted tokens have moved; ``value(z, j)``: what row j takes instead."""
    out = buffer.clone()
    C = buffer.shape[2]
    for z, row in enumerate(tokens):
        start = max(0, min(int(lengths[z]), C))
        n = len(row) if counts is None else max(0, min(len(row), int(counts[z])))
        for j, t in enumerate(row[:n]):
            if t >= 0 and start + t < C and start + j < C:
                out[z, :, start + j] = buffer[z, :, start + t] if value is None else value(z, j)
    return out
