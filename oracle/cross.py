"""Definition of cross attention and its gradients, in float64, with bounds on what the kernels may be off by."""
import math

import torch


def attend(q, k, v, lengths, scale):
    """(o, lse) of q [Z, Hq, T, D] over the first lengths[z] rows of k, v [Z, H, N, D] (None: all)."""
    Z, Hq, T, D = q.shape
    H, N = k.shape[1], k.shape[2]
    o, lse = [], []
    for z in range(Z):
        n = N if lengths is None else max(0, min(N, int(lengths[z])))
        for i in range(Hq):
            a, b, c = q[z, i].double(), k[z, i * H // Hq, :n].double(), v[z, i * H // Hq, :n].double()
            if n == 0:
                o.append(a * 0.0)
                lse.append(torch.full((T,), -math.inf, dtype=torch.float64, device=q.device))
                continue
            s = a @ b.T * scale
            lse.append(torch.logsumexp(s, -1))
            o.append(torch.exp(s - lse[-1][:, None]) @ c)
    return torch.stack(o).reshape(Z, Hq, T, D), torch.stack(lse).reshape(Z, Hq, T)


def _like(*shapes, device):
    return [torch.zeros(s, dtype=torch.float64, device=device) for s in shapes]


def expect(q, k, v, lengths, scale, go=None, glse=None):
    """{name: (value, bound)} of o, lse and, with ``go``, dq, dk, dv.

    With h half a step of the type (a rounding is off by h of the value; below the smallest normal number by half a
    subnormal step: float16 2^-25, bfloat16, whose subnormals are 2^-133 apart, 2^-134) and u = 2^-24:

    * a score is off by r = (D + 6) u scale sum |q||k| at most, the sums of exponentials by (n + 16) 2 u, lse
      by both and two roundings of itself; a softmax weight p by e = 2 r + (n + 16) 2 u relative to
      itself, in the gradients' kernels, which take it from lse, by two roundings of lse more;
    * o: weights are rounded to the type, o itself too: (h + e) sum p |v| + h |o|;
    * dv: (h + e + (rows + 16) 2 u) sum p |do| + h |dv|;
    * ds = p (do v - delta): do v is off by (D + 4) u sum |do||v|, delta by the bound of o times |do| (it is made from
      the rounded o) and (D + 6) u sum |o||do|; ds by those times p and (h + e + 4 u) |ds|;
    * float16 weights are scaled by 2^12 before they are rounded for dv, so that half a subnormal step is 2^-37; ds by 2^k, and it is
      2^(-25 - k).  With |do|, |v| the 2-norms of rows, B = |do| max|v| + |delta| of a row for dq, and of a key, with the largest |do|
      and |delta| of the key head's rows, for dk, bounds |ds|.  For dk k is 12 - floor(log2 B), at most 40, so that 2^-k <= 2^-12 B, one
      binade more if B, as 32 bits have it, falls into the next: 2^-11 B.  For dq k may be that of |do| |o| + |delta|, at most
      B (and 2^-11 of it, as o is rounded), less 6, 2^-5 B, or of the largest |do v| + |delta|, at most 2 B: 2^-4 B is more, or 2^-34.  Half a subnormal step is max(2^-36 B, 2^-65) for dk, max(2^-29 B, 2^-59) for dq;
    * k in the exponent, at most 40 where all is finite, adds up to three roundings of (|lse| + 0.7 k) u each to a weight of ds;
    * dq: scale times sum ds' bound |k|, (n + 16) 2 u scale sum |ds||k| for the sums, h |dq|; dk the same with rows and |q|.
    """
    Z, Hq, T, D = q.shape
    H, N = k.shape[1], k.shape[2]
    h, u = torch.finfo(q.dtype).eps / 2, 2.0 ** -24
    tiny = 2.0 ** -25 if q.dtype == torch.float16 else 2.0 ** -134
    dev = q.device
    o, lse = attend(q.detach(), k.detach(), v.detach(), lengths, scale)
    bo, bl = _like(q.shape, q.shape[:3], device=dev)
    dq, dk, dv, bq, bk, bv = _like(q.shape, k.shape, k.shape, q.shape, k.shape, k.shape, device=dev)
    rows = Hq // H * T

    for z in range(Z):
        n = N if lengths is None else max(0, min(N, int(lengths[z])))
        if n == 0:
            continue
        for i in range(Hq):
            j = i * H // Hq
            a, b, c = q[z, i].detach().double(), k[z, j, :n].detach().double(), v[z, j, :n].detach().double()
            s = a @ b.T * scale
            m = lse[z, i][:, None]
            p = torch.exp(s - m)
            r = ((D + 6) * u * abs(scale) * (a.abs() @ b.abs().T)).amax(-1, keepdim=True)
            sums = (n + 16) * 2 * u
            e = 2 * r + sums
            bl[z, i] = (r + sums + 4 * u * m.abs())[:, 0]
            bo[z, i] = (h + e) * (p @ c.abs()) * (1 + h) + h * o[z, i].abs() + tiny * (1 + n * c.abs().amax())
            if go is None:
                continue
            e = e + bl[z, i][:, None] + 4 * u * m.abs()
            d = go[z, i].double()
            heads = slice(j * Hq // H, (j + 1) * Hq // H)
            deltas = (go[z, heads].double() * o[z, heads]).sum(-1, keepdim=True)
            if glse is not None:
                deltas = deltas - glse[z, heads].double()[..., None]
            delta, norms = deltas[i - heads.start], c.norm(dim=-1)[None]
            least_q = least_k = least_v = tiny
            if q.dtype == torch.float16:
                least_v = 2.0 ** -37
                least_q = (2.0 ** -29 * (d.norm(dim=-1, keepdim=True) * norms.max() + delta.abs())).clamp(min=2.0 ** -59)
                least_k = (2.0 ** -36 * (go[z, heads].double().norm(dim=-1).max() * norms + deltas.abs().max())).clamp(min=2.0 ** -65)
                e = e + u * 3 * (m.abs() + 28)
            many = (rows + 16) * 2 * u
            dv[z, j, :n] += p.T @ d
            bv[z, j, :n] += ((h + e + many) * p + least_v).T @ d.abs()
            x = d @ c.T
            ds = p * (x - delta)
            off = (D + 4) * u * (d.abs() @ c.abs().T) + (d.abs() * bo[z, i]).sum(-1, keepdim=True)
            off = off + (D + 6) * u * (d.abs() * o[z, i].abs()).sum(-1, keepdim=True) + 4 * u * (x.abs() + delta.abs())
            bs = p * off + (h + e + 4 * u) * ds.abs()
            dq[z, i] = scale * (ds @ b)
            bq[z, i] = abs(scale) * ((bs + least_q + sums * ds.abs()) @ b.abs())
            dk[z, j, :n] += scale * (ds.T @ a)
            bk[z, j, :n] += abs(scale) * ((bs + least_k + many * ds.abs()).T @ a.abs())
    out = {"o": (o, bo), "lse": (lse, bl)}
    if go is not None:
        for name, x, b in (("dq", dq, bq), ("dk", dk, bk), ("dv", dv, bv)):
            out[name] = (x, b * 1.01 + h * x.abs() * 1.01 + tiny)
    return out
