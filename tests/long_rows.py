"""Rows of a cache of which each slot, or one, decides an output, so that a part of a long row that
is lost, taken twice or read from elsewhere shows.

Marks: all scores are 0, and V is 1 in one dim of each slot, 0 in the others. Every softmax weight is
1 / n, and no sum rounds (whole numbers below 2^24), so o is count / n to the
division and product (4 units of 2^-24) and its own rounding, half a step. What is wrong by more than
two half steps cannot round into that: one slot of up to 2^10 a dim in float16, of 2^7 in bfloat16, where 32
neighbours, a dim's own where 32 share it, show in longer rows.

Peaks: row i scores 40 for one slot and 0 for the others, whose weights, n * e^-40 in all, are below 2^-40.
The peak's own, exp2 of the difference of two roundings of 40 log2 e, is within 2^-18 of 1: o is that slot's V,
which rounds to itself, as V has two significant bits.
"""
import torch


def marked(n, C, D, dtype, step):
    """V [1, 1, C, D]: slot s marks dim s // step % D; past n (other slots' memory) all are 1."""
    v = torch.zeros((C, D))
    s = torch.arange(n)
    v[s, s // step % D] = 1.0
    v[n:] = 1.0
    return v.to(dtype)[None, None]


def marks_hold(o, n, v):
    """Whether o [..., D], attention of equal scores over the first n rows of v, is right."""
    want = v[0, 0, :n].double().sum(0) / n
    half = torch.finfo(o.dtype).eps / 2
    tol = want * (half + 4 * 2.0 ** -24 * (1 + half)) + (2.0 ** -25 if o.dtype == torch.float16 else 0.0)
    return bool(((o.double() - want).abs() <= tol).all())


def peaks(slots, n, C, D, dtype, seed):
    """(k, v [1, 1, C, D], q [len(slots), D]): with a scale of 1 row i of q has its peak at slots[i] (at most D)."""
    k = torch.zeros((C, D))
    for i, s in enumerate(slots):
        k[s, i] = 4.0
    k[n:] = 4.0
    q = 10.0 * torch.eye(D)[: len(slots)]
    # V of codes that append keeps: each block's largest is 6 times its scale
    g = torch.Generator().manual_seed(seed)
    v = torch.tensor([0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])[torch.randint(0, 7, (C, D), generator=g)]
    v = v * (torch.randint(0, 2, (C, D), generator=g) * 2 - 1)
    v[:, ::32] = 6.0
    return k.to(dtype)[None, None], v.to(dtype)[None, None], q.to(dtype)
