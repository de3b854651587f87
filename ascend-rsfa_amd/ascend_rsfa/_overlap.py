"""Whether strided tensors share bytes.

A tensor is taken as runs: its trailing ``dense`` dims (each row of a run after the other) are one run
of bytes, the dims before them, of any strides, place the runs.  Exact, from strides alone
where one stride after another holds all that lies within it, as in heads or tokens of a fused
buffer; other placements are compared run by run.
"""
import functools

import torch

__all__ = ["span", "meet", "meets_itself"]


def _placed(t, dense):
    """(first byte, ((stride, size) of the outer dims, in bytes), bytes of a run)."""
    size = t.element_size()
    run = size
    for n in t.shape[t.dim() - dense:]:
        run *= n
    dims = tuple((s * size, n) for s, n in zip(t.stride()[:t.dim() - dense], t.shape) if n > 1)
    return t.data_ptr(), dims, run


def _end(at, dims, run):
    return at + sum(s * (n - 1) for s, n in dims) + run


def span(t):
    """First byte of a tensor and the one behind its last."""
    return t.data_ptr(), _end(*_placed(t, 0))


def _starts(at, dims):
    x = torch.tensor([at], dtype=torch.int64, device="cpu")
    for s, n in dims:
        x = (x[:, None] + s * torch.arange(n, device="cpu")).flatten()
    return x


@functools.lru_cache(maxsize=1024)
def _runs_meet(at, a, run_a, b, run_b):
    """Runs at `at` and at 0, one by one."""
    other = _starts(0, b).sort()[0]
    mine = _starts(at, a)
    # the last run of b that starts before the end of a run of a reaches past its start, or none does
    i = torch.searchsorted(other, mine + run_a) - 1
    return bool(((i >= 0) & (other[i.clamp(min=0)] + run_b > mine)).any())


def meet(a, b, dense_a=1, dense_b=1):
    """Whether a and b (not empty) share a byte."""
    at, da, ra = _placed(a, dense_a)
    bt, db, rb = _placed(b, dense_b)
    at -= bt
    while True:
        first, last = min(at, 0), max(_end(at, da, ra), _end(0, db, rb))
        if last - first >= _end(0, da, ra) + _end(0, db, rb):
            return False
        if not da and not db:
            return True
        # a step that both have and that holds the rest of both: a block of one meets the same block of the
        # other at most, and all of them as the first ones do
        for s in sorted({s for s, _ in da} & {s for s, _ in db}, reverse=True):
            ia, ib = (next(i for i, d in enumerate(dims) if d[0] == s) for dims in (da, db))
            rest_a, rest_b = da[:ia] + da[ia + 1:], db[:ib] + db[ib + 1:]
            if max(_end(at, rest_a, ra), _end(0, rest_b, rb)) - min(at, 0) <= s:
                da, db = rest_a, rest_b
                break
        else:
            return _runs_meet(at, da, ra, db, rb)


@functools.lru_cache(maxsize=1024)
def _runs_overlap(dims, run):
    x = _starts(0, dims).sort()[0]
    return bool((x[1:] - x[:-1] < run).any())


def meets_itself(t, dense=1):
    """Whether two runs of t (not empty) share a byte."""
    _, dims, run = _placed(t, dense)
    need = run
    for s, n in sorted(dims):
        if s < need:
            return _runs_overlap(dims, run)
        need += s * (n - 1)
    return False
