"""The 4-bit cache on the GPU against the float64 definitions.

append, read, claim and evict are exact.  attend's tolerances follow from what it rounds:

* a score's products (an 11- or 8-bit q times a 2-bit code) are exact in 32 bits; their D sums, the
  product with scale * log2 e and the exponential's argument are off by at most
  r = (D + 4) * 2^-24 * reach, with reach the largest scale * sum |q||k| of a visible key,
  the same for scores of one row, so a softmax weight by 2 r relative to itself;
* the exponential (1 unit) and sums over up to n slots: (n + 16) * 2^-23;
* a weight is rounded to the type before P V, half a step (float16 below 2^-14: 2^-25 at most, of
  weights of which the largest is at least 1), and so is o.
"""
import math

import long_rows
import pytest
import torch

from ascend_rsfa.cache4 import Cache4
from oracle import serving as S

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def _randn(shape, seed, dtype=None, std=1.0):
    t = torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std
    return (t if dtype is None else t.to(dtype)).cuda()


def _filled(Z, H, C, D, dtype, seed, weights=True):
    """A cache whose slots all hold rows (and weights), and their values."""
    cache = Cache4(Z, H, C, D, dtype, weights=weights)
    cache.append(_randn((Z, H, C, D), seed, dtype), _randn((Z, H, C, D), seed + 1, dtype), 0)
    if weights:
        cache.weights.copy_(_randn((Z, H, C), seed + 2).exp())
    return cache


def _ints(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


def _values(cache):
    return S.values(cache.k_codes, cache.k_scales), S.values(cache.v_codes, cache.v_scales)


def _check_attend(cache, got, q, lengths, scale, before=None, positions=None, first=None, counts=None):
    """o, lse and (with `before`, the weights ahead of the call) the cache's weights."""
    o, lse = got
    k, v = _values(cache)
    wo, wl, ww, total, reach = S.attend(q, k, v, lengths, scale, positions, first, counts)
    n = max([int(x) for x in lengths] + [1])
    D, half = q.shape[3], torch.finfo(q.dtype).eps / 2
    r = (D + 4) * 2.0 ** -24 * reach
    sums = (n + 16) * 2.0 ** -23
    rel = 2 * r + sums
    tol = total * (half + rel[..., None]) * (1 + half) + wo.abs() * half
    if q.dtype == F16:
        vmax = torch.nan_to_num(v).abs().amax()
        tol = tol + n * 2.0 ** -25 * vmax + 2.0 ** -25
    assert torch.equal(torch.isnan(o), torch.isnan(wo))
    off = torch.nan_to_num((o.double() - wo).abs() - tol)
    assert (off <= 0).all(), f"o off its tolerance by {off.max().item()}"
    empty = wl == -math.inf
    assert torch.equal(lse == -math.inf, empty) and torch.equal(torch.isnan(lse), torch.isnan(wl))
    off = torch.nan_to_num((lse.double() - wl).abs() - (r + sums + wl.abs() * 2.0 ** -22))
    assert (off[~empty] <= 0).all(), f"lse off its tolerance by {off[~empty].max().item()}"
    if before is not None:
        want = before.double() + ww
        rows = q.shape[1] // cache.H * q.shape[2]
        tol = ww * (2 * reach.amax() * (D + 4) * 2.0 ** -24 + sums + (rows + 4) * 2.0 ** -23) + want.abs() * 2.0 ** -23 + 1e-37
        off = (cache.weights.double() - want).abs() - tol
        assert torch.equal(torch.isnan(cache.weights), torch.isnan(want))
        assert (torch.nan_to_num(off) <= 0).all(), f"weights off their tolerance by {off.max().item()}"


# -- append and read ----------------------------------------------------------
def _expect_rows(cache, k, v, slots, positions):
    """What append leaves in clones of the cache's buffers; slots [Z][H][T] (-1: not written)."""
    want = {n: getattr(cache, n).clone() for n in ("k_codes", "k_scales", "v_codes", "v_scales", "positions", "weights")}
    packed = dict(zip(("k_codes", "k_scales"), S.quantise(k, cache.dtype)))
    packed.update(zip(("v_codes", "v_scales"), S.quantise(v, cache.dtype)))
    for z in range(cache.Z):
        for h in range(cache.H):
            for t, s in enumerate(slots[z][h]):
                if 0 <= s < cache.capacity:
                    for n, rows in packed.items():
                        want[n][z, h, s] = rows[z, h, t]
                    want["positions"][z, h, s] = positions[z] + t
                    want["weights"][z, h, s] = 0.0
    return want


def _same(cache, want):
    for n, t in want.items():
        assert torch.equal(getattr(cache, n), t), n


def _spread(shape, seed, dtype):
    """Rows whose blocks' sizes span the type's range, with zeros and signed zeros."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g, dtype=torch.float64)
    lo, hi = (-24, 15) if dtype == F16 else (-130, 126)
    e = torch.randint(lo, hi, shape[:-1] + (shape[-1] // 32,), generator=g).repeat_interleave(32, -1)
    x = x * torch.pow(torch.tensor(2.0, dtype=torch.float64), e.double())
    x = torch.where(torch.rand(shape, generator=g) < 0.05, torch.zeros_like(x) * x, x)
    top = torch.finfo(dtype).max
    return x.clamp(-top, top).to(dtype).cuda()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
def test_append_and_read_are_exact(D, dtype):
    Z, H, C = 3, 2, 37
    for seed, T in enumerate((1, 5, 37)):
        print(f"append D={D} {dtype} T={T}", flush=True)
        cache = _filled(Z, H, C, D, dtype, 10 * seed)
        k, v = _spread((Z, H, T, D), seed, dtype), _spread((Z, T, H, D), seed + 50, dtype).transpose(1, 2)
        at = [C - T, 0, min(3, C - T)]
        want = _expect_rows(cache, k, v, [[[a + t for t in range(T)]] * H for a in at], at)
        cache.append(k, v, _ints(at))
        _same(cache, want)
        rk, rv = cache.read(_ints(at), T)
        for got, codes, scales in ((rk, cache.k_codes, cache.k_scales), (rv, cache.v_codes, cache.v_scales)):
            full = S.values(codes, scales)
            want_v = torch.stack([full[z, :, a:a + T] for z, a in enumerate(at)])
            assert got.dtype == dtype and torch.equal(got.double(), want_v)  # every value exists in the type


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_every_float16_or_bfloat16_value_is_quantised_exactly(dtype):
    # each finite 16-bit pattern as the only value beside a block's largest
    bits = torch.arange(-(1 << 15), 1 << 15, dtype=torch.int32).to(torch.int16)
    x = bits.view(dtype)
    x = x[torch.isfinite(x)]
    x = x[: x.numel() // 32 * 32]
    near = x.sort()[0].reshape(1, 1, -1, 32).cuda()  # blocks of neighbours
    far = x[torch.randperm(x.numel(), generator=torch.Generator().manual_seed(0))].reshape(1, 1, -1, 32).cuda()
    cache = Cache4(1, 1, near.shape[2], 32, dtype)
    cache.append(near, far, 0)
    for rows, codes, scales in ((near, cache.k_codes, cache.k_scales), (far, cache.v_codes, cache.v_scales)):
        wc, ws = S.quantise(rows, dtype)
        assert torch.equal(scales, ws) and torch.equal(codes, wc)


def test_read_every_code_and_scale():
    for dtype in (F16, BF16):
        cache = Cache4(1, 1, 256, 32, dtype)
        codes = torch.arange(256, dtype=torch.int32).to(torch.uint8).cuda()
        cache.k_codes.copy_((codes[:16] % 16 * 17).expand(256, 16)[None, None])
        cache.v_codes.copy_((codes[:16] * 16 + 15 - codes[:16]).expand(256, 16)[None, None])
        cache.k_scales.copy_(codes[None, None, :, None])
        cache.v_scales.copy_(codes[None, None, :, None])
        k, v = cache.read()
        for got, c, s in ((k, cache.k_codes, cache.k_scales), (v, cache.v_codes, cache.v_scales)):
            want = S.values(c, s).to(dtype)
            assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.nan_to_num(got, 7.0, 8.0, 9.0),
                                                                                   torch.nan_to_num(want, 7.0, 8.0, 9.0))


def test_append_counts_slots_and_edges():
    Z, H, C, D, T = 3, 2, 20, 64, 6
    k, v = _randn((Z, H, T, D), 1, F16), _randn((Z, H, T, D), 2, F16)
    # counts, lengths that leave no room or are out of range
    for lengths, counts in (([0, 17, 20], None), ([-5, 400, 14], [6, 6, 6]), ([3, 3, 3], [0, 2, 9]), ([3, 3, 3], [-1, 1, 6])):
        cache = _filled(Z, H, C, D, F16, 5)
        at = [min(max(x, 0), C) for x in lengths]
        n = [T if counts is None else max(0, min(T, counts[z])) for z in range(Z)]
        slots = [[[at[z] + t if t < n[z] else -1 for t in range(T)]] * H for z in range(Z)]
        want = _expect_rows(cache, k, v, slots, at)
        cache.append(k, v, _ints(lengths), counts=None if counts is None else _ints(counts))
        _same(cache, want)
    # slots of each head, some outside, one named twice (the last token has it), with positions
    g = torch.Generator().manual_seed(4)
    slots = torch.rand((Z, H, C), generator=g).argsort(-1)[..., :T].int()
    slots[0, 0, 2] = -1
    slots[1, 1, 4] = C
    slots[2, 0, 1] = slots[2, 0, 5]
    slots[2, 1, :] = 7
    cache = _filled(Z, H, C, D, F16, 5)
    plain = slots.tolist()
    plain[2][0][1] = -1
    plain[2][1][:5] = [-1] * 5
    want = _expect_rows(cache, k, v, plain, [100, 200, 300])
    cache.append(k, v, C, positions=_ints([100, 200, 300]), slots=slots.cuda())
    _same(cache, want)
    # with counts, a token left out does not take a slot from an earlier one
    cache = _filled(Z, H, C, D, F16, 5)
    plain = slots.tolist()
    plain[2][0][1] = slots[2, 0, 1].item()
    plain[2][1][:] = [-1, -1, 7, -1, -1, -1]
    for z in range(Z):
        for h in range(H):
            plain[z][h][3:] = [-1] * 3
    want = _expect_rows(cache, k, v, plain, [C] * Z)
    cache.append(k, v, C, slots=slots.cuda(), counts=_ints([3, 3, 3]))
    _same(cache, want)


@pytest.mark.parametrize("D", [64, 128])
def test_append_of_many_rows(D):
    # blocks of four rows a thread: counts, slots and lengths that end inside of a block
    Z, H, T = 3, 7, 128 * 256 * 8 // D // 7
    k = _randn((Z, T, H, D), 1, BF16).transpose(1, 2)
    v = _randn((Z, H, T, D), 2, BF16)
    packed = dict(zip(("k_codes", "k_scales", "v_codes", "v_scales"), (*S.quantise(k, BF16), *S.quantise(v, BF16))))
    for use_slots in (False, True):
        cache = _filled(Z, H, T + 50, D, BF16, 7)
        want = {n: getattr(cache, n).clone() for n in (*packed, "positions", "weights")}
        counts, at = [T, 0, T // 2 + 3], [50, 7, 80]
        slots = None
        if use_slots:
            slots = torch.rand((Z, H, T + 50), generator=torch.Generator().manual_seed(3)).argsort(-1)[..., :T].int().cuda()
        for z in range(Z):
            n = min(counts[z], T + 50 - at[z]) if slots is None else counts[z]
            i = torch.arange(n).cuda()
            for h in range(H):
                s = at[z] + i if slots is None else slots[z, h, :n].long()
                for name, rows in packed.items():
                    want[name][z, h, s] = rows[z, h, :n]
                want["positions"][z, h, s] = (at[z] + i).int()
                want["weights"][z, h, s] = 0.0
        cache.append(k, v, _ints(at), counts=_ints(counts), slots=slots)
        _same(cache, want)
        rk, _ = cache.read(_ints(at), T)
        full = S.values(cache.k_codes, cache.k_scales)
        for z in range(Z):
            n = min(T, T + 50 - at[z])
            assert torch.equal(rk[z, :, :n].double(), full[z, :, at[z]:at[z] + n]) and (rk[z, :, n:] == 0).all()


def _owned(cache, k, v, slots, counts, start):
    """What append with slots leaves, of many tokens: the last token that names a slot has it."""
    want = {n: getattr(cache, n).clone() for n in ("k_codes", "k_scales", "v_codes", "v_scales", "positions", "weights")}
    packed = dict(zip(("k_codes", "k_scales", "v_codes", "v_scales"), (*S.quantise(k, cache.dtype), *S.quantise(v, cache.dtype))))
    T, slots = k.shape[2], slots.cpu()
    for z in range(cache.Z):
        n = max(0, min(T, counts[z]))
        for h in range(cache.H):
            s = slots[z, h, :n].long()
            inside = (s >= 0) & (s < cache.capacity)
            owner = torch.full((cache.capacity,), -1).scatter_reduce_(0, s[inside], torch.arange(n)[inside], "amax")
            at = (owner >= 0).nonzero()[:, 0].cuda()
            tok = owner.cuda()[at]
            for name, rows in packed.items():
                want[name][z, h, at] = rows[z, h, tok]
            want["positions"][z, h, at] = (start[z] + tok).int()
            want["weights"][z, h, at] = 0.0
    return want


@pytest.mark.parametrize("Z, H, T, C, D", [
    # few and many tokens, a row or four a thread, more tokens than slots
    (2, 3, 96, 60, 64), (2, 3, 97, 60, 64), (2, 3, 97, 3000, 32), (1, 2, 2000, 1500, 256), (4, 8, 1100, 900, 128), (2, 16, 1100, 5000, 128),
    (3, 7, 1300, 1300, 256),
])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_append_of_many_tokens_into_slots(Z, H, T, C, D, dtype):
    print(f"slots {(Z, H, T, C, D)} {dtype}", flush=True)
    k = _randn((Z, T, H, D), 1, dtype).transpose(1, 2)
    v = _randn((Z, H, T, D), 2, dtype)
    g = torch.Generator().manual_seed(T)
    counts, start = [T, T // 2 + 1, 0, -3][:Z], [2 ** 31 - 3 * T, -7, 100, 5][:Z]
    for kind in range(4):
        slots = torch.randint(-2, C + 2, (Z, H, T), generator=g).int()
        if kind == 1:
            slots[:] = slots[..., :1]  # all one slot
        if kind == 2:
            slots = torch.arange(T).expand(Z, H, T).int().contiguous()  # each its own
        if kind == 3:
            slots = torch.arange(T).flip(0).expand(Z, H, T).div(2, rounding_mode="floor").int().contiguous()
        cache = _filled(Z, H, C, D, dtype, 5, weights=kind != 2)
        if kind == 2:
            before = {n: getattr(cache, n).clone() for n in ("k_codes", "k_scales", "v_codes", "v_scales", "positions")}
        else:
            want = _owned(cache, k, v, slots, counts, start)
        cache.append(k, v, 0, positions=_ints(start), counts=_ints(counts), slots=slots.cuda())
        if kind != 2:
            _same(cache, want)
        else:
            other = Cache4(Z, H, C, D, dtype)
            for n, t in before.items():
                getattr(other, n).copy_(t)
            want = _owned(other, k, v, slots, counts, start)
            del want["weights"]
            _same(cache, want)


def test_append_of_many_tokens_into_slots_in_a_graph():
    Z, H, T, C, D = 2, 4, 500, 700, 64
    k, v = _randn((Z, H, T, D), 1, F16), _randn((Z, H, T, D), 2, F16)
    slots = torch.zeros((Z, H, T), dtype=torch.int32).cuda()
    n = _ints([3, 90])
    cache = _filled(Z, H, C, D, F16, 5)
    cache.append(k, v, n, slots=slots)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.append(k, v, n, slots=slots)
    for turn in range(4):
        slots.copy_(torch.randint(0, C, slots.shape, generator=torch.Generator().manual_seed(turn)))
        k.copy_(k.flip(2))
        n.add_(7)
        want = _owned(cache, k, v, slots, [T] * Z, n.tolist())
        graph.replay()
        torch.cuda.synchronize()
        _same(cache, want)


def test_append_into_slots_grows_with_the_tokens():
    # (when each token looked through all later ones, 4096 tokens of 32 rows took 200 times what consecutive slots take,
    # and twice the tokens twice that; measured: 2.7 times here)
    Z, H, T, D = 1, 8, 16384, 64
    cache = Cache4(Z, H, T, D, BF16)
    k = _randn((Z, H, T, D), 1, BF16)
    slots = torch.rand((Z, H, T), generator=torch.Generator().manual_seed(3)).argsort(-1).int().cuda()

    def us(**more):
        times = []
        for _ in range(7):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            for _ in range(4):
                cache.append(k, k, 0, **more)
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        return sorted(times)[3]

    us()
    assert us(slots=slots) < 40 * us()


def test_non_finite_blocks_are_stored_as_nan():
    cache = Cache4(1, 1, 4, 64, BF16)
    k = _randn((1, 1, 4, 64), 1, BF16)
    v = k.clone()
    k[0, 0, 1, 5] = math.nan
    k[0, 0, 2, 40] = -math.inf
    v[0, 0, 0, 63] = math.inf
    cache.append(k, v, 0)
    assert cache.k_scales[0, 0].eq(255).tolist() == [[False] * 2, [True, False], [False, True], [False] * 2]
    assert cache.v_scales[0, 0].eq(255).tolist() == [[False, True], [False] * 2, [False] * 2, [False] * 2]
    rk, _ = cache.read()
    assert torch.isnan(rk[0, 0, 1, :32]).all() and not torch.isnan(rk[0, 0, 1, 32:]).any()


def test_read_outside_and_by_slots():
    cache = _filled(2, 3, 10, 128, F16, 3)
    k, v = _values(cache)
    rk, rv = cache.read(_ints([-2, 7]), 5)
    for z, a in enumerate((-2, 7)):
        for t in range(5):
            s = a + t
            for got, want in ((rk, k), (rv, v)):
                assert torch.equal(got[z, :, t].double(), want[z, :, s] if 0 <= s < 10 else torch.zeros_like(want[z, :, 0]))
    slots = _ints([[[3, -1, 9], [10, 0, 0], [1, 2, 3]], [[9, 9, 9], [-7, 5, 6], [1 << 30, 4, 8]]])
    rk, rv = cache.read(slots=slots)
    for z in range(2):
        for h in range(3):
            for t in range(3):
                s = int(slots[z, h, t])
                want = v[z, h, s] if 0 <= s < 10 else torch.zeros(128, dtype=torch.float64).cuda()
                assert torch.equal(rv[z, h, t].double(), want)
    a, b = cache.read(4, 3)
    assert torch.equal(a.double(), k[:, :, 4:7]) and torch.equal(b.double(), v[:, :, 4:7])
    assert cache.read(10)[0].shape == (2, 3, 0, 128)


# -- attend -------------------------------------------------------------------
SHAPES = [
    # Z, Hq, H, T, C, D, lengths
    (1, 1, 1, 1, 1, 64, [1]), (2, 4, 2, 1, 33, 128, [33, 0]), (3, 8, 1, 1, 200, 128, [1, 31, 200]),
    (2, 2, 2, 3, 130, 256, [129, 5]), (1, 16, 1, 1, 1000, 64, [999]), (2, 6, 2, 7, 257, 32, [257, 40]),
    (1, 8, 2, 8, 500, 128, [500]), (1, 20, 1, 1, 300, 128, [300]), (1, 4, 1, 40, 700, 64, [700]), (2, 4, 2, 100, 384, 128, [384, 130]),
    (1, 2, 1, 70, 300, 256, [301 - 1]), (1, 3, 3, 260, 290, 32, [290]), (1, 5, 1, 33, 5000, 128, [4097]), (1, 2, 2, 1, 20000, 128, [20000]),
]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("shape", SHAPES)
def test_attend_matches_the_definition(shape, dtype, causal):
    Z, Hq, H, T, C, D, lengths = shape
    print(f"attend {shape} {dtype} causal={causal}", flush=True)
    cache = _filled(Z, H, C, D, dtype, 7)
    q = _randn((Z, T, Hq, D), 8, dtype).transpose(1, 2)
    scale = D ** -0.5
    before = cache.weights.clone()
    got = cache.attend(q, _ints(lengths), causal, scale, accumulate=True, return_lse=True)
    first = [n - T for n in lengths]
    _check_attend(cache, got, q, lengths, scale, before, cache.positions if causal else None, first)
    # without weights, with a bound on the lengths: another division of the work
    plain = cache.attend(q.contiguous(), _ints(lengths), causal, scale, max_length=max(max(lengths), 1), return_lse=True)
    _check_attend(cache, plain, q, lengths, scale, None, cache.positions if causal else None, first)


LONG = [
    # query heads (of one key head), T, slots, length, D
    (1, 1, 20000, 19999, 128), (4, 1, 16000, 16000, 64), (2, 1, 9000, 8130, 256), (1, 1, 4000, 3977, 32), (4, 8, 20000, 16385, 128),
    (1, 32, 9000, 8999, 256), (5, 8, 20000, 19990, 128), (2, 60, 9000, 8190, 64), (1, 100, 9000, 8192, 256), (1, 100, 4000, 3977, 32),
    (3, 150, 20000, 20000, 128), (2, 200, 9000, 8999, 256),
]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("shape", LONG)
def test_every_slot_of_a_long_row_counts(shape, dtype):
    Hq, T, C, n, D = shape
    print(f"long rows {shape} {dtype}", flush=True)
    q = torch.zeros((1, Hq, T, D), dtype=dtype).cuda()
    k = _randn((1, 1, C, D), 3, dtype)
    for step in (1, 32, 512):
        v = long_rows.marked(n, C, D, dtype, step)
        cache = Cache4(1, 1, C, D, dtype)
        cache.append(k, v.cuda(), 0)
        for causal in (False, True):
            cache.weights.zero_()
            pos = _ints([n - 1])  # (causal: every token sees all slots in use)
            o, lse = cache.attend(q, _ints([n]), causal, 1.0, positions=pos, accumulate=causal, return_lse=True)
            assert long_rows.marks_hold(o.cpu(), n, v), (step, causal)
            assert (lse.double() - math.log(n)).abs().max() <= 4 * 2.0 ** -23 * math.log(n)
        want = Hq * T / n
        assert (cache.weights[0, 0, :n].double() - want).abs().max() <= want * (Hq * T + 8) * 2.0 ** -23
        assert not cache.weights[0, 0, n:].any()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("shape", LONG)
def test_peaks_in_every_part_of_a_long_row(shape, dtype):
    Hq, T, C, n, D = shape
    rows = min(Hq * T, D)
    print(f"peaks {shape} {dtype}", flush=True)
    # the ends, and slots all over the row: as many as there are rows, in several calls where those are few
    spread = [0, n - 1, n - 2, 31, 32, 127, 128, 511, n // 32 * 32 - 1, n // 2] + [(i * 617 + 300) % n for i in range(64)]
    spread = list(dict.fromkeys(spread))
    for first in range(0, len(spread), D):
        some = spread[first:first + D]
        k, v, peaks = long_rows.peaks(some, n, C, D, dtype, first)
        cache = Cache4(1, 1, C, D, dtype)
        cache.append(k.cuda(), v.cuda(), 0)
        assert torch.equal(cache.read()[1].cpu(), v)
        for turn in range(0, len(some), rows):
            slots = torch.tensor(some[turn:turn + rows])
            # row i is token i // Hq, head i % Hq; rows without a peak of their own repeat the first ones'
            at = torch.arange(Hq * T) % len(slots)
            q = peaks[turn + at].reshape(T, Hq, D).transpose(0, 1)[None].cuda()
            want = v[0, 0][slots[at]].reshape(T, Hq, D).transpose(0, 1)[None]
            for causal in (False, True):
                cache.weights.zero_()
                o = cache.attend(q, n, causal, 1.0, positions=_ints([n - 1]), accumulate=True)
                assert torch.equal(o.cpu(), want), causal
                count = torch.zeros(C).index_add_(0, slots[at], torch.ones(Hq * T))
                # (a peak's weight is 1 to 2^-16, the others' n e^-40 in all)
                assert ((cache.weights[0, 0].cpu() - count).abs() <= count * 2.0 ** -16 + 2.0 ** -30).all()


@pytest.mark.parametrize("T", [1, 3, 9, 50, 90])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
def test_attend_masks_by_position(D, T):
    # positions in no order, some rows seeing nothing, some tiles seen by no row
    Z, H, Hq, C = 2, 2, 4, 333
    cache = _filled(Z, H, C, D, F16, 3)
    g = torch.Generator().manual_seed(D + T)
    cache.positions.copy_(torch.randint(0, 400, (Z, H, C), generator=g))
    cache.positions[0, 0, 64:256] = 100000
    q = _randn((Z, Hq, T, D), 5, F16)
    for first in ([350, -1 - T // 2], [0, 399], [-100, 2 ** 31 - 1 - T]):
        before = cache.weights.clone()
        got = cache.attend(q, 320, True, 0.1, positions=_ints(first), accumulate=True, return_lse=True)
        _check_attend(cache, got, q, [320] * Z, 0.1, before, cache.positions, first)


@pytest.mark.parametrize("T", [1, 5, 9, 50])
def test_attend_with_counts_of_a_padded_batch(T):
    Z, H, Hq, C, D = 4, 2, 4, 150, 128
    cache = _filled(Z, H, C, D, BF16, 3)
    q = _randn((Z, Hq, T, D), 5, BF16)
    counts, lengths = [T, 0, max(1, T // 2), 1], [150, 70, 33, 1]
    for z in range(Z):
        q[z, :, counts[z]:] = math.nan  # padding
    for causal in (False, True):
        before = cache.weights.clone()
        got = cache.attend(q, _ints(lengths), causal, 0.1, counts=_ints(counts), accumulate=True, return_lse=True)
        _check_attend(cache, got, q, lengths, 0.1, before, cache.positions if causal else None,
                      [n - c for n, c in zip(lengths, counts)], counts)
        for z in range(Z):
            assert (got[0][z, :, counts[z]:] == 0).all() and (got[1][z, :, counts[z]:] == -math.inf).all()


@pytest.mark.parametrize("T", [1, 4, 40, 97])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
def test_non_finite_rows_reach_only_the_queries_that_see_them(D, T):
    Z, H, Hq, C = 1, 2, 4, 140
    cache = _filled(Z, H, C, D, F16, 3)
    # past the length: whatever memory holds
    cache.k_scales[:, :, 100:] = 255
    cache.v_scales[:, :, 100:] = 255
    q = _randn((Z, Hq, T, D), 5, F16)
    for causal in (False, True):
        got = cache.attend(q, 100, causal, 0.1, return_lse=True)
        _check_attend(cache, got, q, [100], 0.1, None, cache.positions if causal else None, [100 - T])
        assert torch.isfinite(got[0]).all()
    # a NaN block of V and of K among the last tokens: seen by the later queries only
    cache.v_scales[0, 0, 100 - (T + 1) // 2, D // 32 - 1] = 255
    cache.k_scales[0, 1, 100 - (T + 1) // 2, 0] = 255
    cache.positions[:, :, 5:9] = 1000  # seen by no query
    before = cache.weights.clone()
    got = cache.attend(q, 100, True, 0.1, accumulate=True, return_lse=True)
    assert torch.equal(cache.weights[:, :, 5:9], before[:, :, 5:9])
    o = got[0]
    seen = T - (T + 1) // 2  # the first query token that sees it
    assert torch.isnan(o[0, :2, seen:, D - 32:]).all() and torch.isfinite(o[0, :2, :, :D - 32]).all()
    assert torch.isfinite(o[0, :, :seen]).all() and torch.isnan(o[0, 2:, seen:]).all()
    _check_attend(cache, got, q, [100], 0.1, before, cache.positions, [100 - T])


def test_scales_and_score_sizes():
    cache = _filled(1, 1, 300, 128, F16, 3)
    q = _randn((1, 2, 3, 128), 5, F16)
    for scale in (-0.2, 0.0, 1.5, 1e-30):
        for T in (3, 1):
            before = cache.weights.clone()
            got = cache.attend(q[:, :, :T], 300, False, scale, accumulate=True, return_lse=True)
            _check_attend(cache, got, q[:, :, :T], [300], scale, before)
    # scores far below and above 0, all alike and peaked
    for dtype, size in ((F16, 300.0), (BF16, 1e4)):
        cache = Cache4(1, 1, 64, 128, dtype)
        k = torch.full((1, 1, 64, 128), 1.0, dtype=dtype).cuda()
        cache.append(k, _randn((1, 1, 64, 128), 3, dtype), 0)
        for sign in (1.0, -1.0):
            q = torch.full((1, 1, 1, 128), sign * size, dtype=dtype).cuda()
            got = cache.attend(q, 64, False, 1.0, return_lse=True)
            _check_attend(cache, got, q, [64], 1.0)


@pytest.mark.parametrize("group, T", [(1, 401), (5, 107), (3, 211), (40, 9)])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
def test_weights_of_many_rows(D, group, T):
    # rows in several parts, which end inside of a block; scales of either sign; fewer tokens than the batch's most
    Z, H, C = 2, 1, 530
    cache = _filled(Z, H, C, D, BF16, 3)
    q = _randn((Z, T, group, D), 5, BF16).transpose(1, 2)
    counts, lengths = [T, T // 2 + 1], [C, 413]
    q[1, :, counts[1]:] = math.nan
    for scale, causal in ((0.11, True), (-0.11, False), (-0.07, True), (0.0, False)):
        before = cache.weights.clone()
        got = cache.attend(q, _ints(lengths), causal, scale, counts=_ints(counts), accumulate=True, return_lse=True)
        _check_attend(cache, got, q, lengths, scale, before, cache.positions if causal else None,
                      [n - c for n, c in zip(lengths, counts)], counts)


def test_overflowing_scores_are_nan_or_dominate_as_in_ieee():
    cache = Cache4(1, 1, 40, 64, BF16)
    k = torch.zeros((1, 1, 40, 64), dtype=BF16).cuda()
    k[0, 0, 7] = 2.0 ** 100
    cache.append(k, _randn((1, 1, 40, 64), 3, BF16), 0)
    q = torch.full((1, 1, 1, 64), 2.0 ** 100, dtype=BF16).cuda()
    o, lse = cache.attend(q, 40, False, 1.0, return_lse=True)
    assert torch.isnan(o).all() and torch.isnan(lse).all()  # inf - inf
    o, lse = cache.attend(-q, 40, False, 1.0, return_lse=True)  # the others share the weight
    v = S.values(cache.v_codes, cache.v_scales)[0, 0]
    want = torch.cat((v[:7], v[8:])).mean(0)
    assert torch.allclose(o[0, 0, 0].double(), want, rtol=0, atol=2.0 ** -8 * v.abs().max().item())


@pytest.mark.parametrize("Hq, T, C", [(2, 1, 40), (2, 1, 5000), (4, 8, 700), (2, 60, 90), (2, 60, 5000)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_rows_whose_scores_are_all_minus_infinity_see_nothing(Hq, T, C, dtype):
    # an infinite q: each visible score is -inf, which is how hidden ones enter the softmax
    D = 64
    cache = Cache4(1, 1, C, D, dtype)
    k = _randn((1, 1, C, D), 1, dtype)
    k[..., 0] = 4.0
    cache.append(k, _randn((1, 1, C, D), 2, dtype), 0)
    cache.weights.copy_(_randn((1, 1, C), 3).exp())
    q = _randn((1, Hq, T, D), 5, dtype)
    q[0, 0, 0] = 0.0
    q[0, 0, 0, 0] = -math.inf
    for causal, scale, n in ((False, 0.1, C), (True, 0.1, C - 3), (False, 1e-30, C - 3)):
        before = cache.weights.clone()
        got = cache.attend(q, n, causal, scale, accumulate=True, return_lse=True)
        assert (got[0][0, 0, 0] == 0).all() and got[1][0, 0, 0] == -math.inf
        first = cache.positions if causal else None
        _check_attend(cache, got, q, [n], scale, None, first, [n - T])
        _, _, ww, _, reach = S.attend(q, *_values(cache), [n], scale, first, [n - T])
        tol = ww * (2 * reach[torch.isfinite(reach)].amax() * (D + 4) * 2.0 ** -24 + (n + 16 + Hq * T + 4) * 2.0 ** -23)
        want = before.double() + ww
        assert ((cache.weights.double() - want).abs() <= tol + want * 2.0 ** -23).all()
    # +inf leaves inf - inf
    q[0, 0, 0, 0] = math.inf
    o, lse = cache.attend(q, C, False, 0.1, return_lse=True)
    assert torch.isnan(o[0, 0, 0]).all() and torch.isnan(lse[0, 0, 0]) and torch.isfinite(o[0, 1:]).all()


def test_strides_of_caches_and_rows():
    # a layer's part of buffers that all layers share, q with gaps, out given
    Z, H, C, D = 2, 3, 50, 64
    big = {"k_codes": torch.zeros((Z, 4, H, C, D // 2), dtype=torch.uint8), "k_scales": torch.zeros((Z, 4, H, C, D // 32), dtype=torch.uint8),
           "v_codes": torch.zeros((Z, 4, H, C, D // 2), dtype=torch.uint8), "v_scales": torch.zeros((Z, 4, H, C, D // 32), dtype=torch.uint8),
           "positions": torch.zeros((Z, 4, H, C), dtype=torch.int32), "weights": torch.zeros((Z, 4, H, C))}
    big = {n: t.cuda() for n, t in big.items()}
    cache = Cache4.from_buffers(**{n: t[:, 2] for n, t in big.items()}, dtype=F16)
    k, v = _randn((Z, H, C, D), 1, F16), _randn((Z, H, C, D), 2, F16)
    cache.append(k, v, 0)
    for n, t in big.items():
        if n != "weights":
            assert (t[:, 2] != 0).any() and not (t[:, [0, 1, 3]] != 0).any(), n
    q = _randn((Z, 6, 2, 2 * D), 3, F16)[..., :D]
    out = torch.full((Z, 2, 6, D), 7.0, dtype=F16).cuda().transpose(1, 2)
    got = cache.attend(q, C, False, 0.2, return_lse=True, accumulate=True, out=out)
    assert got[0] is out
    _check_attend(cache, got, q, [C, C], 0.2, torch.zeros_like(cache.weights))
    odd = torch.zeros((Z, 6, 2, D + 1), dtype=F16).cuda()[..., :D]  # rows that are not 16-byte aligned are copied
    odd.copy_(q)
    assert torch.equal(cache.attend(odd, C, False, 0.2), out)
    assert torch.equal(cache.attend(q[:, :1].expand(Z, 6, 2, D), C, False, 0.2)[:, 5],
                       cache.attend(q[:, :1].expand(Z, 6, 2, D).contiguous(), C, False, 0.2)[:, 5])


@pytest.mark.parametrize("T", [3, 60])
def test_out_beside_q_in_one_buffer(T):
    # heads of q and others' of out in one [Z, T, heads, D] buffer; out and q side by side in each row
    cache = _filled(2, 4, 100, 128, BF16, 3)
    heads = _randn((2, T, 24, 128), 5, BF16)
    rows = _randn((2, 8, T, 256), 6, BF16)
    for whole, q, out in ((heads, heads[:, :, :8].transpose(1, 2), heads[:, :, 16:].transpose(1, 2)),
                          (rows, rows[..., :128], rows[..., 128:])):
        want, before = cache.attend(q, 100, True, 0.1, accumulate=True), whole.clone()
        got = cache.attend(q, 100, True, 0.1, accumulate=True, out=out)
        assert got is out and torch.equal(out, want)
        out.copy_((before[:, :, 16:].transpose(1, 2) if whole is heads else before[..., 128:]))
        assert torch.equal(whole, before)  # nothing beside out was written
    tokens = _randn((1, 48, 32, 128), 7, BF16)
    with pytest.raises(ValueError, match="share memory"):  # tokens 16 .. 31 are both's
        Cache4(1, 4, 64, 128, BF16).attend(tokens[:, :32].transpose(1, 2), 64, False, 1.0, out=tokens[:, 16:].transpose(1, 2))


def test_a_cache_past_four_gibibytes():
    # 2^25 + 1000 slots of 128 code bytes: the last rows' offsets pass 32 bits
    C, D, last = (1 << 25) + 1000, 256, 500
    cache = Cache4(1, 1, C, D, BF16)
    k, v = _randn((1, 1, last, D), 1, BF16), _randn((1, 1, last, D), 2, BF16)
    cache.positions.fill_(1 << 30)  # the others are hidden
    cache.append(k, v, C - last, positions=_ints([0]))
    q = _randn((1, 2, 1, D), 3, BF16)
    small = Cache4(1, 1, last, D, BF16)
    small.append(k, v, 0)
    o, lse = cache.attend(q, C, True, 0.1, positions=_ints([last]), return_lse=True)
    want, want_lse = small.attend(q, last, False, 0.1, return_lse=True)
    assert torch.allclose(o.double(), want.double(), rtol=0, atol=2.0 ** -7 * 4) and torch.allclose(lse, want_lse, rtol=1e-5, atol=1e-5)
    rk, rv = cache.read(C - last, last)
    sk, sv = small.read()
    assert torch.equal(rk, sk) and torch.equal(rv, sv)


def test_results_do_not_change_from_call_to_call():
    cache = _filled(3, 2, 3000, 128, BF16, 3)
    for T in (1, 6, 80):
        q = _randn((3, 8, T, 128), 5, BF16)
        runs = []
        for _ in range(3):
            cache.weights.zero_()
            runs.append((*cache.attend(q, _ints([3000, 17, 1234]), True, 0.1, accumulate=True, return_lse=True),
                         cache.weights.clone()))
        assert all(torch.equal(a, b) for r in runs[1:] for a, b in zip(runs[0], r))


# -- claim and evict ------------------------------------------------------------
def _weights(shape, seed, kind):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(shape, generator=g)
    if kind == "spread":
        w = w.exp()
    elif kind == "ties":
        w = torch.randint(0, 4, shape, generator=g).float()
    elif kind == "zeros":
        w = torch.where(torch.rand(shape, generator=g) < 0.9, torch.zeros_like(w), w)
        w = torch.where(torch.rand(shape, generator=g) < 0.3, -w, w)
    elif kind == "odd":
        r = torch.rand(shape, generator=g)
        w = torch.where(r < 0.1, torch.full_like(w, math.inf), torch.where(r < 0.2, torch.full_like(w, -math.inf), w))
        w = torch.where(r > 0.9, torch.full_like(w, math.nan), torch.where(r > 0.8, w * 1e-42, w * 1e30))
    return w


@pytest.mark.parametrize("kind", ["spread", "ties", "zeros", "odd"])
@pytest.mark.parametrize("C", [1, 5, 64, 2048, 2100, 8192, 8193, 16384, 16385, 32768, 32769, 40000, 140000])
def test_claim_matches_the_definition(C, kind):
    Z, H = 3, 2
    cache = Cache4(Z, H, C, 32)
    w = _weights((Z, H, C), C, kind)
    pos = torch.rand((Z, H, C), generator=torch.Generator().manual_seed(1)).argsort(-1).int()
    cache.weights.copy_(w)
    cache.positions.copy_(pos)
    for lengths in ([C, C, C], [C, C // 2, 0], [max(0, C - 1), 1, C]):
        for n, budget, recent, sinks in ((1, C, 0, 0), (3, C, C // 4, 0), (min(C, 40), C, C // 3, min(2, C // 2)),
                                         (2 * C if C < 100 else 70, max(1, C // 2), 0, 0)):
            got = cache.claim(_ints(lengths), n, budget=budget, recent=recent, sinks=sinks)
            want = S.claim(w, pos, lengths, n, budget, recent, sinks)
            assert torch.equal(got.cpu(), want), (lengths, n, budget, recent, sinks)


@pytest.mark.parametrize("kind", ["spread", "ties", "zeros", "odd"])
@pytest.mark.parametrize("C,D", [(1, 32), (70, 64), (700, 128), (3000, 256), (20000, 64), (40000, 32), (66000, 32),
                                 (70000, 32), (140000, 32)])
def test_evict_matches_the_definition(C, D, kind):
    Z, H = (2, 2) if C < 10000 else (1, 2)
    cache = _filled(Z, H, C, D, F16, 3)
    w = _weights((Z, H, C), C, kind)
    pos = torch.rand((Z, H, C), generator=torch.Generator().manual_seed(1)).argsort(-1).int()
    cache.weights.copy_(w)
    cache.positions.copy_(pos)
    w, pos = w.cpu(), pos.cpu()
    for budget, recent, sinks, lengths in ((max(1, C // 4), C // 16, 0, [C, C // 8][:Z]), (max(1, C - 1), 0, 0, [C, 0][:Z]),
                                           (max(1, C // 2), C // 5, min(4, C // 8), [C, C - 1][:Z])):
        into = _filled(Z, H, max(1, C // 2) + (budget > C // 2) * C, D, F16, 9)
        want = {n: getattr(into, n).clone() for n in ("k_codes", "k_scales", "v_codes", "v_scales", "positions", "weights")}
        kept = S.evict(w, pos, lengths, budget, recent, sinks)
        for z in range(Z):
            for h in range(H):
                at = torch.tensor(kept[z][h], dtype=torch.int64).cuda()
                assert len(at) == min(lengths[z], budget)
                for n, t in want.items():
                    t[z, h, :len(at)] = getattr(cache, n)[z, h][at]
        cache.evict(into, _ints(lengths), budget=budget, recent=recent, sinks=sinks)
        for n, t in want.items():
            assert torch.equal(getattr(into, n).view(torch.int32) if n == "weights" else getattr(into, n),
                               t.view(torch.int32) if n == "weights" else t), n


def test_evict_between_layers_of_one_buffer():
    # two caches whose sequences alternate in memory share none of it
    big = {n: torch.zeros((3, 2, 2, 20) + ((32,) if "codes" in n else (2,) if "scales" in n else ()), dtype=t).cuda() for n, t in (
        ("k_codes", torch.uint8), ("k_scales", torch.uint8), ("v_codes", torch.uint8), ("v_scales", torch.uint8),
        ("positions", torch.int32), ("weights", torch.float32))}
    a, b = (Cache4.from_buffers(**{n: t[:, i] for n, t in big.items()}) for i in range(2))
    k = _randn((3, 2, 20, 64), 1, F16)
    a.append(k, k, 0)
    a.weights.copy_(_randn((3, 2, 20), 2))
    kept = S.evict(a.weights.cpu(), a.positions.cpu(), [20] * 3, 6)
    a.evict(b, 20, budget=6)
    assert b.positions[..., :6].tolist() == kept and (b.positions[..., 6:] == 0).all()


def test_protected_slots_beyond_the_budget_go_by_slot():
    cache = _filled(1, 1, 12, 32, F16, 3)
    cache.positions.fill_(5)  # all of one position: all among the most recent
    into = Cache4(1, 1, 4, 32)
    cache.evict(into, 12, recent=2)
    assert torch.equal(into.k_codes[0, 0], cache.k_codes[0, 0, 8:])
    assert cache.claim(12, 3, recent=2).tolist() == [[[-1, -1, -1]]]


# -- the operators together ---------------------------------------------------
def test_a_generation_under_a_budget():
    """A prompt's rows, its attention's weights, eviction to the budget, then tokens that take over
    the slots of least weight: every step against the definitions."""
    from ascend_rsfa import rotary as R

    Z, H, Hq, D, N, budget = 2, 2, 4, 64, 150, 48
    plan = R.rotary_plan(D, scaling="linear", factor=2.0)
    prompts = [150, 61]
    big, cache = Cache4(Z, H, N, D, BF16), Cache4(Z, H, budget, D, BF16)
    q, k, v = (_randn((Z, h, N, D), s, BF16) for s, h in ((1, Hq), (2, H), (3, H)))
    q, k = R.rotary(q, k, 0, plan)
    counts = _ints(prompts)
    big.append(k, v, 0, counts=counts)
    before = big.weights.clone()
    got = big.attend(q, counts, True, 0.125, counts=counts, accumulate=True, return_lse=True)
    _check_attend(big, got, q, prompts, 0.125, before, big.positions, [0, 0], prompts)
    big.evict(cache, counts, recent=8, sinks=2)
    kept = S.evict(big.weights.cpu(), big.positions.cpu(), prompts, budget, 8, 2)
    for z in range(Z):
        for h in range(H):
            assert cache.positions[z, h].tolist() == kept[z][h]
    for step in range(6):
        q, k, v = (_randn((Z, h, 1, D), 100 * step + s, BF16) for s, h in ((1, Hq), (2, H), (3, H)))
        at = _ints([n + step for n in prompts])
        q, k = R.rotary(q, k, at[:, None], plan)
        w, p = cache.weights.cpu(), cache.positions.cpu()
        slots = cache.claim(budget, 1, recent=8, sinks=2)
        assert torch.equal(slots.cpu(), S.claim(w, p, [budget] * Z, 1, budget, 8, 2))
        cache.append(k, v, budget, positions=at, slots=slots)
        assert torch.equal(cache.positions.gather(2, slots.long())[..., 0], at[:, None].expand(Z, H))
        before = cache.weights.clone()
        assert (before.gather(2, slots.long()) == 0).all()
        got = cache.attend(q, budget, True, 0.125, positions=at, accumulate=True, return_lse=True)
        _check_attend(cache, got, q, [budget] * Z, 0.125, before, cache.positions, at.tolist())


def test_read_rows_feed_the_attention_operator():
    """attention() over read()'s rows is attend() over the cache, to both ones' roundings."""
    from ascend_rsfa.flash_attention_forward import forward

    cache = _filled(2, 4, 128, 64, F16, 3)
    q = _randn((2, 4, 128, 64), 5, F16)
    k, v = cache.read()
    o, lse = forward(q, k, v, True, 0.125, return_lse=True)
    o4, lse4 = cache.attend(q, 128, True, 0.125, return_lse=True)
    _check_attend(cache, (o4, lse4), q, [128, 128], 0.125, None, cache.positions, [0, 0])
    # both round P and o to float16: 2 * 3 half steps of values up to max |v|
    assert (o.double() - o4.double()).abs().max() <= 6 * 2.0 ** -11 * v.abs().max().item()
    assert (lse - lse4).abs().max() <= 2.0 ** -10


def test_steps_in_graphs_with_lengths_that_advance():
    """Two captured graphs of one cache (token and chunk) and eager calls between their replays."""
    Z, H, Hq, C, D = 3, 2, 8, 600, 128
    q1, k1, v1 = (_randn((Z, h, 1, D), s, BF16) for s, h in ((1, Hq), (2, H), (3, H)))
    q5, k5, v5 = (_randn((Z, h, 60, D), s, BF16) for s, h in ((4, Hq), (5, H), (6, H)))
    caches = [_filled(Z, H, C, D, BF16, 20) for _ in range(2)]
    lengths = [_ints([3, 200, 450]) for _ in range(2)]

    def step(cache, n, q, k, v, T):
        cache.append(k, v, n)
        n.add_(T)
        return cache.attend(q, n, True, 0.1, accumulate=True, return_lse=True)

    start = lengths[0].clone()
    for c, n in zip(caches, lengths):  # warm-up
        step(c, n, q1, k1, v1, 1)
        step(c, n, q5, k5, v5, 60)
        n.copy_(start)
        c.weights.zero_()
    torch.cuda.synchronize()
    graphs = []
    for q, k, v, T in ((q1, k1, v1, 1), (q5, k5, v5, 60)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(caches[0], lengths[0], q, k, v, T)
        graphs.append((g, out, q, k, v, T))
    for turn in (0, 1, 0, 0, 1):
        g, out, q, k, v, T = graphs[turn]
        for t in (q, k, v):
            t.copy_(t.flip(-1))
        g.replay()
        torch.cuda.synchronize()
        want = step(caches[1], lengths[1], q, k, v, T)
        assert torch.equal(lengths[0], lengths[1])
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        assert torch.equal(caches[0].weights, caches[1].weights)
        _check_attend(caches[0], out, q, lengths[0].tolist(), 0.1, None, caches[0].positions, [n - T for n in lengths[0].tolist()])


def test_two_streams_at_once():
    caches = [_filled(2, 2, 3000, 128, F16, s) for s in (1, 50)]
    qs = [_randn((2, 8, 1, 128), s, F16) for s in (2, 3)]
    want = [c.attend(q, 3000, False, 0.1) for c, q in zip(caches, qs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(caches[i].attend(qs[i], 3000, False, 0.1))
                got[i].append(caches[i].claim(3000, 4))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i][::2]) and all(torch.equal(s, got[i][1]) for s in got[i][1::2])


# -- refusals -----------------------------------------------------------------
def test_buffers_that_share_memory_are_refused():
    def buffers(C=20):
        return {n: torch.zeros((3, 2, C) + ((32,) if "codes" in n else (2,) if "scales" in n else ()), dtype=t).cuda() for n, t in (
            ("k_codes", torch.uint8), ("k_scales", torch.uint8), ("v_codes", torch.uint8), ("v_scales", torch.uint8),
            ("positions", torch.int32), ("weights", torch.float32))}

    a, big = buffers(), buffers(40)
    first, second = ({n: t[:, :, i:i + 20] for n, t in big.items()} for i in (0, 20))  # halves of one cache's slots
    into, cache = Cache4.from_buffers(**second), Cache4.from_buffers(**first)
    cache.evict(into, 20, budget=3)
    swapped = dict(first, k_codes=second["v_codes"], v_codes=second["k_codes"])
    for bad in (lambda: Cache4.from_buffers(**dict(a, v_codes=a["k_codes"])),
                lambda: Cache4.from_buffers(**dict(a, weights=a["positions"].view(torch.float32))),
                lambda: Cache4.from_buffers(**dict(a, k_scales=a["k_codes"].view(-1)[:240].view(3, 2, 20, 2))),
                # heads 16 slots apart, of 20 each; sequences that meet the heads of the one before
                lambda: Cache4.from_buffers(**{n: t.as_strided(t.shape, (64 * t[0, 0, 0].numel(), 16 * t[0, 0, 0].numel()) + t.stride()[2:])
                                               for n, t in big.items()}),
                lambda: Cache4.from_buffers(**{n: t.as_strided((3, 2) + t.shape[2:], (t.stride(1), t.stride(1)) + t.stride()[2:])
                                               for n, t in a.items()}),
                lambda: cache.evict(Cache4.from_buffers(**first), 20, budget=3),
                lambda: into.evict(Cache4.from_buffers(**swapped), 20, budget=3)):
        with pytest.raises(ValueError, match="share memory"):
            bad()


def test_refusals():
    cache = Cache4(2, 2, 16, 64, F16)
    bare = Cache4(2, 2, 16, 64, F16, weights=False)
    k = torch.zeros((2, 2, 4, 64), dtype=F16).cuda()
    q = torch.zeros((2, 4, 4, 64), dtype=F16).cuda()
    n = _ints([4, 4])
    for bad in (lambda: cache.append(k, k[:, :, :2], 0), lambda: cache.append(k[:, :1], k[:, :1], 0), lambda: cache.append(k, k, 13),
                lambda: cache.append(k, k, -1), lambda: cache.append(k[:1], k[:1], 0), lambda: cache.append(k[..., :32], k[..., :32], 0),
                lambda: cache.append(k, k, 0, slots=torch.zeros((2, 2, 3), dtype=torch.int32).cuda()),
                lambda: cache.append(k, k, 0, slots=torch.zeros((2, 2, 4)).cuda()),
                lambda: cache.append(k, k, n.cpu()), lambda: cache.read(10, 7), lambda: cache.read(n), lambda: cache.read(-1, 2),
                lambda: cache.attend(q[:, :3], n, False, 1.0), lambda: cache.attend(q[:1], n, False, 1.0),
                lambda: cache.attend(q, 17, False, 1.0), lambda: cache.attend(q, n, False, math.nan),
                lambda: cache.attend(q, n, False, 1.0, max_length=0), lambda: cache.attend(q, n, False, 1.0, max_length=17),
                lambda: cache.attend(q, 5, False, 1.0, max_length=4), lambda: cache.attend(q, n, False, 1.0, out=q[:, :2]),
                lambda: bare.attend(q, n, False, 1.0, accumulate=True), lambda: bare.claim(4, 1), lambda: bare.evict(cache, 4),
                lambda: cache.claim(n, 0), lambda: cache.claim(n, 1, budget=17), lambda: cache.claim(n, 1, budget=0),
                lambda: cache.claim(n, 1, recent=10, sinks=7), lambda: cache.claim(n, 1, recent=-1), lambda: cache.claim(17, 1),
                lambda: cache.evict(cache, n), lambda: cache.evict(Cache4.from_buffers(**{
                    x: getattr(cache, x)[:, :, :8] for x in ("k_codes", "k_scales", "v_codes", "v_scales", "positions", "weights")}), n),
                lambda: cache.attend(q, n, False, 1.0, out=q), lambda: cache.attend(q, n, False, 1.0, out=q[:, :1].expand(2, 4, 4, 64)),
                lambda: cache.evict(Cache4(2, 2, 8, 64, BF16), n),
                lambda: cache.evict(Cache4(2, 2, 8, 32, F16), n), lambda: cache.evict(Cache4(1, 2, 8, 64, F16), n),
                lambda: cache.evict(Cache4(2, 2, 8, 64, F16), n, budget=9), lambda: cache.evict(Cache4(2, 2, 8, 64, F16), n, recent=9)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: cache.append(k.bfloat16(), k.bfloat16(), 0), lambda: cache.attend(q.float(), n, False, 1.0),
                lambda: cache.append(k, k, n.long()), lambda: cache.attend(q, n[:1], False, 1.0),
                lambda: cache.attend(q, n, False, 1.0, counts=[4, 4]), lambda: cache.append(k, k, 1.5), lambda: cache.evict(None, n)):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: cache.attend(q.clone().requires_grad_(), n, False, 1.0), lambda: cache.append(k.clone().requires_grad_(), k, 0)):
        with pytest.raises(RuntimeError, match="no gradients"):
            bad()
        with torch.no_grad():
            bad()
    b = {x: getattr(cache, x) for x in ("k_codes", "k_scales", "v_codes", "v_scales", "positions", "weights")}
    for over in ({"k_codes": b["k_codes"][..., :24]}, {"k_scales": b["k_scales"].float()}, {"v_codes": b["v_codes"].cpu()},
                 {"positions": b["positions"].long()}, {"weights": b["weights"][:, :, :8]},
                 {"v_codes": torch.zeros((2, 2, 17, 32), dtype=torch.uint8).cuda()[:, :, :16]},
                 {"k_codes": torch.zeros((2, 2, 32, 16), dtype=torch.uint8).cuda().transpose(2, 3)},
                 {"positions": torch.zeros((1, 2, 16), dtype=torch.int32).cuda().expand(2, 2, 16), "weights": None},
                 {"k_codes": torch.zeros(2 * 2 * 16 * 32 + 8, dtype=torch.uint8).cuda()[8:].reshape(2, 2, 16, 32)}):
        with pytest.raises(ValueError):
            Cache4.from_buffers(**{**b, **over})
    with pytest.raises(TypeError):
        Cache4.from_buffers(**b, dtype=torch.float32)


def test_empty_calls():
    cache = _filled(2, 2, 16, 64, F16, 1)
    want = {n: getattr(cache, n).clone() for n in ("k_codes", "positions", "weights")}
    none = torch.empty((2, 2, 0, 64), dtype=F16).cuda()
    cache.append(none, none, 16)
    o, lse = cache.attend(none, 16, True, 1.0, accumulate=True, return_lse=True)
    assert o.shape == (2, 2, 0, 64) and lse.shape == (2, 2, 0)
    o, lse = cache.attend(_randn((2, 4, 3, 64), 1, F16), 0, False, 1.0, accumulate=True, return_lse=True)
    assert (o == 0).all() and (lse == -math.inf).all()
    _same(cache, want)
