"""Trees of drafted tokens on the GPU against the definitions: tables and moved rows exactly, attention in float64.

attend's tolerances are those of attention over the cache without a tree: a score is off by at most
r = (D + 4) * 2^-24 * reach, a softmax weight by 2 r relative to itself, sums and exponentials by
(n + 16) * 2^-23, and a weight and o are rounded to the type once each, half a step (float16 below 2^-14:
2^-25 at most, of weights of which the largest is at least 1).
"""
import math

import pytest
import torch

from ascend_rsfa.cache4 import Cache4
from ascend_rsfa.draft import DraftTree, draft_tree
from oracle import draft as O
from oracle import serving as S

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
BUFFERS = ("k_codes", "k_scales", "v_codes", "v_scales", "positions", "weights")


def _randn(shape, seed, dtype=None, std=1.0):
    t = torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std
    return (t if dtype is None else t.to(dtype)).cuda()


def _ints(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


def _parents(T, seed, kind="random"):
    g = torch.Generator().manual_seed(seed)
    if kind == "chain":
        return list(range(-1, T - 1))
    if kind == "roots":
        return [-1] * T
    return [int(torch.randint(-1, i, (1,), generator=g)) if i else -1 for i in range(T)]


def _filled(Z, H, C, D, dtype, seed):
    cache = Cache4(Z, H, C, D, dtype)
    cache.append(_randn((Z, H, C, D), seed, dtype), _randn((Z, H, C, D), seed + 1, dtype), 0)
    cache.weights.copy_(_randn((Z, H, C), seed + 2).exp())
    return cache


def _check(cache, got, q, see, scale):
    o, lse = got
    k, v = S.values(cache.k_codes, cache.k_scales), S.values(cache.v_codes, cache.v_scales)
    wo, wl, total, reach = O.attend(q, k, v, see, scale)
    n = max(int(see.sum(-1).max()), 1)
    D, half = q.shape[3], torch.finfo(q.dtype).eps / 2
    r = (D + 4) * 2.0 ** -24 * reach
    sums = (n + 16) * 2.0 ** -23
    tol = total * (half + (2 * r + sums)[..., None]) * (1 + half) + wo.abs() * half
    if q.dtype == F16:
        tol = tol + n * 2.0 ** -25 * torch.nan_to_num(v).abs().amax() + 2.0 ** -25
    assert torch.equal(torch.isnan(o), torch.isnan(wo))
    off = torch.nan_to_num((o.double() - wo).abs() - tol)
    assert (off <= 0).all(), f"o off its tolerance by {off.max().item()}"
    empty = wl == -math.inf
    assert torch.equal(lse == -math.inf, empty) and torch.equal(torch.isnan(lse), torch.isnan(wl))
    off = torch.nan_to_num((lse.double() - wl).abs() - (r + sums + wl.abs() * 2.0 ** -22))
    assert (off[~empty] <= 0).all(), f"lse off its tolerance by {off[~empty].max().item()}"


# -- tables -------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["random", "chain", "roots"])
@pytest.mark.parametrize("T", [1, 2, 7, 31, 32, 33, 64, 100, 511, 512])
def test_tables_and_depths(T, kind):
    parents = [_parents(T, 5 + i, kind) for i in range(3)]
    tree = draft_tree(_ints(parents))
    assert torch.equal(tree.bits.cpu(), O.pack(torch.stack([O.seen(p) for p in parents])))
    assert torch.equal(tree.depths.cpu(), torch.tensor([O.depths(p) for p in parents], dtype=torch.int32))
    one = draft_tree(_ints(parents)[1])
    assert (one.trees, one.tokens) == (1, T) and torch.equal(one.bits, tree.bits[1:2])
    # every second tree and token of a larger table
    wide = _ints([[x for p in row for x in (p, 7)] for row in parents for _ in range(2)])[::2, ::2]
    assert torch.equal(draft_tree(wide).bits, tree.bits)


def test_parents_that_are_no_earlier_token_are_the_context():
    parents = [0, 0, 2, 9, -7, 3, 6, 2 ** 31 - 1]
    tree = draft_tree(_ints(parents))
    assert torch.equal(tree.bits.cpu(), O.pack(O.seen(parents))[None])
    assert tree.depths.tolist() == [O.depths(parents)] == [[0, 1, 0, 0, 0, 1, 0, 0]]


# -- attention ----------------------------------------------------------------
# (Z, Hq, H, T, lengths, counts): few rows and many, one tree and one a sequence, drafts across tiles and parts of a row
SHAPES = [
    (1, 2, 2, 1, [1], None), (2, 4, 2, 5, [5, 70], None), (3, 4, 1, 8, [40, 8, 1000], [8, 0, 3]),
    (2, 2, 2, 31, [500, 31], [31, 30]), (2, 4, 2, 16, [16, 4100], None), (1, 8, 1, 25, [2050], None),
    (2, 4, 4, 64, [64, 777], [64, 50]), (1, 2, 1, 97, [97 + 61], None), (1, 1, 1, 200, [3333], None), (1, 4, 2, 130, [9000], None),
    (2, 4, 1, 25, [4100, 30], [25, 17]), (1, 2, 2, 128, [900], None), (1, 2, 1, 33, [333], None),
]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("shape", SHAPES)
def test_attend_matches_the_definition(shape, D, dtype):
    Z, Hq, H, T, lengths, counts = shape
    C = max(lengths) + 3
    cache = _filled(Z, H, C, D, dtype, 3)
    q = _randn((Z, Hq, T, D), 9, dtype)
    trees = [_parents(T, 11 + z) for z in range(Z)]
    for parents in (trees, trees[:1]):
        tree = draft_tree(_ints(parents) if len(parents) > 1 else _ints(parents[0]))
        table = torch.stack([O.seen(p) for p in parents]).expand(Z, T, T)
        see = O.visible(table, lengths, counts, C)
        got = cache.attend(q, _ints(lengths), True, D ** -0.5, counts=None if counts is None else _ints(counts), return_lse=True, tree=tree)
        _check(cache, got, q, see, D ** -0.5)


@pytest.mark.parametrize("T", [6, 70])
def test_tables_of_the_callers_own_and_rows_that_see_nothing(T):
    # any table, tokens that do not see themselves, words past the tokens; sequences without a context
    Z, H, D = 3, 2, 64
    table = torch.rand((Z, T, T), generator=torch.Generator().manual_seed(1)) < 0.2
    table[:, 1] = False
    bits = O.pack(table)
    if T % 32:
        bits[..., -1] |= -1 << T % 32  # of no token
    lengths, counts = [T, T + 40, 4], [T, T, 4]
    cache = _filled(Z, H, T + 50, D, BF16, 5)
    q = _randn((Z, 4, T, D), 2, BF16)
    o, lse = cache.attend(q, _ints(lengths), True, 0.2, counts=_ints(counts), return_lse=True, tree=DraftTree(bits.cuda()))
    see = O.visible(table, lengths, counts, T + 50)
    assert not see[0, 1].any()
    _check(cache, (o, lse), q, see, 0.2)
    # fewer slots in use than drafted tokens: the first ones have no slot
    see = O.visible(table, [4] * Z, None, T + 50)
    _check(cache, cache.attend(q, 4, True, -0.3, return_lse=True, tree=DraftTree(bits.cuda())), q, see, -0.3)
    o, lse = cache.attend(q, 0, True, 0.2, return_lse=True, tree=DraftTree(bits.cuda()))
    assert (o == 0).all() and (lse == -math.inf).all()


@pytest.mark.parametrize("T", [4, 40, 97])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
def test_non_finite_rows_reach_only_the_tokens_that_see_them(D, T):
    Z, H, context = 1, 2, 45
    C = context + T
    k, v = _randn((Z, H, C, D), 1, F16), _randn((Z, H, C, D), 2, F16)
    v[:, 0, context + 1] = math.nan
    v[:, 1, context + 2, :D // 2] = math.inf
    k[:, 1, context] = math.nan
    cache = Cache4(Z, H, C, D, F16)
    cache.append(k, v, 0)
    parents = _parents(T, 4)
    q = _randn((Z, 4, T, D), 3, F16)
    see = O.visible(O.seen(parents)[None], [C], None, C)
    got = cache.attend(q, C, True, 0.1, return_lse=True, tree=draft_tree(_ints(parents)))
    assert torch.isnan(got[0]).any() and not torch.isnan(got[0]).all()
    _check(cache, got, q, see, 0.1)


def test_positions_do_not_hide_the_context():
    # slots of an evicted cache hold positions in no order
    cache = _filled(1, 2, 60, 64, F16, 1)
    cache.positions.copy_(torch.randperm(1000, generator=torch.Generator().manual_seed(1))[:120].reshape(1, 2, 60).int())
    q, parents = _randn((1, 2, 9, 64), 2, F16), _parents(9, 3)
    got = cache.attend(q, 60, True, 0.125, return_lse=True, tree=draft_tree(_ints(parents)))
    _check(cache, got, q, O.visible(O.seen(parents)[None], [60], None, 60), 0.125)


@pytest.mark.parametrize("T", [6, 40, 130])
def test_into_an_output_of_the_callers_with_a_bound_on_the_lengths(T):
    cache, q = _filled(2, 2, 900, 64, BF16, 1), _randn((2, 4, T, 64), 2, BF16)
    parents = _parents(T, 3)
    wide = torch.full((2, T, 4, 80), 7.0, dtype=BF16, device="cuda")
    out = wide[..., :64].transpose(1, 2)
    o, lse = cache.attend(q, _ints([T + 300, T]), True, 0.1, tree=draft_tree(_ints(parents)), max_length=T + 300, out=out, return_lse=True)
    assert o is out and (wide[..., 64:] == 7.0).all()
    _check(cache, (o, lse), q, O.visible(O.seen(parents)[None].repeat(2, 1, 1), [T + 300, T], None, 900), 0.1)


def test_keep_with_counts_outside_and_a_token_twice():
    cache = _filled(3, 2, 60, 64, BF16, 4)
    tokens, lengths, counts = [[4, 4, 4], [2, 2, 9], [0, 1, 2]], [20, 30, 40], [99, 3, -5]
    want = _expect_kept(cache, tokens, lengths, [3, 3, 0], lengths)
    cache.keep(_ints(tokens), _ints(lengths), counts=_ints(counts))
    _same(cache, want)


def test_a_chain_sees_what_causal_tokens_see():
    for T in (7, 60):
        cache = _filled(2, 2, 500, 128, BF16, 1)
        q, n = _randn((2, 8, T, 128), 2, BF16), _ints([500, 333])
        tree = draft_tree(_ints(_parents(T, 0, "chain")))
        assert torch.equal(cache.attend(q, n, True, 0.1, tree=tree), cache.attend(q, n, True, 0.1))


# -- keep ---------------------------------------------------------------------
def _expect_kept(cache, tokens, lengths, counts, positions=None):
    at = positions if positions is not None else lengths
    want = {n: O.keep(getattr(cache, n), tokens, lengths, counts) for n in BUFFERS if getattr(cache, n) is not None}
    want["positions"] = O.keep(cache.positions, tokens, lengths, counts, lambda z, j: at[z] + j)
    return want


def _same(cache, want):
    for n, t in want.items():
        assert torch.equal(getattr(cache, n), t), n


@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("n", [1, 5, 40, 300, 512])
def test_keep_moves_rows_exactly(n, D):
    Z, H, T = 3, 2, 512
    cache = _filled(Z, H, 700, D, F16, n)
    g = torch.Generator().manual_seed(n)
    paths = [sorted(torch.randperm(T, generator=g)[:n].tolist()) for _ in range(Z)]
    mixed = [torch.randint(-3, T + 200, (n,), generator=g).tolist() for _ in range(Z)]  # any order, twice, outside
    for tokens in (paths, mixed):
        for lengths, counts, positions in (([0, 100, 188], None, None), ([3, 500, 700], [n, n // 2, n], [7, 9000, 5]), ([1, 2, 3], [0, -4, n + 9], None)):
            want = _expect_kept(cache, tokens, lengths, counts, positions)
            cache.keep(_ints(tokens), _ints(lengths), counts=None if counts is None else _ints(counts),
                       positions=None if positions is None else _ints(positions))
            _same(cache, want)
    want = _expect_kept(cache, paths, [10] * Z, None)
    cache.keep(_ints(paths), 10)
    _same(cache, want)


def test_keep_in_strided_buffers_without_weights():
    big = _filled(4, 6, 64, 64, BF16, 1)
    part = {n: getattr(big, n)[1::2, ::3] for n in BUFFERS[:5]}
    cache = Cache4.from_buffers(**part, dtype=BF16)
    rest = {n: getattr(big, n).clone() for n in BUFFERS}
    tokens, lengths = [[2, 3, 9], [0, 8, 1]], [5, 50]
    want = _expect_kept(cache, tokens, lengths, None)
    cache.keep(_ints(tokens), _ints(lengths))
    _same(cache, want)
    for n in BUFFERS:
        t = getattr(big, n).clone()
        if n != "weights":
            t[1::2, ::3] = rest[n][1::2, ::3]
        assert torch.equal(t, rest[n]), n


def test_lengths_outside_the_cache_are_its_ends():
    cache = _filled(2, 1, 30, 32, F16, 1)
    tokens = [[1, 2], [0, 1]]
    want = _expect_kept(cache, tokens, [-5, 99], None, [0, 30])
    cache.keep(_ints(tokens), _ints([-5, 99]))
    _same(cache, want)


# -- in a program ------------------------------------------------------------
def test_steps_in_a_graph():
    Z, H, T, D = 2, 2, 12, 64
    cache, other = _filled(Z, H, 300, D, F16, 1), _filled(Z, H, 300, D, F16, 1)
    q, k, v = _randn((Z, 4, T, D), 4, F16), _randn((Z, H, T, D), 5, F16), _randn((Z, H, T, D), 6, F16)
    parents, path = _ints([_parents(T, z) for z in range(Z)]), _ints([[0, 3, 7], [1, 2, 11]])
    lengths, counts = _ints([100, 90]), _ints([3, 2])

    def step(c, n):
        tree = draft_tree(parents)
        c.append(k, v, n)
        o = c.attend(q, n + T, True, 0.1, tree=tree)
        c.keep(path, n, counts=counts)
        n += counts
        return o

    mine = lengths.clone()
    step(other, mine.clone())  # (first calls outside of the capture)
    for name in BUFFERS:
        getattr(other, name).copy_(getattr(cache, name))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = step(cache, lengths)
    for i in range(4):
        parents.copy_(_ints([_parents(T, 10 * i + z) for z in range(Z)]))
        q.mul_(1.1)
        graph.replay()
        want = step(other, mine)
        torch.cuda.synchronize()
        assert torch.equal(o, want) and torch.equal(lengths, mine)
        _same(cache, {n: getattr(other, n) for n in BUFFERS})


def test_other_streams():
    caches = [_filled(2, 2, 3000, 128, F16, s) for s in (1, 50)]
    qs = [_randn((2, 8, T, 128), T, F16) for T in (5, 40)]
    trees = [_ints(_parents(T, T)) for T in (5, 40)]
    want = [c.attend(q, 3000, True, 0.1, tree=draft_tree(p)) for c, q, p in zip(caches, qs, trees)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(caches[i].attend(qs[i], 3000, True, 0.1, tree=draft_tree(trees[i])))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in range(2) for o in got[i])


# -- refusals -----------------------------------------------------------------
def test_refusals():
    cache = _filled(2, 2, 40, 64, F16, 1)
    q, n = _randn((2, 4, 6, 64), 1, F16), _ints([20, 30])
    tree, three = draft_tree(_ints(_parents(6, 1))), draft_tree(_ints([_parents(6, 1)] * 3))
    path = _ints([[0, 1], [0, 2]])
    for bad in (lambda: cache.attend(q, n, False, 1.0, tree=tree), lambda: cache.attend(q, n, True, 1.0, tree=tree, accumulate=True),
                lambda: cache.attend(q, n, True, 1.0, tree=tree, positions=n), lambda: cache.attend(q[:, :, :5], n, True, 1.0, tree=tree),
                lambda: cache.attend(q, n, True, 1.0, tree=three), lambda: draft_tree(_ints([[]])), lambda: draft_tree(_ints([0] * 513)),
                lambda: DraftTree(tree.bits.expand(1, 6, 1).transpose(0, 1).contiguous().transpose(0, 1)[:, ::2]),
                lambda: DraftTree(tree.bits, tree.depths.long()), lambda: DraftTree(tree.bits, [[0] * 6]), lambda: cache.keep(path.cpu(), n), lambda: cache.keep(path, 41),
                lambda: cache.keep(torch.zeros((2, 513), dtype=torch.int32).cuda(), n)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: cache.attend(q, n, True, 1.0, tree=tree.bits), lambda: draft_tree(_ints(_parents(6, 1)).long()), lambda: draft_tree([-1, 0]),
                lambda: DraftTree(tree.bits.long()), lambda: DraftTree(tree.bits[0]), lambda: DraftTree(torch.zeros((1, 40, 1), dtype=torch.int32).cuda()),
                lambda: cache.keep(path.long(), n), lambda: cache.keep(path[:1], n), lambda: cache.keep(path, n, counts=[1, 1]),
                lambda: cache.keep(path, n.long())):
        with pytest.raises(TypeError):
            bad()
    with pytest.raises(RuntimeError, match="no gradients"):
        cache.attend(q.clone().requires_grad_(), n, True, 1.0, tree=tree)
    want = {x: getattr(cache, x).clone() for x in BUFFERS}
    cache.keep(torch.empty((2, 0), dtype=torch.int32).cuda(), n)
    _same(cache, want)
    assert cache.attend(q[:, :, :0], n, True, 1.0).shape == (2, 4, 0, 64)


def test_a_tree_stays_as_it_was_made():
    cache, q = _filled(2, 2, 90, 64, F16, 1), _randn((2, 4, 70, 64), 2, F16)
    tree = draft_tree(_ints(_parents(70, 1)))
    want = cache.attend(q, 90, True, 0.1, tree=tree)
    for name, x in (("bits", tree.bits[:, :1, :1].clone()), ("depths", None), ("trees", 2), ("tokens", 3)):
        with pytest.raises(AttributeError):
            setattr(tree, name, x)
    assert torch.equal(cache.attend(q, 90, True, 0.1, tree=tree), want)
