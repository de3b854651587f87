"""Cross attention and its gradients on the GPU against the float64 definition; bounds: oracle/cross.py."""
import math

import pytest
import torch

from ascend_rsfa.cross import cross_attention
from oracle import cross as O

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def _randn(shape, seed, dtype, std=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype).cuda()


def _ints(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


def _inputs(Z, Hq, H, T, N, D, dtype, seed=0):
    return _randn((Z, Hq, T, D), seed, dtype), _randn((Z, H, N, D), seed + 1, dtype), _randn((Z, H, N, D), seed + 2, dtype)


def _hold(name, got, want):
    value, bound = want
    assert got.shape == value.shape, name
    same = (got == value) | (torch.isnan(got) & torch.isnan(value))  # infinities, NaN
    off = torch.where(same, torch.full_like(value, -1.0), (got.double() - value).abs() - bound)
    assert (off <= 0).all(), f"{name} off its bound by {off.max().item()} (values up to {value.abs().max().item()})"


def _train(q, k, v, scale, lengths, go, glse=None):
    """{name: tensor} of a forward and backward pass."""
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    o, lse = cross_attention(q, k, v, scale, lengths, return_lse=True)
    if glse is None:
        grads = torch.autograd.grad(o, (q, k, v), go)
    else:
        grads = torch.autograd.grad((o, lse), (q, k, v), (go, glse))
    return dict(zip(("o", "lse", "dq", "dk", "dv"), (o.detach(), lse.detach(), *grads)))


def _check(q, k, v, scale, lengths, go, glse=None):
    listed = None if lengths is None else lengths.tolist()
    got, want = _train(q, k, v, scale, lengths, go, glse), O.expect(q, k, v, listed, scale, go, glse)
    for name, value in want.items():
        _hold(name, got[name], value)
    return got


# (Z, Hq, H, T, N, lengths): one token to many, one state to many, tiles and parts that end inside, shared heads
SHAPES = [
    (1, 1, 1, 1, 1, None), (2, 4, 2, 1, 100, [100, 1]), (2, 4, 2, 3, 1531, [17, 1531]), (1, 8, 1, 5, 4000, None),
    (3, 4, 4, 16, 333, [1, 32, 333]), (2, 2, 2, 17, 31, [31, 30]), (2, 2, 2, 40, 77, [77, 5]), (1, 2, 1, 130, 1000, None),
    (2, 4, 2, 300, 515, [515, 64]), (1, 2, 2, 600, 4100, None), (8, 8, 8, 260, 129, None), (4, 16, 8, 257, 640, [640, 1, 65, 200]),
    (1, 3, 1, 65, 2048, [2047]), (1, 2, 2, 3000, 77, None), (3, 2, 2, 64, 128, [128, 127, 0]), (1, 40, 1, 9, 65, None),
]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("shape", SHAPES)
def test_matches_the_definition(shape, D, dtype):
    Z, Hq, H, T, N, lengths = shape
    q, k, v = _inputs(Z, Hq, H, T, N, D, dtype)
    glse = _randn((Z, Hq, T), 9, torch.float32)
    le = None if lengths is None else _ints(lengths)
    if lengths is not None:
        for z, n in enumerate(lengths):  # what lies behind the lengths reaches nothing
            k[z, :, n:], v[z, :, n:] = math.nan, math.inf
        glse[torch.tensor(lengths) == 0] = 0.0
    got = _check(q, k, v, D ** -0.5, le, _randn(q.shape, 5, dtype), glse)
    # without gradients: the same forward pass
    o, lse = cross_attention(q, k, v, D ** -0.5, le, return_lse=True)
    assert torch.equal(o, got["o"]) and torch.equal(lse, got["lse"])
    assert torch.equal(cross_attention(q, k, v, D ** -0.5, le), o)


# every forward variant, whole and in parts (tests/test_cross_cpu.py holds them to it)
VARIANTS = [
    (46, 16, 2, 1, 1, 32), (1, 2, 1, 2, 4123, 32), (7, 128, 16, 7, 1, 32), (1, 8, 8, 34, 2123, 32), (59, 32, 4, 5, 1, 32),
    (1, 32, 8, 9, 30654, 32), (1, 8, 8, 1, 2, 64), (2, 4, 2, 1, 927, 64), (4, 64, 8, 21, 1, 64), (2, 2, 2, 20, 8794, 64),
    (8, 128, 16, 10, 1, 64), (1, 8, 8, 202, 1757, 64), (1, 2, 2, 1, 1, 128), (1, 2, 2, 1, 1078, 128), (21, 16, 8, 10, 1, 128),
    (1, 64, 8, 9, 1702, 128), (5, 8, 8, 198, 1, 128), (2, 32, 8, 17, 3773, 128), (1, 1, 1, 5, 1, 256), (5, 1, 1, 2, 379, 256),
    (3, 16, 16, 88, 1, 256), (4, 2, 1, 33, 2340, 256), (1, 2, 1, 3, 1, 32), (10, 1, 1, 66, 2529, 32), (2, 1, 1, 3, 111, 32),
    (2, 2, 2, 142, 7000, 32), (17, 2, 1, 305, 1, 64), (7, 8, 4, 103, 4960, 64), (3, 4, 4, 3574, 345, 64), (11, 2, 2, 356, 3985, 64),
    (5, 64, 8, 56, 1, 128), (1, 8, 8, 137, 10984, 128), (5, 32, 16, 140, 1, 128), (5, 8, 1, 231, 2676, 128), (38, 4, 4, 36, 1, 256),
    (4, 4, 2, 65, 2605, 256), (74, 2, 2, 153, 1, 256), (20, 1, 1, 139, 4193, 256),
]


@pytest.mark.parametrize("shape", VARIANTS)
def test_every_forward_variant(shape):
    Z, Hq, H, T, N, D = shape
    for dtype in (F16, BF16):
        q, k, v = _inputs(Z, Hq, H, T, N, D, dtype)
        for lengths in (None, [N - (z * 7919) % (N + 1) for z in range(Z)]):
            le = None if lengths is None else _ints(lengths)
            got = cross_attention(q, k, v, D ** -0.5, le, return_lse=True)
            want = O.expect(q, k, v, lengths, D ** -0.5)
            for name, x in zip(("o", "lse"), got):
                _hold(name, x, want[name])


@pytest.mark.parametrize("T", [1, 3, 40, 300])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
def test_sequences_without_keys_and_lengths_outside(D, T):
    q, k, v = _inputs(4, 4, 2, T, 200, D, BF16)
    go, glse = _randn(q.shape, 4, BF16), _randn(q.shape[:3], 5, torch.float32)
    got = _train(q, k, v, 0.1, _ints([-7, 10 ** 9, 0, 64]), go, glse)
    want = _train(q, k, v, 0.1, _ints([0, 200, 0, 64]), go, glse)
    for name in got:
        assert torch.equal(got[name], want[name]), name
    for z in (0, 2):
        assert (got["o"][z] == 0).all() and (got["lse"][z] == -math.inf).all()
        assert all((got[n][z] == 0).all() for n in ("dq", "dk", "dv"))
    assert (got["dk"][3, :, 64:] == 0).all() and (got["dv"][3, :, 64:] == 0).all()


@pytest.mark.parametrize("T", [2, 100])
def test_gradients_against_differences(T):
    # the derivative along a direction, of the definition's sum of o go + lse glse in float64
    q, k, v = _inputs(2, 4, 2, T, 90, 64, BF16)
    lengths = [90, 41]
    go, glse = _randn(q.shape, 4, BF16), _randn(q.shape[:3], 5, torch.float32)
    got = _train(q, k, v, 0.125, _ints(lengths), go, glse)
    bounds = O.expect(q, k, v, lengths, 0.125, go, glse)

    def value(x):
        o, lse = O.attend(*x, lengths, 0.125)
        return float((o * go.double()).sum() + (lse * glse.double()).sum())

    for i, name in enumerate(("dq", "dk", "dv")):
        at = [t.double() for t in (q, k, v)]
        way = torch.randn(at[i].shape, generator=torch.Generator().manual_seed(i), dtype=torch.float64).cuda()
        base, step = at[i], 2.0 ** -12
        at[i] = base + step * way
        up = value(at)
        at[i] = base - step * way
        slope = (up - value(at)) / (2 * step)
        mine = float((got[name].double() * way).sum())
        # a central difference is off by the third derivative (of these sums below 2^10) times step^2 / 6
        assert abs(mine - slope) <= float((bounds[name][1] * way.abs()).sum()) + 2.0 ** 10 * step ** 2, name


@pytest.mark.parametrize("scale", [0.0, -0.3, 1.7, 1e-38, -1e-6])
@pytest.mark.parametrize("T", [3, 70])
def test_scales(scale, T):
    for dtype in (F16, BF16):
        q, k, v = _inputs(2, 2, 1, T, 150, 64, dtype)
        _check(q, k, v, scale, _ints([150, 33]), _randn(q.shape, 4, dtype), _randn(q.shape[:3], 5, torch.float32))


@pytest.mark.parametrize("std", [2.0 ** -20, 2.0 ** -12, 1.0, 2.0 ** 9])
@pytest.mark.parametrize("T, D", [(3, 64), (90, 32), (200, 128), (70, 256)])
def test_gradients_of_every_size(T, D, std):
    # (rows of q and k large enough for gradients within float16's normal numbers, and a row of dO far above the others)
    for dtype in (F16, BF16):
        q, k, v = _inputs(2, 4, 2, T, 333, D, dtype)
        go = _randn(q.shape, 4, dtype, std)
        go[1, 3, T // 2] *= 64
        up = 2.0 ** 7 if std < 1 else 1.0
        _check(q * up, k * up, v, D ** -0.5 / up ** 2, _ints([333, 200]), go)
        _check(q, k, v, D ** -0.5, None, go, _randn(q.shape[:3], 5, torch.float32, std))


@pytest.mark.parametrize("std", [2.0 ** 4, 2.0 ** 7, 2.0 ** 9])
@pytest.mark.parametrize("T, D", [(3, 64), (90, 32), (200, 128), (70, 256)])
def test_gradients_over_large_states(T, D, std):
    for dtype in (F16, BF16):
        q, k, v = _inputs(2, 4, 2, T, 200, D, dtype)
        for scale in (D ** -0.5, 1.0):  # (weights spread, and on few keys)
            _check(q, k, (v * std).to(dtype), scale, _ints([200, 7]), _randn(q.shape, 4, dtype, 2.0 ** -10))


@pytest.mark.parametrize("T", [2, 90])
def test_one_score_far_above_the_rest(T):
    # each row's weight on one key, anywhere along a long row, and rows of equal scores
    N = 5000
    q, k, v = _inputs(1, 2, 2, T, N, 64, BF16)
    k.mul_(0.01)
    for i in range(T):
        k[:, :, (i * 977 + 13) % N] = q[:, :, i]
    _check(q, k, v, 2.0, None, _randn(q.shape, 4, BF16))
    q.zero_()
    _check(q, k, v, 1.0, None, _randn(q.shape, 4, BF16))


@pytest.mark.parametrize("T", [1, 50, 200])
def test_non_finite_values_of_visible_keys(T):
    q, k, v = _inputs(2, 2, 2, T, 96, 64, F16)
    v[0, 0, 5, 3], v[0, 1, 7] = math.inf, math.nan
    k[1, 0, 9] = math.nan
    o = cross_attention(q, k, v, 0.125)
    want, _ = O.attend(q, k, v, None, 0.125)
    assert torch.equal(torch.isnan(o), torch.isnan(want)) and torch.equal(torch.isinf(o), torch.isinf(want))


@pytest.mark.parametrize("N", [33, 97, 1001])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("T", [1, 50, 1500])
def test_infinite_values_of_the_last_key(T, D, N):
    # (what fills its tile up has no part in the sums)
    q, k, v = _inputs(2, 4, 2, T, N, D, BF16)
    n = _ints([N, N - 9])
    v[0, 0, N - 1], v[1, 1, N - 10, 5] = math.inf, -math.inf
    o = cross_attention(q, k, v, 0.01, n)
    want, _ = O.attend(q, k, v, n, 0.01)
    assert torch.equal(torch.isnan(o), torch.isnan(want)) and torch.equal(torch.isinf(o), torch.isinf(want))


@pytest.mark.parametrize("N", [40, 700])
@pytest.mark.parametrize("T", [2, 150])
def test_rows_whose_scores_are_all_minus_infinity_are_nan(T, N):
    q, k, v = _inputs(2, 2, 1, T, N, 64, BF16)
    k[..., 0] = 1.0 + k[..., 0].abs()
    want = cross_attention(q, k, v, 0.125)
    q[1, 0, T - 1, 0] = -math.inf
    o = cross_attention(q, k, v, 0.125)
    assert torch.isnan(o[1, 0, T - 1]).all()
    o[1, 0, T - 1] = want[1, 0, T - 1]
    assert torch.equal(o, want)


def _strided(t, kind):
    Z, H, N, D = t.shape
    if kind == "bshd":
        return t.transpose(1, 2).contiguous().transpose(1, 2)
    if kind == "wide":  # part of a fused projection
        big = torch.zeros((Z, N, H, 2 * D + 8), dtype=t.dtype).cuda()
        big[..., 8:D + 8] = t.transpose(1, 2)
        return big[..., 8:D + 8].transpose(1, 2)
    if kind == "odd":  # rows that are not aligned: copied
        big = torch.zeros((Z, H, N, D + 1), dtype=t.dtype).cuda()
        big[..., 1:] = t
        return big[..., 1:]
    return t.transpose(2, 3).contiguous().transpose(2, 3)  # "columns"


@pytest.mark.parametrize("T", [2, 90])
@pytest.mark.parametrize("kind", ["bshd", "wide", "odd", "columns"])
def test_strides(kind, T):
    q, k, v = _inputs(2, 4, 2, T, 150, 64, BF16)
    go, n = _randn(q.shape, 4, BF16), _ints([150, 77])
    want = _train(q, k, v, 0.125, n, go)
    got = _train(*(_strided(t, kind) for t in (q, k, v)), 0.125, n, _strided(go, kind))
    for name in want:
        assert torch.equal(got[name], want[name]), name


@pytest.mark.parametrize("T", [1, 70])
def test_broadcast_inputs(T):
    # one sequence's states for all (beams), one head's for all; the gradient of a sum
    q, k, v = _inputs(4, 4, 4, T, 90, 64, BF16)
    k, v = k[:1, :1].clone().requires_grad_(), v[:1].clone().requires_grad_()
    q = q[:, :, :1].clone().requires_grad_()
    wide = (q.expand(4, 4, T, 64), k.expand(4, 4, 90, 64), v.expand(4, 4, 90, 64))
    o = cross_attention(*wide, 0.125)
    grads = torch.autograd.grad(o.sum(), (q, k, v))
    dense = [t.detach().clone() for t in wide]
    got = _check(*dense, 0.125, None, torch.ones_like(dense[0]))
    assert torch.equal(o, got["o"])
    for g, t, name in zip(grads, (q, k, v), ("dq", "dk", "dv")):
        assert torch.equal(g, got[name].sum_to_size(t.shape)), name


def test_single_gradients_equal_those_together():
    q, k, v = _inputs(2, 4, 2, 100, 300, 128, F16)
    go = _randn(q.shape, 4, F16)
    want = _train(q, k, v, 0.1, None, go)
    for names in (("q",), ("k",), ("v",), ("q", "v"), ("k", "v")):
        t = {n: x.detach().clone().requires_grad_(n in names) for n, x in zip("qkv", (q, k, v))}
        o = cross_attention(t["q"], t["k"], t["v"], 0.1)
        for n, g in zip(names, torch.autograd.grad(o, [t[n] for n in names], go)):
            assert torch.equal(g, want["d" + n]), names
    # lse alone
    q.requires_grad_(), k.requires_grad_()
    _, lse = cross_attention(q, k, v, 0.1, return_lse=True)
    glse = _randn(q.shape[:3], 6, torch.float32)
    want = O.expect(q, k, v, None, 0.1, torch.zeros_like(go), glse)
    for n, g in zip(("dq", "dk"), torch.autograd.grad(lse, (q, k), glse)):
        _hold(n, g, want[n])


def test_rows_past_two_to_the_31_elements():
    # 300 keys 8 Mi elements apart
    step = 1 << 23
    big = torch.zeros(300 * step + 128, dtype=BF16, device="cuda")
    q, k, v = _inputs(1, 2, 2, 100, 300, 64, BF16)
    kb = big.as_strided((1, 2, 300, 64), (0, 64, step, 1))
    vb = torch.zeros_like(big).as_strided((1, 2, 300, 64), (0, 64, step, 1))
    kb.copy_(k), vb.copy_(v)
    go = _randn(q.shape, 4, BF16)
    want = _train(q, k, v, 0.125, None, go)
    o = cross_attention(q, kb, vb, 0.125)
    assert torch.equal(o, want["o"])
    assert torch.equal(cross_attention(q[:, :, :1], kb, vb, 0.125), cross_attention(q[:, :, :1], k, v, 0.125))
    q.requires_grad_()
    assert torch.equal(torch.autograd.grad(cross_attention(q, kb, vb, 0.125), q, go)[0], want["dq"])


def test_results_do_not_change_from_call_to_call():
    q, k, v = _inputs(4, 8, 2, 500, 700, 64, BF16)
    n, go = _ints([700, 3, 650, 64]), _randn(q.shape, 4, BF16)
    want = _train(q, k, v, 0.125, n, go)
    for _ in range(5):
        got = _train(q, k, v, 0.125, n, go)
        assert all(torch.equal(got[x], want[x]) for x in want)


def test_two_streams_at_once():
    sets = [_inputs(2, 8, 2, T, 3000, 64, F16, seed=T) for T in (1, 200)]
    gos = [_randn(s[0].shape, 3, F16) for s in sets]
    want = [_train(*s, 0.125, None, g) for s, g in zip(sets, gos)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(_train(*sets[i], 0.125, None, gos[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            assert all(torch.equal(g[x], want[i][x]) for x in g)


@pytest.mark.parametrize("T", [1, 300])
def test_forward_in_a_graph_with_lengths_that_change(T):
    q, k, v = _inputs(3, 4, 2, T, 2000, 64, BF16)
    n = _ints([5, 2000, 77])
    cross_attention(q, k, v, 0.125, n)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, lse = cross_attention(q, k, v, 0.125, n, return_lse=True)
    for i in range(4):
        n.copy_(_ints([2000 - 300 * i, i, 64 * i + 1]))
        q.mul_(1.05)
        graph.replay()
        wo, wl = cross_attention(q, k, v, 0.125, n, return_lse=True)
        torch.cuda.synchronize()
        assert torch.equal(o, wo) and torch.equal(lse, wl)


def test_a_training_step_in_a_graph():
    # under torch's conditions: tried on a side stream first, no eager graph of the same leaves alive
    q, k, v = (t.requires_grad_() for t in _inputs(2, 4, 2, 200, 333, 64, BF16))
    n, go = _ints([333, 100]), _randn(q.shape, 4, BF16)

    def step():
        return torch.autograd.grad(cross_attention(q, k, v, 0.125, n), (q, k, v), go)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grads = step()
    for i in range(4):
        with torch.no_grad():
            k.mul_(1.03)
            n.copy_(_ints([333 - 50 * i, 7 * i]))
        graph.replay()
        torch.cuda.synchronize()
        got = [g.clone() for g in grads]
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_refusals():
    q, k, v = _inputs(2, 4, 2, 5, 9, 64, F16)
    n = _ints([9, 4])
    for bad in (lambda: cross_attention(q[0], k, v, 1.0), lambda: cross_attention(q, k, v[:, :, :8], 1.0), lambda: cross_attention(q[:1], k, v, 1.0),
                lambda: cross_attention(q[:, :3], k, v, 1.0), lambda: cross_attention(q[..., :32], k, v, 1.0), lambda: cross_attention(q, k[:, :0], v[:, :0], 1.0),
                lambda: cross_attention(q[..., :16], k[..., :16], v[..., :16], 1.0), lambda: cross_attention(q.cpu(), k, v, 1.0),
                lambda: cross_attention(q.cpu(), k.cpu(), v.cpu(), 1.0), lambda: cross_attention(q, k, v, math.nan),
                lambda: cross_attention(q, k, v, 1.0, n.cpu())):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: cross_attention(q, k.bfloat16(), v, 1.0), lambda: cross_attention(q.float(), k.float(), v.float(), 1.0),
                lambda: cross_attention(q, k, v, 1.0, [9, 4]), lambda: cross_attention(q, k, v, 1.0, n.long()), lambda: cross_attention(q, k, v, 1.0, n[:1])):
        with pytest.raises(TypeError):
            bad()
    x = q.clone().requires_grad_()
    g, = torch.autograd.grad(cross_attention(x, k, v, 1.0).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    with torch.autograd.forward_ad.dual_level(), pytest.raises(RuntimeError):
        cross_attention(torch.autograd.forward_ad.make_dual(q, torch.ones_like(q)), k, v, 1.0)
    # lengths that change between the passes are noticed
    o = cross_attention(x, k, v, 1.0, n)
    n.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.sum().backward()


def test_empty_calls():
    q, k, v = _inputs(2, 4, 2, 5, 9, 64, F16)
    o, lse = cross_attention(q[:, :, :0], k, v, 1.0, return_lse=True)
    assert o.shape == (2, 4, 0, 64) and lse.shape == (2, 4, 0)
    assert cross_attention(q[:0], k[:0], v[:0], 1.0, _ints([1])[:0]).shape == (0, 4, 5, 64)
    none = k[:, :, :0].clone().requires_grad_()
    x = q.clone().requires_grad_()
    o, lse = cross_attention(x, none, none, 1.0, return_lse=True)
    assert (o == 0).all() and (lse == -math.inf).all()
    gq, gk = torch.autograd.grad(o.sum(), (x, none))
    assert (gq == 0).all() and gk.shape == none.shape
    x = k.clone().requires_grad_()
    g, = torch.autograd.grad(cross_attention(q[:, :, :0], x, v, 1.0).sum(), x)
    assert (g == 0).all()


@pytest.mark.parametrize("pin", [False, True])
@pytest.mark.parametrize("order", ["kept first", "hook first"])
@pytest.mark.parametrize("kind", ["bshd", "wide"])
def test_saved_tensors_kept_on_the_host(kind, order, pin):
    # a hook may bring saved tensors back in another layout; sizes of this test's own, so that nothing of them is kept before
    T, N = 61 + 2 * pin, 131 + (order == "hook first") + 2 * (kind == "wide")
    plain = _inputs(2, 4, 2, T, N, 64, BF16)
    go, glse, n = _randn(plain[0].shape, 4, BF16), _randn(plain[0].shape[:3], 5, torch.float32), _ints([N, 77])
    q, k, v = (_strided(t, kind).requires_grad_() for t in plain)

    def step(hook):
        if not hook:
            return torch.autograd.grad(cross_attention(q, k, v, 0.125, n, return_lse=True), (q, k, v), (go, glse))
        with torch.autograd.graph.save_on_cpu(pin_memory=pin):
            o = cross_attention(q, k, v, 0.125, n, return_lse=True)
        return torch.autograd.grad(o, (q, k, v), (go, glse))

    want = None
    for hook in (False, True, False, True) if order == "kept first" else (True, False, True, False):
        got = step(hook)
        if want is None:
            bounds = O.expect(*plain, n.tolist(), 0.125, go, glse)
            for name, g in zip(("dq", "dk", "dv"), got):
                _hold(name, g, bounds[name])
            want = got
        assert all(torch.equal(a, b) for a, b in zip(got, want)), (order, hook)


@pytest.mark.parametrize("signs", ["alike", "random"])
@pytest.mark.parametrize("states", [1.0, 64.0, 300.0, 1024.0])
@pytest.mark.parametrize("grads", [2.0 ** -10, 1.0, 64.0, 512.0])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
def test_float16_gradients_whose_sums_pass_the_type(D, grads, states, signs):
    # dO v, of all signs alike D grads states, lies above 2^16, the gradients themselves do not
    for T, N, lengths in ((3, 2, None), (3, 200, [200, 150]), (70, 64, None), (90, 333, [333, 30]), (5, 1500, None)):
        q, k, v = _inputs(2, 2, 2, T, N, D, F16, seed=T)
        go = _randn(q.shape, 4, F16)
        if signs == "alike":
            v = torch.sign(v[..., :1]).expand_as(v).contiguous()
            go = torch.ones_like(go)
        v, go = v * states, go * grads
        # (dq is at most the scale times |ds| times a few keys' values, dk that times the rows')
        scale = min(D ** -0.5, 2.0 ** 12 / (grads * states * (D if signs == "alike" else 8 * D ** 0.5) * max(1.0, T / N)))
        le = None if lengths is None else _ints(lengths)
        glse = _randn(q.shape[:3], 5, torch.float32, grads)
        want = O.expect(q, k, v, lengths, scale, go, glse)
        assert all(x.abs().max() < 2.0 ** 15.9 for x, _ in want.values())
        got = _train(q, k, v, scale, le, go, glse)
        for name, value in want.items():
            _hold(name, got[name], value)


@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("T, N", [(3, 200), (90, 700), (2, 9000)])
def test_float16_gradients_of_keys_far_above_the_first(T, N, D):
    # the first keys' values, which the scale of dS goes by, are small or 0, some later ones' large; of the last rows' dO too
    for small in (0.0, 2.0 ** -12):
        for at in (33, N - 1):
            q, k, v = _inputs(2, 2, 1, T, N, D, F16)
            v *= small
            v[:, :, at], v[0, 0, at - 1] = 512.0, -512.0
            go = torch.ones_like(q)
            go[1, 1, T - 1] = 8.0
            _check(q, k, v, 2.0 ** -7, _ints([N, at + 1]), go)
            # (equal weights of opposite values: delta is 0 and tells nothing of them; every second row like that)
            v[:, :, at - 1] = -512.0
            q[:, :, ::2] = 0.0
            _check(q, k, v, 2.0 ** -7, _ints([N, at + 1]), go)


def test_float16_rows_beside_one_that_is_not_finite():
    # gradients of v and of q that a row's infinite dO does not reach are what they were
    q, k, v = _inputs(2, 2, 2, 90, 150, 64, F16)
    go = _randn(q.shape, 4, F16)
    want = _train(q, k, v, 0.125, None, go)
    go[1, 0, 40, 7] = math.inf
    got = _train(q, k, v, 0.125, None, go)
    assert torch.isnan(got["dq"][1, 0, 40]).all() and torch.isinf(got["dv"][1, 0, :, 7]).all()
    for x, name in ((got["dq"], "dq"), (got["dv"], "dv")):
        x[1, 0, 40 if name == "dq" else slice(None), slice(None) if name == "dq" else 7] = want[name][1, 0, 40 if name == "dq" else slice(None), slice(None) if name == "dq" else 7]
        assert torch.allclose(x.double(), want[name].double(), rtol=2.0 ** -9, atol=2.0 ** -14)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("T", [1, 31, 33, 90, 700])
def test_an_infinite_gradient_of_the_last_row(T, D, dtype):
    # (what fills its tile up has no part in the sums: dv is infinite where the row's dO is, not NaN)
    q, k, v = _inputs(2, 4, 2, T, 200, D, dtype)
    n, go = _ints([200, 77]), _randn(q.shape, 4, dtype)
    want = O.expect(q, k, v, [200, 77], 0.01, go)["dv"]
    go[0, 1, T - 1, 3], go[1, 2, T - 1, D - 1] = math.inf, -math.inf
    got = _train(q, k, v, 0.01, n, go)["dv"]
    assert (got[0, 0, :, 3] == math.inf).all() and (got[1, 1, :77, D - 1] == -math.inf).all()
    got[0, 0, :, 3], got[1, 1, :77, D - 1] = want[0][0, 0, :, 3], want[0][1, 1, :77, D - 1]
    _hold("dv", got, want)


@pytest.mark.parametrize("hidden", [1, 130, 600])
@pytest.mark.parametrize("shape", [(2, 4, 2, T, 700) for T in (1, 6, 50, 300)] + [(1, 8, 8, 137, 10984), (2, 32, 8, 17, 3773), (1, 2, 1, 1, 9000)])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
def test_keys_whose_scores_are_minus_infinity(D, shape, hidden):
    # the first keys, tiles and whole parts of them; then every second tile of 128: as if the others were all
    Z, Hq, H, T, N = shape
    hidden = hidden * N // 700
    q, k, v = _inputs(Z, Hq, H, T, N, D, BF16)
    q[..., 0] = 1.0 + q[..., 0].abs()
    n = [N - 5 * z for z in range(Z)]
    for gone in (torch.arange(N) < hidden, torch.arange(N) // 128 % 2 == (0 if hidden > 1 else 1)):
        x = k.clone()
        x[:, :, gone.cuda(), 0] = -math.inf
        got = cross_attention(q, x, v, D ** -0.5, _ints(n), return_lse=True)
        at = (~gone).cuda()
        want = O.expect(q, k[:, :, at], v[:, :, at], [int((~gone)[:m].sum()) for m in n], D ** -0.5)
        for name, y in zip(("o", "lse"), got):
            _hold(name, y, want[name])


@pytest.mark.parametrize("T", [3, 70])
def test_small_scales_of_large_values(T):
    # scores of the usual size, of q and k 2^52 times as large: the same bits, but for the gradients' exponents
    q, k, v = _inputs(2, 4, 2, T, 150, 64, BF16)
    go, glse, n = _randn(q.shape, 4, BF16), _randn(q.shape[:3], 5, torch.float32), _ints([150, 33])
    want = _train(q, k, v, 0.125, n, go, glse)
    got = _train(q * 2.0 ** 52, k * 2.0 ** 52, v, 2.0 ** -107, n, go, glse)
    for name in want:
        up = 2.0 ** 52 if name in ("dq", "dk") else 1.0
        assert torch.equal(got[name].double() * up, want[name].double()), name
