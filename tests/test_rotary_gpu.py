"""rotary on the GPU against the float64 definition, its gradients, layouts and refusals.

Tolerance of a value: half a step of its type, and in 32 bits the angle's
fraction (2^-26 of a turn: 1.6 * 2^-24), sine and cosine (2 units: 2 * 2^-24),
the amplitude, two products and their sum (half a unit, 2^-24, each, on values of at
most amplitude * (|u| + |w|)): 8 * 2^-24 * amplitude * (|u| + |w|) in all; and
the 64-bit products of position and frequency, here and in the definition: 4 * 2^-53 * |angle|.
"""
import math

import pytest
import torch
from torch.autograd import forward_ad

from ascend_rsfa import rotary as R
from oracle import serving as S

pytestmark = pytest.mark.gpu


def _plan(dim, layout, scaling=None):
    kw = {None: {}, "linear": {"factor": 4.0}, "ntk": {"factor": 8.0},
          "by_parts": {"factor": 16.0, "original_length": 4096, "base": 500000.0, "amplitude": 1.2772}}[scaling]
    return R.rotary_plan(dim, layout=layout, scaling=scaling, **kw)


def _tolerance(x, want, positions, plan, layout):
    dim = plan.rotary_dim
    a = x.detach().double().abs()
    i = torch.arange(dim // 2, device=x.device)
    lo, hi = (i, i + dim // 2) if layout == "half" else (2 * i, 2 * i + 1)
    both = a[..., lo] + a[..., hi]
    pos = positions if positions.dim() == 2 else positions[None]
    angle = pos[:, None, :, None].double().abs() * plan.frequencies.to(x.device)
    err = abs(plan.amplitude) * both * (8 * 2.0 ** -24 + 4 * 2.0 ** -53 * angle)
    tol = want.abs() * torch.finfo(x.dtype).eps / 2 + 2.0 ** -25 * (x.dtype == torch.float16)
    tol[..., lo] += err * (1 + torch.finfo(x.dtype).eps)
    tol[..., hi] += err * (1 + torch.finfo(x.dtype).eps)
    return tol


def _inputs(Z, Hq, Hk, N, D, dtype, order, seed):
    g = torch.Generator().manual_seed(seed)

    def one(H):
        if order == "bshd":
            return torch.randn((Z, N, H, D), generator=g).to(dtype).cuda().transpose(1, 2)
        if order == "slice":  # part of a fused projection, odd strides
            return torch.randn((Z, H, N, D + 5), generator=g).to(dtype).cuda()[..., 2:D + 2]
        return torch.randn((Z, H, N, D), generator=g).to(dtype).cuda()

    return one(Hq), one(Hk)


def _check(got, x, positions, plan, inverse=False):
    want = S.rotary(x, positions, plan.frequencies, plan.amplitude, plan.layout, inverse)
    off = (got.double() - want).abs() - _tolerance(x, want, positions, plan, plan.layout)
    assert got.dtype == x.dtype and (off <= 0).all(), off.max().item()
    assert torch.equal(got[..., plan.rotary_dim:], x.detach()[..., plan.rotary_dim:])


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [
    # Z, Hq, Hk, N, D, rotary_dim
    (1, 1, 1, 1, 16, 16), (2, 4, 2, 33, 64, 64), (3, 5, 1, 7, 128, 64), (1, 3, 3, 1000, 128, 128),
    (2, 2, 1, 17, 256, 250), (2, 2, 2, 5, 80, 26), (1, 2, 1, 3, 7, 6), (4, 40, 3, 1, 128, 32),
])
def test_matches_the_definition(shape, dtype, layout):
    Z, Hq, Hk, N, D, dim = shape
    for n, (order, scaling) in enumerate([("bhsd", None), ("bshd", "linear"), ("slice", "ntk"), ("bshd", "by_parts")]):
        print(f"rotary {shape} {dtype} {layout} {order} {scaling}", flush=True)
        q, k = _inputs(Z, Hq, Hk, N, D, dtype, order, seed=n)
        plan = _plan(dim, layout, scaling)
        positions = torch.randint(0, 100000, (Z, N), generator=torch.Generator().manual_seed(n)).cuda()
        yq, yk = R.rotary(q, k, positions, plan)
        _check(yq, q, positions, plan)
        _check(yk, k, positions, plan)


@pytest.mark.parametrize("positions", [
    0, 12345, -7, 2 ** 31 + 5,
    torch.arange(19, dtype=torch.int32), torch.arange(19).flip(0) * 3 + 2 ** 40,
    torch.arange(38, dtype=torch.int32).reshape(2, 19) - 20, torch.arange(76).reshape(2, 38)[:, ::2],
    torch.arange(19)[None],
])
def test_positions(positions):
    q, k = _inputs(2, 3, 2, 19, 64, torch.float32, "bhsd", 5)
    plan = _plan(64, "half")
    t = positions
    if isinstance(positions, int):
        p = positions + torch.arange(19).cuda()
    else:
        t = positions.cuda()
        p = t
    yq, yk = R.rotary(q, k, t, plan)
    _check(yq, q, p, plan)
    _check(yk, k, p, plan)
    assert torch.equal(R.rotary(q, None, t, plan), yq)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gradients(layout, dtype):
    q, k = _inputs(2, 4, 2, 33, 64, dtype, "bshd", 9)
    plan = _plan(48, layout, "by_parts")
    positions = torch.randint(0, 5000, (2, 33)).cuda()
    g = torch.Generator().manual_seed(1)
    gq = torch.randn(q.shape, generator=g).to(dtype).cuda()
    gk = torch.randn(k.shape, generator=g).to(dtype).cuda()
    q.requires_grad_(), k.requires_grad_()
    yq, yk = R.rotary(q, k, positions, plan)
    dq, dk = torch.autograd.grad((yq, yk), (q, k), (gq, gk))
    _check(dq, gq, positions, plan, inverse=True)
    _check(dk, gk, positions, plan, inverse=True)
    # one tensor alone, an output that no gradient reaches, an expanded gradient
    yq, yk = R.rotary(q, k.detach(), positions, plan)
    _check(torch.autograd.grad(yq, q, gq)[0], gq, positions, plan, inverse=True)
    yq, yk = R.rotary(q, k, positions, plan)
    dk, = torch.autograd.grad(yk.sum(), k)
    _check(dk, torch.ones_like(k), positions, plan, inverse=True)
    # positions changed after the forward call are caught by autograd
    yq, yk = R.rotary(q, k, positions, plan)
    positions.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(yq, q, gq)


def test_gradients_of_gradients():
    # linear: the gradient of <d, grad> in the output gradient is the forward turn of d
    q = _inputs(1, 2, 1, 5, 64, torch.float32, "bhsd", 3)[0].requires_grad_()
    plan = _plan(64, "half")
    g, d = (torch.randn_like(q).requires_grad_() for _ in range(2))
    dq, = torch.autograd.grad(R.rotary(q, None, 9, plan), q, g, create_graph=True)
    dg, = torch.autograd.grad(dq, g, d)
    _check(dg, d, torch.arange(9, 14).cuda(), plan)


def test_tangents():
    q, k = _inputs(2, 3, 2, 9, 64, torch.float32, "bshd", 3)
    tq, tk = _inputs(2, 3, 2, 9, 64, torch.float32, "bhsd", 4)
    plan = _plan(48, "half", "ntk")
    positions = torch.arange(9).cuda() * 1000
    for inverse, turn in ((False, lambda a, b: R.rotary(a, b, positions, plan)), (True, lambda a, b: R._turn(a, b, positions, plan, True))):
        with forward_ad.dual_level():
            got = [forward_ad.unpack_dual(y) for y in turn(forward_ad.make_dual(q, tq), forward_ad.make_dual(k, tk))]
            for y, x, t in zip(got, (q, k), (tq, tk)):
                _check(y.primal, x, positions, plan, inverse)
                _check(y.tangent, t, positions, plan, inverse)
            with pytest.raises(RuntimeError, match="in place"):
                R.rotary_(forward_ad.make_dual(q, tq), None, 0, plan)


def test_gradient_against_differences():
    # float32, directional: (f(x + h d) - f(x - h d)) / 2h of f = <g, rotary(x)>; f is linear, so h may be
    # large: the difference's error is that of the two sums, 2 * 24 * 2^-24 * sum |g||y| / 2h, at h = 8
    g = torch.Generator().manual_seed(2)
    x, d, w = (torch.randn((1, 2, 5, 16), generator=g).cuda() for _ in range(3))
    plan = _plan(8, "interleaved", "ntk")

    def f(t):
        return (w.double() * R.rotary(t, None, 3, plan).double()).sum()

    x.requires_grad_()
    dx, = torch.autograd.grad(R.rotary(x, None, 3, plan), x, w)
    with torch.no_grad():
        difference = (f(x + 8 * d) - f(x - 8 * d)) / 16
        size = (w.double().abs() * (x.double().abs() + 8 * d.double().abs()) * 2).sum() / 8
    assert abs((dx.double() * d.double()).sum() - difference) <= size * 24 * 2.0 ** -24


def test_in_place_touches_the_rotated_values_only():
    for order in ("bhsd", "bshd", "slice"):
        q, k = _inputs(2, 4, 2, 9, 128, torch.float16, order, 3)
        plan = _plan(64, "half")
        yq, yk = R.rotary(q, k, 11, plan)
        rq, rk = R.rotary_(q, k, 11, plan)
        assert rq is q and rk is k and torch.equal(q, yq) and torch.equal(k, yk)


def test_q_and_k_slices_of_one_projection_in_place():
    qkv = torch.randn((2, 9, 8, 64)).cuda().half()
    q, k = qkv[:, :, :4].transpose(1, 2), qkv[:, :, 4:6].transpose(1, 2)
    v = qkv[:, :, 6:].clone()
    plan = _plan(64, "interleaved")
    yq, yk = R.rotary(q, k, 0, plan)
    R.rotary_(q, k, 0, plan)
    assert torch.equal(q, yq) and torch.equal(k, yk) and torch.equal(qkv[:, :, 6:], v)


def test_expanded_and_unaligned_inputs():
    plan = _plan(64, "half")
    x = torch.randn((1, 1, 9, 64)).cuda().half().expand(2, 3, 9, 64)
    _check(R.rotary(x, None, 5, plan), x, torch.arange(5, 14).cuda(), plan)
    flat = torch.randn(2 * 3 * 9 * 64 + 1).cuda().half()[1:].reshape(2, 3, 9, 64)  # 2-byte aligned
    _check(R.rotary(flat, None, 5, plan), flat, torch.arange(5, 14).cuda(), plan)
    t = torch.randn((2, 3, 64, 9)).cuda().half().transpose(2, 3)  # head dim not unit-stride
    _check(R.rotary(t, None, 5, plan), t, torch.arange(5, 14).cuda(), plan)


def test_non_finite_values_stay_in_their_pairs():
    plan = _plan(32, "half")
    x = torch.randn((1, 1, 4, 64)).cuda()
    x[0, 0, 1, 3] = math.nan
    x[0, 0, 2, 40] = math.inf
    y = R.rotary(x, None, 7, plan)
    bad = ~torch.isfinite(y)
    assert bad.nonzero().tolist() == [[0, 0, 1, 3], [0, 0, 1, 19], [0, 0, 2, 40]]


def test_empty_tensors():
    plan = _plan(32, "half")
    q, k = torch.empty((2, 3, 0, 64)).cuda(), torch.empty((2, 1, 0, 64)).cuda()
    yq, yk = R.rotary(q, k, 0, plan)
    assert yq.shape == q.shape and yk.shape == k.shape
    assert R.rotary(torch.empty((0, 3, 5, 64)).cuda(), None, 0, plan).shape == (0, 3, 5, 64)


def test_on_a_side_stream_and_in_a_graph():
    q, k = _inputs(2, 4, 2, 33, 128, torch.bfloat16, "bhsd", 4)
    plan = _plan(128, "half", "by_parts")
    positions = torch.arange(33).cuda()
    want = R.rotary(q, k, positions, plan)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = R.rotary(q, k, positions, plan)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = R.rotary(q, k, positions, plan)
    for step in (0, 5, 100000):
        positions.copy_(torch.arange(33).cuda() + step)
        q.copy_(q.flip(0))
        graph.replay()
        torch.cuda.synchronize()
        eager = R.rotary(q, k, positions, plan)
        assert all(torch.equal(a, b) for a, b in zip(out, eager)), step


def test_backward_in_a_graph():
    # as torch asks of a captured backward pass: tried on a side stream first, no eager graph of the leaves alive
    q, k = _inputs(2, 4, 2, 33, 64, torch.bfloat16, "bshd", 4)
    gq, gk = _inputs(2, 4, 2, 33, 64, torch.bfloat16, "bhsd", 5)
    plan = _plan(48, "half", "linear")
    positions = torch.arange(33).cuda()
    q.requires_grad_(), k.requires_grad_()

    def step():
        return torch.autograd.grad(R.rotary(q, k, positions, plan), (q, k), (gq, gk))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        dq, dk = step()
    for start in (0, 7, 90000):
        with torch.no_grad():
            positions.copy_(torch.arange(33).cuda() + start)
            gq.copy_(gq.flip(0))
            gk.copy_(gk.flip(0))
        graph.replay()
        torch.cuda.synchronize()
        _check(dq, gq, positions, plan, inverse=True)
        _check(dk, gk, positions, plan, inverse=True)


def test_refusals():
    plan = _plan(64, "half")
    x = torch.zeros((1, 2, 3, 64)).cuda().half()
    with pytest.raises(TypeError):
        R.rotary(x.double(), None, 0, plan)
    with pytest.raises(TypeError):
        R.rotary(x, x.float(), 0, plan)
    with pytest.raises(ValueError):
        R.rotary(x[0], None, 0, plan)
    with pytest.raises(ValueError):
        R.rotary(x, x[:, :, :2], 0, plan)
    with pytest.raises(ValueError):
        R.rotary(x[..., :32], None, 0, plan)
    with pytest.raises(TypeError):
        R.rotary(x, None, 1.5, plan)
    with pytest.raises(TypeError):
        R.rotary(x, None, torch.zeros(3).cuda(), plan)
    with pytest.raises(ValueError):
        R.rotary(x, None, torch.zeros(4, dtype=torch.int32).cuda(), plan)
    with pytest.raises(ValueError):
        R.rotary(x, None, torch.zeros(3, dtype=torch.int32), plan)
    with pytest.raises(TypeError):
        R.rotary(x, None, 0, None)
    with pytest.raises(ValueError):
        R.rotary_(x.expand(2, 2, 3, 64), None, 0, plan)
    with pytest.raises(ValueError):
        R.rotary_(x, x, 0, plan)
    with pytest.raises(ValueError):
        R.rotary(x, None, 1 << 53, plan)
    with pytest.raises(RuntimeError):
        R.rotary_(x.clone().requires_grad_(), None, 0, plan)
