"""What the serving operators do on the host around their launches, on CPU tensors with the launches replaced."""
import copy
import pickle
import random
import weakref

import pytest
import torch
from torch.autograd import forward_ad

from ascend_rsfa import _native, _overlap, cache4, rotary
from oracle import serving as S

F16, BF16 = torch.float16, torch.bfloat16


class Launches(list):
    """Names of the entry points that a test's calls reach."""


@pytest.fixture
def host(monkeypatch):
    """The operators take CPU tensors, and end where their kernels would start."""
    launches = Launches()
    monkeypatch.setattr(torch.Tensor, "is_cuda", True)
    monkeypatch.setattr(cache4.Cache4, "_call", lambda self, name, args: launches.append(name))
    monkeypatch.setattr(cache4.Cache4, "_on_device", lambda self, fn, *args: fn(*args))
    monkeypatch.setattr(rotary, "_launch", lambda parts, xs, ys, positions: launches.append("rsfa_rotary"))
    monkeypatch.setattr(rotary.RotaryPlan, "turns", lambda self, device: torch.zeros(self.rotary_dim // 2, dtype=torch.float64))
    return launches


def _cache(Z=1, H=2, C=16, D=32, dtype=BF16, **more):
    return cache4.Cache4(Z, H, C, D, dtype, device="cpu", **more)


# -- tensors that share memory --------------------------------------------------
def _bytes(t):
    at = torch.tensor([t.data_ptr()])
    for s, n in zip(t.stride(), t.shape):
        at = (at[:, None] + s * t.element_size() * torch.arange(n)).flatten()
    return (at[:, None] + torch.arange(t.element_size())).flatten().tolist()


def test_shared_bytes_of_strided_tensors():
    rng = random.Random(1)
    memory = torch.zeros(4096, dtype=torch.uint8)
    seen = set()
    for _ in range(4000):
        steps = [rng.choice((0, 1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64)) for _ in range(3)]
        a, b = (memory.as_strided([rng.randint(1, 4) for _ in range(3)] + [rng.choice((1, 2, 4, 8))],
                                  [rng.choice((x, x, rng.choice((0, 1, 3, 4, 8, 16, 32, 40, 64, 128)))) for x in steps] + [1],
                                  rng.choice((0, 8, 16, 64, rng.randint(0, 200)))) for _ in range(2))
        x, y = _bytes(a), _bytes(b)
        want = bool(set(x) & set(y)), len(set(x)) < len(x)
        assert (_overlap.meet(a, b), _overlap.meets_itself(a)) == want, (a.shape, a.stride(), b.shape, b.stride())
        assert _overlap.span(a) == (min(x), max(x) + 1)
        seen.add(want)
    assert len(seen) == 4


def test_out_beside_q_in_one_buffer(host):
    cache = _cache(1, 4, 64, 128)
    heads = torch.zeros((1, 24, 24, 128), dtype=BF16)  # [Z, T, heads, D]: heads of q, others', of out
    q, out = heads[:, :, :8].transpose(1, 2), heads[:, :, 16:].transpose(1, 2)
    assert cache.attend(q, 64, False, 1.0, out=out) is out
    both = torch.zeros((1, 8, 24, 256), dtype=BF16)  # q and out side by side in each row
    out = both[..., 128:]
    assert cache.attend(both[..., :128], 64, False, 1.0, out=out) is out
    # a q that is copied into rows first may lie anywhere, as here with the head dim outside
    flat = torch.zeros(1 << 16, dtype=BF16)
    q = flat.as_strided((1, 4, 16, 128), (0, 16, 1, 64))
    out = flat.as_strided((1, 4, 16, 128), (0, 2048, 128, 1))
    assert cache.attend(q, 64, False, 1.0, out=out) is out
    assert len(host) == 3


def test_out_that_meets_q_or_itself_is_refused(host):
    cache = _cache(1, 4, 64, 128)
    tokens = torch.zeros((1, 48, 32, 128), dtype=BF16)
    q = tokens[:, :32].transpose(1, 2)
    flat = torch.zeros(1 << 20, dtype=BF16)
    for out in (tokens[:, 16:].transpose(1, 2),  # tokens 16 .. 31 are q's too
                tokens[:, 31:32].transpose(1, 2).expand(1, 32, 32, 128),
                tokens.view(-1)[8:].as_strided(q.shape, q.stride()),
                flat.as_strided((1, 32, 32, 128), (0, 64, 4096, 1)),  # heads half a row apart
                flat.as_strided((1, 32, 32, 128), (0, 128, 2048, 1))):  # tokens that meet the heads of others
        with pytest.raises(ValueError, match="share memory"):
            cache.attend(q, 64, False, 1.0, out=out)
    assert not host


def test_rotary_in_place_refuses_tensors_that_share_memory(host):
    plan = rotary.RotaryPlan([1.0] * 16)
    fused = torch.zeros((2, 9, 8, 32))  # [Z, N, heads of q, k and v, D]
    part = lambda a, b: fused[:, :, a:b].transpose(1, 2)  # noqa: E731
    rotary.rotary_(part(0, 4), part(4, 6), 0, plan)
    rotary.rotary_(part(4, 6), part(0, 4), 0, plan)
    assert len(host) == 2
    flat = torch.zeros(4096)
    for q, k in ((part(0, 4), part(3, 5)), (part(2, 4), part(0, 4)), (part(0, 4), part(0, 4)),
                 (fused[:, :8].transpose(1, 2), fused[:, 1:].transpose(1, 2)),  # tokens 1 .. 7 are both's
                 (flat.as_strided((1, 2, 9, 32), (0, 16, 64, 1)), None)):  # heads half a row apart
        with pytest.raises(ValueError, match="share"):
            rotary.rotary_(q, k, 0, plan)
    assert len(host) == 2


@pytest.fixture
def turned(host, monkeypatch):
    """rotary's values from the definition, which know nothing of derivatives, as the kernel's."""
    def forward(q, k, positions, plan, inverse):
        q, k = forward_ad.unpack_dual(q).primal, k if k is None else forward_ad.unpack_dual(k).primal
        p = positions + torch.arange(q.shape[2]) if isinstance(positions, int) else positions
        ys = tuple(S.rotary(x, p, plan.frequencies, plan.amplitude, plan.layout, inverse).to(x.dtype) for x in (q, k) if x is not None)
        return ys[0] if k is None else ys

    monkeypatch.setattr(rotary, "_forward", forward)


@pytest.mark.parametrize("positions", [5, torch.tensor([4, 0, 9])])
def test_rotary_in_forward_mode(turned, positions):
    g = torch.Generator().manual_seed(3)
    q, k, tq, tk, w = (torch.randn((1, 2, 3, 16), generator=g, dtype=torch.float64) for _ in range(5))
    plan = rotary.RotaryPlan([0.3] * 4, amplitude=1.5)
    want = rotary.rotary(tq, tk, positions, plan)
    with forward_ad.dual_level():
        for mode in (torch.enable_grad, torch.no_grad):
            with mode():
                a, b = rotary.rotary(forward_ad.make_dual(q, tq), forward_ad.make_dual(k, tk), positions, plan)
                assert torch.equal(forward_ad.unpack_dual(a).tangent, want[0]) and torch.equal(forward_ad.unpack_dual(b).tangent, want[1])
                # one of the two, and one alone
                a, b = rotary.rotary(q, forward_ad.make_dual(k, tk), positions, plan)
                assert torch.equal(forward_ad.unpack_dual(b).tangent, want[1])
                assert not torch.count_nonzero(forward_ad.unpack_dual(a).tangent)
                a = rotary.rotary(forward_ad.make_dual(q, tq), None, positions, plan)
                assert torch.equal(forward_ad.unpack_dual(a).tangent, want[0])
                assert forward_ad.unpack_dual(rotary.rotary(q, None, positions, plan)).tangent is None
        # a tangent of a gradient, and a gradient of a tangent
        x = q.clone().requires_grad_()
        dx, = torch.autograd.grad(rotary.rotary(x, None, positions, plan), x, forward_ad.make_dual(w, tk))
        back = rotary._turn(tk, None, positions, plan, True)
        assert torch.equal(forward_ad.unpack_dual(dx).tangent, back)
        t = tq.clone().requires_grad_()
        a = forward_ad.unpack_dual(rotary.rotary(forward_ad.make_dual(q, t), None, positions, plan)).tangent
        assert torch.equal(torch.autograd.grad(a, t, tk)[0], back)
        for mode in (torch.enable_grad, torch.no_grad):
            with mode(), pytest.raises(RuntimeError, match="in place"):
                rotary.rotary_(forward_ad.make_dual(q.float(), tq.float()), None, positions, plan)


def test_cache_calls_refuse_tangents(host):
    cache = _cache()
    k, q = torch.zeros((1, 2, 3, 32), dtype=BF16), torch.zeros((1, 4, 3, 32), dtype=BF16)
    with forward_ad.dual_level():
        dual = lambda x: forward_ad.make_dual(x, torch.ones_like(x))  # noqa: E731
        for mode in (torch.enable_grad, torch.no_grad):
            with mode():
                for bad in (lambda: cache.append(dual(k), k, 0), lambda: cache.append(k, dual(k), 0),
                            lambda: cache.attend(dual(q), 3, False, 1.0)):
                    with pytest.raises(RuntimeError, match="no gradients"):
                        bad()
        assert not host
        cache.append(k, k, 0)
        cache.attend(forward_ad.unpack_dual(dual(q)).primal, 3, False, 1.0)
    assert len(host) == 2


def test_rotary_in_place_is_told_to_autograd(host):
    plan = rotary.RotaryPlan([0.3] * 8)
    fused = torch.randn((1, 4, 3, 32))
    for which in range(2):
        b = torch.randn((1, 4, 3, 32), requires_grad=True)
        y = fused * b  # keeps fused for b's gradient
        q, k = fused[:, :3], fused[:, 3:]
        rotary.rotary_(q, None, 0, plan) if which else rotary.rotary_(torch.randn_like(q), k, 0, plan)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()
    with torch.inference_mode():
        rotary.rotary_(torch.randn_like(q), None, 0, plan)
    rotary.rotary_(torch.randn((1, 2, 0, 32)), None, 0, plan)
    assert len(host) == 3


def test_writes_of_cache_calls_are_told_to_autograd(host):
    cache, into = _cache(), _cache(C=8)
    k, q = torch.zeros((1, 2, 3, 32), dtype=BF16), torch.zeros((1, 4, 3, 32), dtype=BF16)
    out = torch.zeros_like(q)
    every = ("k_codes", "k_scales", "v_codes", "v_scales", "positions", "weights")

    def versions():
        return {**{n: getattr(cache, n)._version for n in every}, **{"into." + n: getattr(into, n)._version for n in every}, "out": out._version}

    for call, written in ((lambda: cache.append(k, k, 0), every), (lambda: cache.attend(q, 3, False, 1.0), ()),
                          (lambda: cache.attend(q, 3, False, 1.0, accumulate=True), ("weights",)),
                          (lambda: cache.attend(q, 3, False, 1.0, out=out), ("out",)), (lambda: cache.read(0, 2), ()),
                          (lambda: cache.claim(3, 2), ()), (lambda: cache.evict(into, 3), tuple("into." + n for n in every)),
                          (lambda: cache.append(k[:, :, :0], k[:, :, :0], 0), ())):
        before = versions()
        call()
        assert {n for n, v in versions().items() if v != before[n]} == set(written)
    # as autograd sees it: weights and an out that an earlier product keeps
    for kept, call in ((cache.weights, lambda: cache.attend(q, 3, False, 1.0, accumulate=True)),
                       (out, lambda: cache.attend(q, 3, False, 1.0, out=out))):
        y = kept * torch.ones_like(kept).requires_grad_()
        call()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()
    with pytest.raises(RuntimeError, match="no gradients"):
        cache.attend(q, 3, False, 1.0, out=out.clone().requires_grad_())
    b = {n: getattr(cache, n) for n in every}
    with pytest.raises(ValueError, match="gradient"):
        cache4.Cache4.from_buffers(**{**b, "weights": b["weights"].clone().requires_grad_()}, dtype=BF16)
    with torch.inference_mode():
        mine = _cache()
        mine.append(k, k, 0)
        mine.attend(q, 3, False, 1.0, accumulate=True)


def test_buffers_and_sizes_of_a_cache_stay(host):
    cache = _cache()
    for name in ("k_codes", "k_scales", "v_codes", "v_scales", "positions", "weights"):
        t = getattr(cache, name)
        with pytest.raises(AttributeError, match="fixed"):
            setattr(cache, name, torch.zeros_like(t))
        with pytest.raises(AttributeError, match="fixed"):
            delattr(cache, name)
        assert getattr(cache, name) is t
    for name, value in (("dtype", F16), ("Z", 2), ("H", 1), ("capacity", 8), ("head_dim", 64), ("device", torch.device("cuda:1"))):
        with pytest.raises(AttributeError, match="fixed"):
            setattr(cache, name, value)
    with pytest.raises(AttributeError, match="fixed"):
        _cache(weights=False).weights = cache.weights
    w = cache.weights
    cache.weights += 2.0
    cache.weights *= 0.5
    cache.weights[0, 0] = 4.0
    assert cache.weights is w and w[0, 0].eq(4.0).all() and w[0, 1].eq(1.0).all()


def test_plans_stay_as_they_were_made():
    plan = rotary.rotary_plan(16, base=50.0, layout="interleaved", amplitude=1.25)
    f = plan.frequencies
    for name, value in (("amplitude", 2.0), ("layout", "half"), ("frequencies", f * 2), ("rotary_dim", 8)):
        with pytest.raises(AttributeError):
            setattr(plan, name, value)
    plan.frequencies.mul_(3.0)
    f.zero_()
    again = rotary.rotary_plan(16, base=50.0, layout="interleaved", amplitude=1.25)
    assert (again.amplitude, again.layout, again.rotary_dim) == (1.25, "interleaved", 16)
    assert torch.equal(again.frequencies, rotary.rotary_plan(16, base=50.0).frequencies) and again.frequencies[0] == 1.0
    mine = torch.ones(4, dtype=torch.float64)
    own = rotary.RotaryPlan(mine)
    mine.zero_()
    assert own.frequencies.eq(1.0).all()


def test_copies_of_plans_hold_no_addresses(host):
    plan = rotary.RotaryPlan([0.5, 0.25], "interleaved", 1.5)
    rotary.rotary(torch.zeros((1, 2, 3, 8)), None, 0, plan)
    assert plan._kept
    for other in (copy.deepcopy(plan), copy.copy(plan), pickle.loads(pickle.dumps(plan))):
        assert not other._kept and not other._turns
        assert torch.equal(other.frequencies, plan.frequencies) and (other.layout, other.amplitude) == ("interleaved", 1.5)


def test_caches_are_not_pickled_or_copied_by_value(host):
    cache = _cache()
    cache.append(torch.zeros((1, 2, 3, 32), dtype=BF16), torch.zeros((1, 2, 3, 32), dtype=BF16), 0)
    for bad in (lambda: pickle.dumps(cache), lambda: copy.deepcopy(cache)):
        with pytest.raises(ValueError, match="cannot be pickled"):
            bad()


def test_a_refused_claim_leaves_nothing_behind(host, monkeypatch):
    cache, sizes = _cache(1, 1, 40000), []
    monkeypatch.setattr(cache4.Cache4, "_call", lambda self, name, args: sizes.append(
        _native.Cache4EvictArgs.from_buffer_copy(args).workspace_bytes))
    with pytest.raises(ValueError, match="n must"):
        cache.claim(40000, (1 << 30) + 1, budget=100)
    cache.claim(40000, 1, budget=100)
    cache.claim(40000, 1 << 10, budget=100)
    assert len(sizes) == 2 and sizes[0] == sizes[1] > 0


@pytest.fixture
def device(monkeypatch):
    """Plans prepare frequencies for a device that is not there; True in the list: under capture."""
    class Stream:
        def synchronize(self):
            pass

    capturing = []
    monkeypatch.setattr(torch.Tensor, "to", lambda self, device: self)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device: Stream())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: bool(capturing))
    return capturing


def test_turns_of_the_current_device(device):
    capturing = device
    plan = rotary.RotaryPlan([0.5, 0.25])
    t = plan.turns("cuda")
    capturing.append(True)  # a graph's calls find what was asked for before
    assert plan.turns(torch.device("cuda", 1)) is t and plan.turns("cuda:1") is t
    for other in ("cuda:0", torch.device("cuda", 2)):
        with pytest.raises(RuntimeError, match="before capturing"):
            plan.turns(other)


def test_frequencies_outlive_a_dropped_plan(device, monkeypatch):
    waits, dead = [], []
    monkeypatch.setattr(torch.cuda, "synchronize", lambda device: waits.append([r() is not None for r in dead]))
    for i in range(600):
        plan = rotary.RotaryPlan([0.5, 0.25])
        dead.append(weakref.ref(plan.turns("cuda")))
        del plan
        # launches on other streams may still read them: none is freed without a wait since its plan's end
        alive = [r() is not None for r in dead]
        last = len(waits[-1]) if waits else 0
        assert all(alive[last:]) and sum(alive) <= 300
    assert 2 <= len(waits) <= 4 and all(w[-1] for w in waits)


def test_plans_of_learned_frequencies_are_refused():
    f = torch.tensor([0.5, 0.25], requires_grad=True)
    for bad in (f, f * 2, torch.nn.Parameter(torch.ones(2, dtype=torch.float64))):
        with pytest.raises(RuntimeError, match="constants"):
            rotary.RotaryPlan(bad)
    with forward_ad.dual_level(), torch.no_grad(), pytest.raises(RuntimeError, match="constants"):
        rotary.RotaryPlan(forward_ad.make_dual(f.detach(), torch.ones(2)))
    with torch.no_grad():
        assert rotary.RotaryPlan(f).frequencies.tolist() == [0.5, 0.25]
    assert rotary.RotaryPlan(f.detach()).frequencies.tolist() == [0.5, 0.25]


def test_plans_of_arguments_that_change():
    # a number in a tensor is taken when the plan is asked for
    factor, base, dim = torch.tensor(2.0, dtype=torch.float64), torch.tensor(100.0), torch.tensor(8)
    first = rotary.rotary_plan(dim, base=base, scaling="linear", factor=factor)
    factor.fill_(4.0)
    base.fill_(50.0)
    dim.fill_(16)
    second = rotary.rotary_plan(dim, base=base, scaling="linear", factor=factor)
    assert torch.equal(first.frequencies, rotary.rotary_plan(8, base=100.0, scaling="linear", factor=2.0).frequencies)
    assert torch.equal(second.frequencies, rotary.rotary_plan(16, base=50.0, scaling="linear", factor=4.0).frequencies)
    assert rotary.rotary_plan(16, base=50) is rotary.rotary_plan(16, base=torch.tensor(50.0))


def test_plans_and_checks_under_another_default_device():
    want = rotary.rotary_plan(12, base=77.0).frequencies
    a, b = torch.zeros(64).as_strided((1, 2, 3, 8), (0, 3, 5, 1)), torch.zeros(64).as_strided((1, 2, 3, 8), (0, 5, 3, 1))
    assert (_overlap.meets_itself(a), _overlap.meet(a, b[..., :4])) == (True, False)
    with torch.device("meta"):
        rotary._plan.cache_clear()
        assert torch.equal(rotary.rotary_plan(12, base=77.0).frequencies, want)
        assert rotary.RotaryPlan([0.5, 0.25]).frequencies.tolist() == [0.5, 0.25]
        for f in (_overlap._runs_overlap, _overlap._runs_meet):
            f.cache_clear()
        assert _overlap.meets_itself(a) and _overlap.meet(a, a.as_strided((1, 2, 3, 4), (0, 5, 3, 1), 1))
