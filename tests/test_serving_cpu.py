"""CPU tests of the serving operators: plans, refusals of the package and of the C ABI.

Nothing here launches a kernel: every call is refused by its argument checks."""
import ctypes
import math

import pytest
import torch

from ascend_rsfa import _native, cache4, rotary


def test_struct_layouts():
    assert ctypes.sizeof(_native.RotaryArgs) == 8 + 32 + 32 + 16 + 128 + 8 + 16 + 8 + 8 + 8
    assert ctypes.sizeof(_native.Cache4) == 48 + 32 + 48 + 8
    assert ctypes.sizeof(_native.Cache4RowsArgs) == 8 + 136 + 24 + 64 + 40
    assert ctypes.sizeof(_native.Cache4AttendArgs) == 8 + 136 + 24 + 16 + 64 + 24 + 16 + 8 + 16
    assert ctypes.sizeof(_native.Cache4EvictArgs) == 8 + 272 + 16 + 32 + 24


def test_strerror_covers_the_new_codes():
    msgs = [_native.strerror(c) for c in (-12, -13, -14)]
    assert len(set(msgs)) == 3 and not any("unknown" in m for m in msgs)


def test_plans():
    p = rotary.rotary_plan(8, base=100.0)
    assert p.rotary_dim == 8 and p.frequencies.dtype == torch.float64
    assert torch.allclose(p.frequencies, torch.tensor([1.0, 100.0 ** -0.25, 0.1, 100.0 ** -0.75], dtype=torch.float64), rtol=1e-15)
    assert torch.equal(rotary.rotary_plan(8, base=100.0, scaling="linear", factor=4.0).frequencies, p.frequencies / 4.0)
    ntk = rotary.rotary_plan(8, base=100.0, scaling="ntk", factor=4.0).frequencies
    # the fastest stays, the slowest is divided by the factor
    assert ntk[0] == 1.0 and math.isclose(ntk[-1], p.frequencies[-1] / 4.0, rel_tol=1e-14)
    parts = rotary.rotary_plan(8, base=100.0, scaling="by_parts", factor=4.0, original_length=round(20 * math.pi), low=1.5,
                               high=9.0, amplitude=1.25)
    # turns within 63 positions: 10.03 (kept), 3.17 (the ramp), 1.003 and 0.32 (divided)
    keep = (63 * p.frequencies[1] / (2 * math.pi) - 1.5) / 7.5
    want = [1.0, float(keep * p.frequencies[1] + (1 - keep) * p.frequencies[1] / 4.0), 0.025, float(p.frequencies[3]) / 4.0]
    assert torch.allclose(parts.frequencies, torch.tensor(want, dtype=torch.float64), rtol=1e-14) and parts.amplitude == 1.25


@pytest.mark.parametrize("call", [
    lambda: rotary.rotary_plan(7), lambda: rotary.rotary_plan(0), lambda: rotary.rotary_plan(8, base=0.0),
    lambda: rotary.rotary_plan(8, scaling="other"), lambda: rotary.rotary_plan(8, layout="other"),
    lambda: rotary.rotary_plan(8, scaling="by_parts", factor=2.0),
    lambda: rotary.rotary_plan(8, scaling="by_parts", factor=2.0, original_length=64, low=4.0, high=4.0),
    lambda: rotary.rotary_plan(2, scaling="ntk", factor=2.0), lambda: rotary.rotary_plan(8, factor=0.0),
    lambda: rotary.RotaryPlan(torch.ones(2, 2)), lambda: rotary.RotaryPlan([math.inf]),
    lambda: rotary.RotaryPlan([1.0], amplitude=math.nan),
])
def test_plan_refusals(call):
    with pytest.raises(ValueError):
        call()


def test_cpu_tensors_are_refused():
    with pytest.raises(ValueError):
        rotary.rotary(torch.zeros(1, 1, 1, 16), None, 0, rotary.rotary_plan(16))
    with pytest.raises(ValueError):
        cache4.Cache4(1, 1, 8, 64, device="cpu")
    for bad in ({"head_dim": 16}, {"head_dim": 96}, {"Z": 0}, {"capacity": 0}):
        with pytest.raises(ValueError):
            cache4.Cache4(**{"Z": 1, "H": 1, "capacity": 8, "head_dim": 64, "device": "cpu", **bad})
    with pytest.raises(TypeError):
        cache4.Cache4(1, 1, 8, 64, dtype=torch.float32, device="cpu")


# -- the C ABI --------------------------------------------------------------
def _rotary(**over):
    a = _native.RotaryArgs()
    a.struct_size = ctypes.sizeof(a)
    a.x[0] = a.y[0] = 0x1000
    a.z, a.n, a.head_dim, a.rotary_dim = 1, 4, 64, 64
    a.heads[:] = (2, 2)
    for i in range(2):
        a.x_stride[i][:] = a.y_stride[i][:] = (512, 256, 64, 1)
    a.turns = 0x1000
    for k, v in over.items():
        setattr(a, k, v)
    return a


def test_rotary_abi_refusals():
    f = lambda a: _native.lib().rsfa_rotary(ctypes.byref(a), None)  # noqa: E731
    assert _native.lib().rsfa_rotary(None, None) == _native.E_NULL
    assert f(_rotary(struct_size=8)) == _native.E_ABI
    assert f(_rotary(turns=None)) == _native.E_NULL
    assert f(_rotary(turns=0x1004)) == _native.E_ALIGN
    assert f(_rotary(dtype=2)) == _native.E_DTYPE
    assert f(_rotary(z=0)) == _native.E_SHAPE
    assert f(_rotary(n=0)) == _native.E_SHAPE
    for dim in (0, 3, 66, -2):
        assert f(_rotary(rotary_dim=dim)) == _native.E_ROTARY
    a = _rotary()
    a.x[1] = 0x1000  # x without y
    assert f(a) == _native.E_NULL
    a = _rotary()
    a.x_stride[0][3] = 2
    assert f(a) == _native.E_ALIGN
    a = _rotary()
    a.x[0] = 0x1001
    assert f(a) == _native.E_ALIGN
    a = _rotary()
    a.y_stride[0][1] = 128  # in place, with other strides
    assert f(a) == _native.E_ALIGN
    a = _rotary()
    a.heads[0] = 0
    assert f(a) == _native.E_SHAPE
    assert f(_rotary(positions=0x1002)) == _native.E_ALIGN
    assert f(_rotary(positions=0x1004, flags=_native.ROTARY_POS64)) == _native.E_ALIGN


def _cache(**over):
    c = _native.Cache4()
    for name in ("k_codes", "k_scales", "v_codes", "v_scales", "positions", "weights"):
        setattr(c, name, 0x1000)
    c.z, c.h, c.capacity, c.head_dim = 2, 3, 40, 128
    c.code_stride[:] = (3 * 40 * 64, 40 * 64)
    c.scale_stride[:] = (3 * 40 * 4, 40 * 4)
    c.slot_stride[:] = (3 * 40, 40)
    for k, v in over.items():
        setattr(c, k, v)
    return c


def _rows(cache=None, **over):
    a = _native.Cache4RowsArgs()
    a.struct_size = ctypes.sizeof(a)
    a.cache = cache if cache is not None else _cache()
    a.k = a.v = 0x1000
    a.t = 2
    a.k_stride[:] = a.v_stride[:] = (768, 256, 128, 1)
    for k, v in over.items():
        setattr(a, k, v)
    return a


def _attend(cache=None, **over):
    a = _native.Cache4AttendArgs()
    a.struct_size = ctypes.sizeof(a)
    a.cache = cache if cache is not None else _cache()
    a.q = a.o = 0x1000
    a.heads, a.t, a.length, a.sm_scale = 6, 2, 40, 1.0
    a.q_stride[:] = a.o_stride[:] = (1536, 256, 128, 1)
    for k, v in over.items():
        setattr(a, k, v)
    return a


def _evict(cache=None, into=None, **over):
    a = _native.Cache4EvictArgs()
    a.struct_size = ctypes.sizeof(a)
    a.cache = cache if cache is not None else _cache()
    a.into = into if into is not None else _cache(capacity=16)
    a.length, a.n, a.budget, a.recent, a.sinks = 40, 4, 16, 4, 2
    a.out, a.workspace, a.workspace_bytes = 0x1000, 0x1000, 1 << 20
    for k, v in over.items():
        setattr(a, k, v)
    return a


BAD_CACHES = [
    ({"k_codes": None}, _native.E_NULL), ({"positions": None}, _native.E_NULL), ({"dtype": 2}, _native.E_DTYPE),
    ({"dtype": 3}, _native.E_DTYPE), ({"head_dim": 16}, _native.E_CACHE), ({"head_dim": 96}, _native.E_CACHE),
    ({"z": 0}, _native.E_CACHE), ({"h": -1}, _native.E_CACHE), ({"capacity": 0}, _native.E_CACHE),
    ({"capacity": 1 << 31}, _native.E_CACHE), ({"v_codes": 0x1008}, _native.E_ALIGN), ({"k_scales": 0x1002}, _native.E_ALIGN),
    ({"weights": 0x1002}, _native.E_ALIGN), ({"code_stride": (ctypes.c_int64 * 2)(8, 8)}, _native.E_ALIGN),
    ({"scale_stride": (ctypes.c_int64 * 2)(2, 2)}, _native.E_ALIGN), ({"slot_stride": (ctypes.c_int64 * 2)(-40, 40)}, _native.E_ALIGN),
]


@pytest.mark.parametrize("over,status", BAD_CACHES)
def test_every_call_refuses_a_bad_cache(over, status):
    lib = _native.lib()
    for fn, make in ((lib.rsfa_cache4_append, _rows), (lib.rsfa_cache4_read, _rows), (lib.rsfa_cache4_attend, _attend),
                     (lib.rsfa_cache4_claim, _evict), (lib.rsfa_cache4_evict, _evict)):
        assert fn(ctypes.byref(make(_cache(**over))), None) == status
    assert lib.rsfa_cache4_evict(ctypes.byref(_evict(into=_cache(**{"capacity": 16, **over}))), None) == status


def test_cache_calls_abi_refusals():
    lib = _native.lib()
    for fn, make in ((lib.rsfa_cache4_append, _rows), (lib.rsfa_cache4_read, _rows), (lib.rsfa_cache4_attend, _attend),
                     (lib.rsfa_cache4_claim, _evict), (lib.rsfa_cache4_evict, _evict)):
        assert fn(None, None) == _native.E_NULL
        assert fn(ctypes.byref(make(struct_size=4)), None) == _native.E_ABI
        assert fn(ctypes.byref(make(**({"lengths": 0x1002}))), None) == _native.E_ALIGN
    r = lambda **k: lib.rsfa_cache4_append(ctypes.byref(_rows(**k)), None)  # noqa: E731
    assert r(k=None) == r(v=None) == _native.E_NULL
    assert r(t=0) == _native.E_CACHE and r(t=1 << 31) == _native.E_CACHE
    assert r(k=0x1008) == _native.E_ALIGN and r(slots=0x1001) == _native.E_ALIGN and r(counts=0x1001) == _native.E_ALIGN
    for st in ((768, 256, 128, 2), (768, 256, 129, 1), (-768, 256, 128, 1)):
        assert r(k_stride=(ctypes.c_int64 * 4)(*st)) == _native.E_ALIGN
        assert r(v_stride=(ctypes.c_int64 * 4)(*st)) == _native.E_ALIGN
    assert lib.rsfa_cache4_read(ctypes.byref(_rows(k=None, v=None)), None) == _native.E_NULL
    t = lambda cache=None, **k: lib.rsfa_cache4_attend(ctypes.byref(_attend(cache, **k)), None)  # noqa: E731
    assert t(q=None) == t(o=None) == _native.E_NULL
    assert t(heads=4) == t(heads=0) == t(t=0) == t(max_length=-1) == _native.E_CACHE
    assert t(q=0x1004) == t(lse=0x1002) == t(pos_start=0x1001) == _native.E_ALIGN
    assert t(_cache(weights=None), accumulate=1) == _native.E_NULL
    need = lib.rsfa_cache4_attend_workspace_bytes(ctypes.byref(_attend(accumulate=1)))
    assert need > 0 and lib.rsfa_cache4_attend_workspace_bytes(ctypes.byref(_attend(heads=4))) == 0
    assert t(accumulate=1) == t(accumulate=1, workspace=0x1000, workspace_bytes=need - 1) == _native.E_WORKSPACE
    assert t(accumulate=1, workspace=0x1008, workspace_bytes=need) == _native.E_ALIGN
    for fn in (lib.rsfa_cache4_claim, lib.rsfa_cache4_evict):
        e = lambda cache=None, into=None, **k: fn(ctypes.byref(_evict(cache, into, **k)), None)  # noqa: E731
        assert e(_cache(weights=None)) == _native.E_NULL
        assert e(budget=0) == e(budget=41) == e(recent=-1) == e(sinks=-1) == _native.E_BUDGET
        assert e(recent=15) == e(recent=1 << 62) == e(sinks=1 << 62) == _native.E_BUDGET
        assert e(out=0x1002) == _native.E_ALIGN
    assert lib.rsfa_cache4_claim(ctypes.byref(_evict(n=0)), None) == _native.E_BUDGET
    need = lib.rsfa_cache4_evict_workspace_bytes(ctypes.byref(_evict()), 1)
    assert need >= 2 * 3 * 16 * 4 and lib.rsfa_cache4_evict_workspace_bytes(ctypes.byref(_evict()), 0) == 0
    assert lib.rsfa_cache4_evict_workspace_bytes(ctypes.byref(_evict(budget=0)), 1) == 0
    long = {"capacity": 40000, "code_stride": (ctypes.c_int64 * 2)(3 * 40000 * 64, 40000 * 64)}
    assert lib.rsfa_cache4_evict_workspace_bytes(ctypes.byref(_evict(_cache(**long))), 0) > 0
    assert lib.rsfa_cache4_claim(ctypes.byref(_evict(out=None)), None) == _native.E_NULL
    for make, fn in ((lambda **k: _evict(**k), lib.rsfa_cache4_evict), (lambda **k: _evict(_cache(**long), **k), lib.rsfa_cache4_claim)):
        for over in ({"workspace": None}, {"workspace_bytes": 8}):
            assert fn(ctypes.byref(make(**over)), None) == _native.E_WORKSPACE
        assert fn(ctypes.byref(make(workspace=0x1008, workspace_bytes=1 << 30)), None) == _native.E_ALIGN
    for over in ({"z": 1}, {"h": 2}, {"head_dim": 64}, {"dtype": 1}, {"capacity": 15}):
        assert lib.rsfa_cache4_evict(ctypes.byref(_evict(into=_cache(**{"capacity": 16, **over}))), None) == _native.E_BUDGET
