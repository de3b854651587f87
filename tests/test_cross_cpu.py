"""CPU tests of cross attention: refusals of the package and of the C ABI, the definition's gradients.

Nothing here launches a kernel: every call is refused by its argument checks."""
import ctypes

import pytest
import torch

from ascend_rsfa import _native, cross
from ascend_rsfa.cross import cross_attention
from cross_launches import variants
from oracle import cross as O
from test_cross_gpu import SHAPES, VARIANTS


def test_struct_layouts():
    assert ctypes.sizeof(_native.CrossArgs) == 8 + 40 + 48 + 128 + 8 + 8 + 16
    assert ctypes.sizeof(_native.CrossBwdArgs) == 8 + 80 + 48 + 256 + 8 + 8 + 16
    assert "cross" in _native.strerror(_native.E_CROSS)


def _args(kind=_native.CrossArgs, **over):
    a = kind()
    a.struct_size = ctypes.sizeof(a)
    for name, _ in kind._fields_:
        if name.endswith("_stride"):
            getattr(a, name)[:] = (1024, 256, 64, 1)
            setattr(a, name[:-7], 0x1000)
    a.z, a.heads, a.key_heads, a.t, a.n, a.head_dim, a.sm_scale = 2, 4, 2, 4, 40, 64, 1.0
    if kind is _native.CrossBwdArgs:
        a.lse = 0x1000
    for k, v in over.items():
        setattr(a, k, v)
    return a


CALLS = [("rsfa_cross_fwd", _native.CrossArgs), ("rsfa_cross_bwd", _native.CrossBwdArgs)]


@pytest.mark.parametrize("name,kind", CALLS)
def test_abi_refusals(name, kind):
    lib = _native.lib()
    f = lambda **k: getattr(lib, name)(ctypes.byref(_args(kind, **k)), None)  # noqa: E731
    size = lambda **k: getattr(lib, name + "_workspace_bytes")(ctypes.byref(_args(kind, **k)))  # noqa: E731
    assert getattr(lib, name)(None, None) == _native.E_NULL
    assert f(struct_size=8) == _native.E_ABI and size(struct_size=8) == 0
    assert f(dtype=2) == f(dtype=3) == f(dtype=-1) == _native.E_DTYPE
    for over in ({"z": 0}, {"heads": 0}, {"heads": 3}, {"key_heads": 0}, {"t": 0}, {"n": 0}, {"t": 1 << 29}, {"n": 1 << 31}, {"head_dim": 16},
                 {"head_dim": 96}, {"z": 1 << 25}, {"heads": 1 << 24}, {"t": -1}, {"heads": 256, "key_heads": 1, "t": 1 << 21}):
        assert f(**over) == _native.E_CROSS and size(**over) == 0, over
    for p in ("q", "k", "v", "o"):
        assert f(**{p: None}) == _native.E_NULL and f(**{p: 0x1008}) == _native.E_ALIGN
        for st in ((1024, 256, 64, 2), (1024, 256, 65, 1), (-1024, 256, 64, 1), (1024, 4, 64, 1), (1024, 256, 1 << 25, 1)):
            assert f(**{p + "_stride": (ctypes.c_int64 * 4)(*st)}) == _native.E_ALIGN
    assert f(lse=0x1002) == f(lengths=0x1001) == _native.E_ALIGN
    need = size(z=1, heads=1, key_heads=1, t=4, n=100000)
    assert need > 0
    small = {"z": 1, "heads": 1, "key_heads": 1, "t": 4, "n": 100000}
    assert f(**small) == f(**small, workspace=0x1000, workspace_bytes=need - 1) == _native.E_WORKSPACE
    assert f(**small, workspace=0x1008, workspace_bytes=need) == _native.E_ALIGN


def test_backward_abi_refusals():
    f = lambda **k: _native.lib().rsfa_cross_bwd(ctypes.byref(_args(_native.CrossBwdArgs, **k)), None)  # noqa: E731
    assert f(lse=None) == f(grad_o=None) == _native.E_NULL
    assert f(grad_lse=0x1002) == f(grad_o=0x1008) == f(grad_q=0x1008) == f(grad_k=0x1004) == f(grad_v=0x1001) == _native.E_ALIGN


def test_cpu_tensors_are_refused():
    x = torch.zeros((1, 1, 4, 64), dtype=torch.float16)
    with pytest.raises(ValueError, match="GPU"):
        cross_attention(x, x, x, 1.0)


def test_the_definitions_gradients_against_differences():
    g = torch.Generator().manual_seed(0)
    q, k, v, go = (torch.randn(s, generator=g, dtype=torch.float64) for s in ((2, 4, 3, 4), (2, 2, 5, 4), (2, 2, 5, 4), (2, 4, 3, 4)))
    glse = torch.randn((2, 4, 3), generator=g, dtype=torch.float64)
    lengths = [5, 3]
    want = O.expect(q, k, v, lengths, 0.7, go, glse)
    for i, name in enumerate(("dq", "dk", "dv")):
        for at in range(0, (q, k, v)[i].numel(), 3):
            def value(step):
                x = [q, k, v]
                x[i] = x[i].clone()
                x[i].view(-1)[at] += step
                o, lse = O.attend(*x, lengths, 0.7)
                return float((o * go).sum() + (lse * glse).sum())

            slope = (value(1e-5) - value(-1e-5)) / 2e-5
            assert abs(slope - float(want[name][0].view(-1)[at])) < 1e-8


def test_the_shapes_of_the_variants_test_run_every_forward_variant(tmp_path):
    seen = set()
    for shape, launches in zip(VARIANTS, variants(VARIANTS, tmp_path)):
        (name, numbers), *rest = launches
        assert [x for x, _ in rest] in ([], ["cross_join_kernel"]) and numbers[0] == shape[5]
        seen.add((name, numbers[:3] if name == "fa_fwd_kernel" else numbers[:2], bool(rest)))
    few = [("cross_few_kernel", (d, nb)) for d in (32, 64, 128, 256) for nb in (1, 2, 4) if (d, nb) != (256, 4)]
    many = [("fa_fwd_kernel", x) for x in ((32, 64, 4), (32, 128, 4), (64, 64, 4), (64, 128, 8), (128, 64, 4), (128, 64, 8),
                                           (256, 32, 4), (256, 32, 8))]
    assert seen == {(name, numbers, parts) for name, numbers in few + many for parts in (False, True)}


def test_the_shapes_of_the_definitions_test_run_every_backward_variant(tmp_path):
    for d in (32, 64, 128, 256):
        seen = set()
        for launches in variants([s[:5] + (d,) for s in SHAPES], tmp_path, "rsfa_cross_bwd"):
            names = [x for x, _ in launches]
            dq = names.index("cross_dkv_kernel")
            assert names[0] == "cross_dq_kernel" and set(names[1:dq] + names[dq + 1:]) <= {"sum_parts_kernel"}
            seen.add((dq > 1, len(names) > dq + 1))
        assert {x for x, _ in seen} == {x for _, x in seen} == {False, True}


class _Calls:
    """cross_attention on the CPU with its launches recorded: what each would read, by its addresses and strides."""

    def __init__(self, monkeypatch):
        self.tensors, self.calls = {}, []
        monkeypatch.setattr(cross, "_PLANS", {})
        monkeypatch.setattr(cross, "_check", lambda *a: None)
        monkeypatch.setattr(cross, "_on_device", lambda index, fn, *a: fn(*a))
        monkeypatch.setattr(cross, "_launch", self.launch)

    def launch(self, index, name, args):
        if name == "rsfa_cross_bwd":
            self.calls.append(_native.CrossBwdArgs.from_buffer_copy(args))

    def known(self, *tensors):
        self.tensors.update({t.data_ptr(): t for t in tensors})

    def last_reads_them(self):
        """The last backward call's strides are those of the tensors at its addresses."""
        a = self.calls[-1]
        return all(tuple(getattr(a, n + "_stride")) == self.tensors[getattr(a, n)].stride() for n in ("q", "k", "v", "o") if getattr(a, n) in self.tensors)


def _fused(Z, N, H, D):
    """K and V, parts of one projection."""
    big = torch.randn((Z, N, 2, H, D)).to(torch.bfloat16)
    return big[:, :, 0].transpose(1, 2).requires_grad_(), big[:, :, 1].transpose(1, 2).requires_grad_()


@pytest.mark.parametrize("order", ["kept first", "hook first"])
def test_saved_tensors_that_a_hook_brings_back_in_another_layout(order, monkeypatch):
    calls = _Calls(monkeypatch)
    q = torch.randn((2, 7, 4, 64)).to(torch.bfloat16).transpose(1, 2).requires_grad_()
    k, v = _fused(2, 5, 4, 64)
    go = torch.ones((2, 4, 7, 64), dtype=torch.bfloat16)
    back = []

    def unpack(t):
        back.append(t)
        if t.dim() == 4:
            calls.known(t)
        return t

    def step(hook):
        if hook:
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().clone(memory_format=torch.contiguous_format), unpack):
                o = cross_attention(q, k, v, 0.125)
        else:
            o = cross_attention(q, k, v, 0.125)
            calls.known(q, k, v, o)
        torch.autograd.grad(o, (q, k, v), go)
        assert calls.last_reads_them(), (order, hook)

    for hook in (False, True, False) if order == "kept first" else (True, False, True):
        step(hook)
    assert len(calls.calls) == 3 and any(t.stride() != k.stride() for t in back if t.shape == k.shape)


def test_saved_tensors_that_are_not_aligned_are_copied(monkeypatch):
    calls = _Calls(monkeypatch)
    q, k, v = (torch.randn((1, 2, n, 32)).to(torch.float16).requires_grad_() for n in (3, 6, 6))
    go = torch.ones((1, 2, 3, 32), dtype=torch.float16)

    def shifted(t):
        big = torch.empty(t.numel() + 1, dtype=t.dtype)
        return big[1:].view(t.shape).copy_(t)

    for _ in range(2):
        torch.autograd.grad(cross_attention(q, k, v, 1.0), (q, k, v), go)
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, shifted):
            o = cross_attention(q, k, v, 1.0)
        torch.autograd.grad(o, (q, k, v), go)
        a = calls.calls[-1]
        assert not any(getattr(a, n) % 16 for n in ("q", "k", "v", "o"))


@pytest.mark.parametrize("wrong", [lambda t: t[..., :t.shape[-1] // 2], lambda t: t.double(), lambda t: t.to("meta"), lambda t: t[:1]])
def test_saved_tensors_that_come_back_as_others_are_refused(wrong, monkeypatch):
    calls = _Calls(monkeypatch)
    q, k, v = (torch.randn((2, 2, n, 32)).to(torch.float16).requires_grad_() for n in (3, 6, 6))
    n = torch.tensor([6, 4], dtype=torch.int32)
    for _ in range(2):
        torch.autograd.grad(cross_attention(q, k, v, 1.0, n).sum(), (q, k, v))
    done = len(calls.calls)
    for which in range(6):  # of q, k, v, o, lse, lengths, in the order in which they come back
        count = iter(range(6))
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: wrong(t) if next(count) == which else t):
            o = cross_attention(q, k, v, 1.0, n)
        with pytest.raises(RuntimeError, match="came back as"):
            torch.autograd.grad(o.sum(), (q, k, v))
    assert len(calls.calls) == done
