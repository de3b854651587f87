"""CPU tests of the operators on drafted tokens: refusals of the package and of the C ABI, the definitions.

Nothing here launches a kernel: every call is refused by its argument checks."""
import ctypes

import pytest
import torch

from ascend_rsfa import _native
from ascend_rsfa.draft import DraftTree, draft_tree
from oracle import draft as O
from test_serving_cpu import BAD_CACHES, _attend, _cache


def test_struct_layouts():
    assert ctypes.sizeof(_native.DraftTreeArgs) == 8 + 8 + 8 + 16 + 16
    assert ctypes.sizeof(_native.Cache4KeepArgs) == 8 + 136 + 16 + 32
    assert "drafted" in _native.strerror(_native.E_DRAFT)


def _tree(**over):
    a = _native.DraftTreeArgs()
    a.struct_size = ctypes.sizeof(a)
    a.parents = a.bits = a.depths = 0x1000
    a.parents_stride, a.trees, a.t = 4, 2, 4
    for k, v in over.items():
        setattr(a, k, v)
    return a


def _keep(cache=None, **over):
    a = _native.Cache4KeepArgs()
    a.struct_size = ctypes.sizeof(a)
    a.cache = cache if cache is not None else _cache()
    a.tokens, a.n, a.length = 0x1000, 4, 10
    for k, v in over.items():
        setattr(a, k, v)
    return a


def test_tree_abi_refusals():
    lib = _native.lib()
    f = lambda **k: lib.rsfa_draft_tree(ctypes.byref(_tree(**k)), None)  # noqa: E731
    assert lib.rsfa_draft_tree(None, None) == _native.E_NULL
    assert f(struct_size=8) == _native.E_ABI
    assert f(parents=None) == f(bits=None) == f(depths=None) == _native.E_NULL
    assert f(parents=0x1002) == f(bits=0x1001) == f(depths=0x1002) == _native.E_ALIGN
    assert f(t=0) == f(t=513) == f(trees=0) == f(trees=1 << 25) == f(parents_stride=-1) == _native.E_DRAFT


@pytest.mark.parametrize("over,status", BAD_CACHES)
def test_keep_and_attend_refuse_a_bad_cache(over, status):
    lib = _native.lib()
    if over.get("weights", 1) != 0:
        assert lib.rsfa_cache4_keep(ctypes.byref(_keep(_cache(**over))), None) == status
    assert lib.rsfa_cache4_attend_tree(ctypes.byref(_attend(_cache(**over))), 0x1000, 0, None) == status


def test_keep_abi_refusals():
    lib = _native.lib()
    f = lambda **k: lib.rsfa_cache4_keep(ctypes.byref(_keep(**k)), None)  # noqa: E731
    assert lib.rsfa_cache4_keep(None, None) == _native.E_NULL
    assert f(struct_size=8) == _native.E_ABI
    assert f(tokens=None) == _native.E_NULL
    assert f(tokens=0x1002) == f(lengths=0x1001) == f(counts=0x1001) == f(pos_start=0x1003) == _native.E_ALIGN
    assert f(n=0) == f(n=513) == _native.E_DRAFT


def test_attend_tree_abi_refusals():
    lib = _native.lib()
    f = lambda bits=0x1000, stride=0, **k: lib.rsfa_cache4_attend_tree(ctypes.byref(_attend(**k)), bits, stride, None)  # noqa: E731
    assert lib.rsfa_cache4_attend_tree(None, 0x1000, 0, None) == f(bits=None) == _native.E_NULL
    assert f(struct_size=8) == _native.E_ABI
    assert f(bits=0x1002) == _native.E_ALIGN
    assert f(accumulate=1) == f(pos_start=0x1000) == f(stride=-1) == f(t=513) == _native.E_DRAFT
    assert f(q=None) == _native.E_NULL and f(heads=4) == _native.E_CACHE and f(q=0x1004) == _native.E_ALIGN


def test_cpu_tensors_are_refused():
    with pytest.raises(ValueError, match="GPU"):
        draft_tree(torch.zeros(4, dtype=torch.int32))
    with pytest.raises(ValueError, match="GPU"):
        DraftTree(torch.zeros((1, 4, 1), dtype=torch.int32))
    with pytest.raises(TypeError):
        draft_tree(torch.zeros(4))


@pytest.mark.parametrize("name", ["bits", "depths", "trees", "tokens"])
def test_a_trees_attributes_are_read_only(name):
    tree = DraftTree.__new__(DraftTree)
    with pytest.raises(AttributeError):
        setattr(tree, name, None)


def test_the_definitions():
    parents = [-1, 0, 0, 2, -1]
    assert O.depths(parents) == [0, 1, 1, 2, 0]
    see = O.seen(parents)
    assert see.int().tolist() == [[1, 0, 0, 0, 0], [1, 1, 0, 0, 0], [1, 0, 1, 0, 0], [1, 0, 1, 1, 0], [0, 0, 0, 0, 1]]
    assert O.pack(see).flatten().tolist() == [1, 3, 5, 13, 16]
    high = torch.zeros(1, 33, 33, dtype=torch.bool)
    high[0, 0, 31:] = True
    assert O.pack(high)[0, 0].tolist() == [-(1 << 31), 1]
    v = O.visible(see[None], [7], [4], 8)[0].int().tolist()
    assert v[3] == [1, 1, 1, 1, 0, 1, 1, 0] and v[4] == [0] * 8
    b = torch.arange(6).reshape(1, 1, 6)
    assert O.keep(b, [[2, 0, 9]], [2], None)[0, 0].tolist() == [0, 1, 4, 2, 4, 5]
