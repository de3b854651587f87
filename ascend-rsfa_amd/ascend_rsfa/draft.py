"""Trees of drafted tokens, on MI355X (gfx950).

A program that drafts proposes several tokens that may follow a sequence's text, more than one
for some places, and has the model look at all of them in one pass: each drafted token attends to the
context and to the drafted tokens on its own path.  ``draft_tree`` makes the table of
who sees whom from the tokens' parents, once a step for all layers (once for all steps where the
tree does not change); ``Cache4.attend(..., tree=tree)`` attends by it, and ``Cache4.keep`` keeps the
path that was accepted::

    tree = draft_tree(parents)                          # int32 [T] or [Z, T]
    q, k = rotary(q, k, lengths[:, None] + tree.depths, plan)
    cache.append(k, v, lengths)                         # lengths: of the contexts
    o = cache.attend(q, lengths + T, True, scale, tree=tree)
    ...                                                 # the path [Z, n] that the model agrees with, counts [Z]
    cache.keep(path, lengths, counts=counts)
    lengths += counts

The table is made by ``rsfa_draft_tree`` of ``lib/librsfa.so`` on the current stream of the tensors'
device; there is no other path.
"""
import ctypes

import torch

from . import _native
from .flash_attention_forward import _raise_for

__all__ = ["DraftTree", "draft_tree"]


class DraftTree:
    """Which drafted tokens each drafted token sees.

    ``bits``: int32 [trees, T, ceil(T / 32)] on the GPU: token i sees token j where bit ``j % 32`` of word
    ``j // 32`` of row i is set.  ``depths``: int32 [trees, T], the number of a token's ancestors, or
    None.  One tree serves all sequences of a call, or there is one for each.  ``draft_tree`` makes one from parents;
    ``DraftTree(bits)`` takes a table of the caller's own (drafts that are not a tree).

    A tree stays as it was made: its attributes are read-only, as the kernels read as many words as it had then.
    Programs may write into ``bits`` (for another step of a captured graph, say).
    """

    def __init__(self, bits, depths=None):
        if not isinstance(bits, torch.Tensor) or bits.dtype != torch.int32 or bits.dim() != 3 or (
                bits.shape[2] != (bits.shape[1] + 31) // 32):
            raise TypeError("bits must be an int32 tensor [trees, T, ceil(T / 32)]")
        if not bits.is_cuda:
            raise ValueError("bits must be a GPU tensor")
        if not 1 <= bits.shape[1] <= _native.DRAFT_TOKENS or bits.shape[0] < 1:
            raise ValueError(f"a tree has 1 to {_native.DRAFT_TOKENS} tokens; got {tuple(bits.shape)}")
        if not bits[0].is_contiguous():
            raise ValueError("the rows of a tree's bits must lie densely")
        if depths is not None and (not isinstance(depths, torch.Tensor) or depths.dtype != torch.int32 or depths.shape != bits.shape[:2]
                                   or depths.device != bits.device):
            raise ValueError(f"depths must be int32 {tuple(bits.shape[:2])} on the device of bits")
        self._bits, self._depths = bits, depths
        self._trees, self._tokens = bits.shape[:2]

    bits = property(lambda self: self._bits)
    depths = property(lambda self: self._depths)
    trees = property(lambda self: self._trees)
    tokens = property(lambda self: self._tokens)


def draft_tree(parents):
    """The ``DraftTree`` of ``parents``: int32 [T] (one tree for all sequences) or [Z, T] on the GPU.

    ``parents[i]`` is the token before token i on its path, an earlier drafted one (below i); any
    other value, as -1, means the context's last token.  T is at most 512."""
    if not isinstance(parents, torch.Tensor) or parents.dtype != torch.int32 or parents.dim() not in (1, 2):
        raise TypeError("parents must be an int32 tensor [T] or [Z, T]")
    if not parents.is_cuda:
        raise ValueError("parents must be a GPU tensor")
    p = parents if parents.dim() == 2 else parents[None]
    trees, T = p.shape
    if not 1 <= T <= _native.DRAFT_TOKENS or trees < 1:
        raise ValueError(f"a tree has 1 to {_native.DRAFT_TOKENS} tokens; got {tuple(parents.shape)}")
    if T > 1 and p.stride(1) != 1:
        p = p.contiguous()
    bits = torch.empty((trees, T, (T + 31) // 32), dtype=torch.int32, device=p.device)
    depths = torch.empty((trees, T), dtype=torch.int32, device=p.device)
    args = _native.DraftTreeArgs()
    args.struct_size = ctypes.sizeof(args)
    args.parents, args.parents_stride = p.data_ptr(), p.stride(0) if trees > 1 else 0
    args.trees, args.t = trees, T
    args.bits, args.depths = bits.data_ptr(), depths.data_ptr()
    fn, dev = _native.lib().rsfa_draft_tree, p.device.index
    stream = torch._C._cuda_getCurrentRawStream(dev)
    if dev == torch.cuda.current_device():
        st = fn(ctypes.byref(args), stream)
    else:
        with torch.cuda.device(p.device):
            st = fn(ctypes.byref(args), stream)
    _raise_for(st)
    return DraftTree(bits, depths)
