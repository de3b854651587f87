"""A key/value cache held in 4 bits, and attention over it, on MI355X (gfx950).

``Cache4`` keeps the K and V rows of one attention layer as e2m1 codes with a
power-of-two scale for each 32 values (the OCP microscaling formats; 4.25 bits a value),
for sequences [Z], key heads [H] and ``capacity`` slots each:

==============  ==================================================================
``append``      quantises new K and V rows into slots
``read``        the values of slots (what ``attention`` takes as K and V)
``attend``      attention of new queries over the slots in use; on request each slot's
                weight grows by the attention it received
``claim``       slots for the next tokens of a full cache: those of least weight
``evict``       copies the slots of most weight into a smaller cache
==============  ==================================================================

How many slots of a sequence are in use is the caller's: every call takes
``lengths``, an int for all sequences or an int32 GPU tensor [Z] (one for all layers of a
model, advanced by the caller; calls with tensors can be captured into a graph).
An int is checked against the capacity; values of a tensor are on the
device and taken as 0 or the capacity where they lie outside of it.  ``counts`` (int32 [Z])
says how many of a call's T tokens a sequence has, in a padded batch.

All arithmetic runs in ``lib/librsfa.so`` (``rsfa_cache4_*`` in ``include/rsfa.h``),
enqueued on the current stream of the cache's device; there is no other path.
No gradients: the cache is for inference.
"""
import ctypes
import math

import torch

from . import _native
from .flash_attention_forward import _as_kernel_layout, _meets_contract, _raise_for

__all__ = ["Cache4"]

_DTYPES = {torch.float16: _native.DTYPE_F16, torch.bfloat16: _native.DTYPE_BF16}
_HEAD_DIMS = (32, 64, 128, 256)


def _is_int(x):
    return isinstance(x, int) and not isinstance(x, bool)


class Cache4:
    """``Cache4(Z, H, capacity, head_dim, dtype=torch.float16, device="cuda", weights=True)``

    ``dtype``: of the rows that are written and read and of q and o.  Without
    ``weights`` the cache keeps no attention weights (no accumulate, claim or evict).
    The buffers are attributes: k_codes, v_codes (uint8 [Z, H, capacity, D / 2]), k_scales,
    v_scales (uint8 [Z, H, capacity, D / 32]), positions (int32) and weights (float32,
    both [Z, H, capacity]).
    """

    def __init__(self, Z, H, capacity, head_dim, dtype=torch.float16, device="cuda", weights=True):
        if head_dim not in _HEAD_DIMS:
            raise ValueError(f"head_dim must be one of {_HEAD_DIMS}; got {head_dim}")
        if min(Z, H, capacity) < 1:
            raise ValueError(f"Z, H and capacity must be at least 1; got {Z}, {H}, {capacity}")
        if dtype not in _DTYPES:
            raise TypeError(f"unsupported dtype {dtype}; float16 and bfloat16 are supported")

        def empty(width, dt):
            return torch.zeros((Z, H, capacity) + width, dtype=dt, device=device)

        self._take(empty((head_dim // 2,), torch.uint8), empty((head_dim // 32,), torch.uint8),
                   empty((head_dim // 2,), torch.uint8), empty((head_dim // 32,), torch.uint8),
                   empty((), torch.int32), empty((), torch.float32) if weights else None, dtype)

    @classmethod
    def from_buffers(cls, k_codes, k_scales, v_codes, v_scales, positions, weights=None, *, dtype=torch.float16):
        """A cache in buffers of the caller's: rows dense, sequences and heads at any
        strides (the same for K and V, and for positions and weights)."""
        self = cls.__new__(cls)
        self._take(k_codes, k_scales, v_codes, v_scales, positions, weights, dtype)
        return self

    def _take(self, kc, ks, vc, vs, positions, weights, dtype):
        if dtype not in _DTYPES:
            raise TypeError(f"unsupported dtype {dtype}; float16 and bfloat16 are supported")
        if kc.dim() != 4 or 2 * kc.shape[3] not in _HEAD_DIMS or min(kc.shape) < 1:
            raise ValueError(f"codes must be [Z, H, capacity, head_dim / 2] with head_dim one of {_HEAD_DIMS}; "
                             f"got {tuple(kc.shape)}")
        Z, H, C, half = kc.shape
        D = 2 * half
        named = [("k_codes", kc, (Z, H, C, half), torch.uint8), ("v_codes", vc, (Z, H, C, half), torch.uint8),
                 ("k_scales", ks, (Z, H, C, D // 32), torch.uint8), ("v_scales", vs, (Z, H, C, D // 32), torch.uint8),
                 ("positions", positions, (Z, H, C), torch.int32)]
        if weights is not None:
            named.append(("weights", weights, (Z, H, C), torch.float32))
        strides = []
        for name, t, shape, dt in named:
            if tuple(t.shape) != shape or t.dtype != dt:
                raise ValueError(f"{name} must be {dt} {shape}; got {t.dtype} {tuple(t.shape)}")
            if not t.is_cuda or t.device != kc.device:
                raise ValueError(f"{name} must be a GPU tensor on the device of k_codes")
            # strides of dims of size 1 mean nothing
            st = [s if n > 1 else 0 for s, n in zip(t.stride(), t.shape)]
            row = shape[3] if len(shape) == 4 else 1
            if (C > 1 and st[2] != row) or (row > 1 and st[3] != 1):
                raise ValueError(f"{name}: the rows of a sequence and head must lie densely")
            if (Z > 1 and st[0] == 0) or (H > 1 and st[1] == 0):
                raise ValueError(f"{name} is expanded: its sequences and heads must not share memory")
            strides.append(tuple(st[:2]))
        for a, b in ((0, 1), (2, 3)) + (((4, 5),) if weights is not None else ()):
            if strides[a] != strides[b]:
                raise ValueError(f"{named[a][0]} and {named[b][0]} must have the same strides")
        if any(s % 16 for s in strides[0]) or (kc.data_ptr() | vc.data_ptr()) % 16:
            raise ValueError("codes must be 16-byte aligned, with strides that are multiples of 16")
        width = D // 32
        if any(s % width for s in strides[2]) or (ks.data_ptr() | vs.data_ptr()) % width:
            raise ValueError(f"scales must be {width}-byte aligned, with strides that are multiples of {width}")
        self.k_codes, self.k_scales, self.v_codes, self.v_scales = kc, ks, vc, vs
        self.positions, self.weights, self.dtype = positions, weights, dtype
        self.Z, self.H, self.capacity, self.head_dim, self.device = Z, H, C, D, kc.device
        c = _native.Cache4()
        c.k_codes, c.k_scales, c.v_codes, c.v_scales = (t.data_ptr() for t in (kc, ks, vc, vs))
        c.positions = positions.data_ptr()
        c.weights = weights.data_ptr() if weights is not None else None
        c.z, c.h, c.capacity, c.head_dim = Z, H, C, D
        c.code_stride[:], c.scale_stride[:], c.slot_stride[:] = strides[0], strides[2], strides[4]
        c.dtype = _DTYPES[dtype]
        self._c = c

    # -- arguments ----------------------------------------------------------
    def _vector(self, t, name):
        """The address of an int32 GPU tensor [Z] (None: NULL)."""
        if t is None:
            return None
        if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or tuple(t.shape) != (self.Z,):
            raise TypeError(f"{name} must be an int32 tensor [{self.Z}]")
        if t.device != self.device:
            raise ValueError(f"{name} must be on the cache's device")
        if self.Z > 1 and t.stride(0) != 1:
            raise ValueError(f"{name} must be contiguous")
        return t.data_ptr()

    def _lengths(self, args, lengths, extra=0):
        if _is_int(lengths):
            if lengths < 0 or lengths + extra > self.capacity:
                raise ValueError(f"{lengths} + {extra} slots do not fit the capacity of {self.capacity}")
            args.length = lengths
        else:
            args.lengths = self._vector(lengths, "lengths (an int, or a tensor)")

    def _rows(self, x, name, T=None):
        if x.dim() != 4 or x.shape[0] != self.Z or x.shape[3] != self.head_dim:
            raise ValueError(f"{name} must be [{self.Z}, heads, T, {self.head_dim}]; got {tuple(x.shape)}")
        if x.dtype != self.dtype:
            raise TypeError(f"{name} must have the cache's dtype {self.dtype}; got {x.dtype}")
        if x.device != self.device:
            raise ValueError(f"{name} must be on the cache's device")
        return x if x.numel() == 0 else _as_kernel_layout(x)

    def _slots(self, slots, T=None):
        if slots.dtype != torch.int32 or slots.dim() != 3 or slots.shape[:2] != (self.Z, self.H) or (
                T is not None and slots.shape[2] != T):
            raise ValueError(f"slots must be int32 [{self.Z}, {self.H}, {'n' if T is None else T}]; "
                             f"got {slots.dtype} {tuple(slots.shape)}")
        if slots.device != self.device:
            raise ValueError("slots must be on the cache's device")
        return slots.contiguous()

    def _on_device(self, fn, *args):
        if self.device.index == torch.cuda.current_device():
            return fn(*args)
        with torch.cuda.device(self.device):
            return fn(*args)

    def _call(self, fn, args):
        _raise_for(self._on_device(fn, ctypes.byref(args), torch._C._cuda_getCurrentRawStream(self.device.index)))

    # -- rows ---------------------------------------------------------------
    def append(self, k, v, lengths, *, positions=None, counts=None, slots=None):
        """Writes the rows of k, v [Z, H, T, D] (float16 / bfloat16, the cache's dtype).

        Token i of sequence z goes to slot ``lengths[z] + i``, or with ``slots`` (int32
        [Z, H, T], as ``claim`` gives) to ``slots[z, h, i]``; its position is
        ``positions[z] + i`` (int32 [Z]; None: ``lengths[z] + i``), its weight 0.
        Not written: tokens ``i >= counts[z]`` and slots outside the cache
        (-1, say).  A slot that ``slots`` names twice holds the last of its tokens.
        """
        if k.shape != v.shape or k.dim() != 4 or k.shape[1] != self.H:
            raise ValueError(f"k and v must share one shape [{self.Z}, {self.H}, T, {self.head_dim}]; "
                             f"got {tuple(k.shape)} and {tuple(v.shape)}")
        T = k.shape[2]
        args = _native.Cache4RowsArgs()
        args.struct_size = ctypes.sizeof(args)
        self._lengths(args, lengths, 0 if slots is not None or counts is not None else T)
        args.counts = self._vector(counts, "counts")
        args.pos_start = self._vector(positions, "positions")
        if slots is not None:
            slots = self._slots(slots, T)
            args.slots = slots.data_ptr()
        k, v = self._rows(k, "k"), self._rows(v, "v")
        if T == 0:
            return
        args.cache = self._c
        args.k, args.v, args.t = k.data_ptr(), v.data_ptr(), T
        args.k_stride[:], args.v_stride[:] = k.stride(), v.stride()
        self._call(_native.lib().rsfa_cache4_append, args)

    def read(self, start=0, count=None, *, slots=None):
        """(k, v): the values of slots ``start[z] .. start[z] + count - 1`` (an int or an
        int32 tensor [Z]; ``count=None``: to the capacity, for an int), or of ``slots``
        (int32 [Z, H, n]); slots outside the cache read as 0."""
        args = _native.Cache4RowsArgs()
        args.struct_size = ctypes.sizeof(args)
        if slots is not None:
            slots = self._slots(slots)
            args.slots = slots.data_ptr()
            count = slots.shape[2]
        elif _is_int(start):
            if count is None:
                count = self.capacity - start
            if start < 0 or count < 0 or start + count > self.capacity:
                raise ValueError(f"slots {start} .. {start + count - 1} are not within the capacity of {self.capacity}")
            args.length = start
        else:
            if not _is_int(count) or count < 0:
                raise ValueError("read needs a count with a tensor of first slots")
            args.lengths = self._vector(start, "start (an int, or a tensor)")
        k, v = (torch.empty((self.Z, self.H, count, self.head_dim), dtype=self.dtype, device=self.device)
                for _ in range(2))
        if count:
            args.cache = self._c
            args.k, args.v, args.t = k.data_ptr(), v.data_ptr(), count
            args.k_stride[:], args.v_stride[:] = k.stride(), v.stride()
            self._call(_native.lib().rsfa_cache4_read, args)
        return k, v

    # -- attention ----------------------------------------------------------
    def attend(self, q, lengths, causal, sm_scale, *, positions=None, counts=None, accumulate=False,
               return_lse=False, max_length=None, out=None):
        """softmax(q k^T sm_scale) v over the slots in use: ``o``, or ``(o, lse)``.

        q [Z, Hq, T, D] in the cache's dtype, Hq a multiple of H: query head i reads key
        head ``i // (Hq // H)``.  ``lengths`` counts the slots with the tokens of this
        call, if they have been appended.  ``causal``: query token i of sequence z sees the
        slots whose position is at most ``positions[z] + i`` (int32 [Z]; None:
        ``lengths[z] - T + i``, with ``counts`` ``lengths[z] - counts[z] + i``, which is right
        while no slot has been evicted); otherwise all slots in use.  Tokens
        ``i >= counts[z]``, and tokens that see no slot, give 0 (lse -inf).

        ``accumulate`` adds to each slot's weight the attention that it received: the sum of
        its softmax weights over all tokens and the query heads of its group.
        ``max_length``: a bound on the lengths (longer ones are cut to it), which
        sizes the call's workspace and its division of the work; the capacity without one.
        ``lse``: the natural logarithm of each row's sum of exponentials, float32 [Z, Hq, T].
        """
        q_ = self._rows(q, "q")
        Z, Hq, T, D = q.shape
        if Hq == 0 or Hq % self.H:
            raise ValueError(f"query heads ({Hq}) must be a multiple of the cache's ({self.H})")
        if accumulate and self.weights is None:
            raise ValueError("this cache keeps no weights")
        if out is None:
            o = torch.empty_like(q_, memory_format=torch.preserve_format)
            if not _meets_contract(o):
                o = torch.empty(q_.shape, dtype=q_.dtype, device=q_.device)
        else:
            o = out
            if o.shape != q.shape or o.dtype != q.dtype or o.device != q.device or not _meets_contract(o):
                raise ValueError("out must match q's shape, dtype and device and have a unit-stride head dim")
        lse = torch.empty((Z, Hq, T), dtype=torch.float32, device=self.device) if return_lse else None
        args = _native.Cache4AttendArgs()
        args.struct_size = ctypes.sizeof(args)
        self._lengths(args, lengths)
        args.counts = self._vector(counts, "counts")
        args.pos_start = self._vector(positions, "positions")
        if max_length is not None:
            if not _is_int(max_length) or not 1 <= max_length <= self.capacity:
                raise ValueError(f"max_length must be within 1 .. {self.capacity}; got {max_length}")
            if _is_int(lengths) and lengths > max_length:
                raise ValueError(f"length {lengths} is more than max_length {max_length}")
            args.max_length = max_length
        elif _is_int(lengths):
            args.max_length = max(1, lengths)
        scale = float(sm_scale)
        if math.isnan(scale):
            raise ValueError("sm_scale is NaN")
        if T == 0:
            return (o, lse) if return_lse else o
        args.cache = self._c
        args.causal, args.accumulate, args.sm_scale = int(bool(causal)), int(bool(accumulate)), scale
        args.q, args.o, args.lse = q_.data_ptr(), o.data_ptr(), lse.data_ptr() if return_lse else None
        args.heads, args.t = Hq, T
        args.q_stride[:], args.o_stride[:] = q_.stride(), o.stride()
        lib = _native.lib()
        nbytes = self._on_device(lib.rsfa_cache4_attend_workspace_bytes, ctypes.byref(args))
        if nbytes:
            ws = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
            args.workspace, args.workspace_bytes = ws.data_ptr(), nbytes
        self._call(lib.rsfa_cache4_attend, args)
        return (o, lse) if return_lse else o

    # -- eviction -----------------------------------------------------------
    def _evict_args(self, lengths, budget, recent, sinks):
        if self.weights is None:
            raise ValueError("this cache keeps no weights")
        for name, x in (("budget", budget), ("recent", recent), ("sinks", sinks)):
            if not _is_int(x) or x < 0:
                raise ValueError(f"{name} must be an int of at least 0; got {x!r}")
        if recent + sinks > budget:
            raise ValueError(f"recent ({recent}) and sinks ({sinks}) are more than the budget of {budget}")
        args = _native.Cache4EvictArgs()
        args.struct_size = ctypes.sizeof(args)
        args.cache = self._c
        self._lengths(args, lengths)
        args.budget, args.recent, args.sinks = budget, recent, sinks
        return args

    def claim(self, lengths, n, *, budget=None, recent=0, sinks=0):
        """Slots for the next n tokens of each sequence and head: int32 [Z, H, n].

        First the slots ``lengths[z], lengths[z] + 1, ...`` below ``budget`` (None: the
        capacity), then the slots of least weight among those in use (ties: the lowest slot),
        in order of slot; -1 where there is none.  Not given away: slots whose
        position is below ``sinks``, or among the ``recent`` last up to the largest
        position of their sequence and head.  For ``append(..., slots=...)``; the length becomes
        ``min(lengths + n, budget)``.
        """
        budget = self.capacity if budget is None else budget
        if not _is_int(n) or n < 1:
            raise ValueError(f"n must be an int of at least 1; got {n!r}")
        args = self._evict_args(lengths, budget, recent, sinks)
        if not 1 <= budget <= self.capacity:
            raise ValueError(f"budget must be within 1 .. {self.capacity}; got {budget}")
        slots = torch.empty((self.Z, self.H, n), dtype=torch.int32, device=self.device)
        args.n, args.out, args.out_bytes = n, slots.data_ptr(), 4 * slots.numel()
        self._call(_native.lib().rsfa_cache4_claim, args)
        return slots

    def evict(self, into, lengths, *, budget=None, recent=0, sinks=0):
        """Copies the slots of most weight to slots 0, 1, ... of the cache ``into``, in their order.

        Of the ``lengths[z]`` slots in use ``budget`` stay (None: the capacity of
        ``into``): those of least weight go first (ties: the lowest slot), protected ones
        (``recent``, ``sinks``: see ``claim``) after all others.  The length becomes
        ``min(lengths, budget)``; slots of ``into`` from there on keep what they hold.
        """
        if not isinstance(into, Cache4):
            raise TypeError("into must be a Cache4")
        if (into.Z, into.H, into.head_dim, into.dtype, into.device) != (
                self.Z, self.H, self.head_dim, self.dtype, self.device):
            raise ValueError("into must have this cache's sequences, heads, head_dim, dtype and device")
        if into.k_codes.data_ptr() == self.k_codes.data_ptr():
            raise ValueError("into must be another cache")
        budget = into.capacity if budget is None else budget
        args = self._evict_args(lengths, budget, recent, sinks)
        if not 1 <= budget <= into.capacity:
            raise ValueError(f"budget must be within 1 .. {into.capacity}; got {budget}")
        args.into = into._c
        kept = torch.empty((self.Z, self.H, budget), dtype=torch.int32, device=self.device)
        args.out, args.out_bytes = kept.data_ptr(), 4 * kept.numel()
        self._call(_native.lib().rsfa_cache4_evict, args)
