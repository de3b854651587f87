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
Calls that write a cache (append, attend with ``accumulate``, evict into it) and
others on the same cache must run one after another: on one stream, or ordered by
events.  No gradients, of either mode: the cache is for inference.  What a call writes has its
version raised, as torch's in-place operators do.
"""
import ctypes
import math
import struct

import torch
from torch.autograd.graph import increment_version

from . import _native, _overlap
from .flash_attention_forward import _as_kernel_layout, _meets_contract, _raise_for
from .rotary import _has_tangent

__all__ = ["Cache4"]

_DTYPES = {torch.float16: _native.DTYPE_F16, torch.bfloat16: _native.DTYPE_BF16}
_HEAD_DIMS = (32, 64, 128, 256)
_FIXED = frozenset(("k_codes", "k_scales", "v_codes", "v_scales", "positions", "weights", "dtype", "Z", "H", "capacity",
                    "head_dim", "device"))

# A call's argument struct is joined from parts that its tensors' shapes settle,
# kept per cache (`_kept`), and packed addresses: filling the struct field by
# field took a third of a call's host time (append 9.4 -> 6.1 us, attend 9.9 -> 7.4).
_ROWS_K, _ROWS_T, _ROWS_LENGTHS = (getattr(_native.Cache4RowsArgs, f).offset for f in ("k", "t", "lengths"))
_ROWS_KV = struct.Struct("=2Q")  # k, v
_ROWS_TAIL = struct.Struct("=QqQQQ")  # lengths, length, slots, counts, pos_start
assert _ROWS_T - _ROWS_K == _ROWS_KV.size and ctypes.sizeof(_native.Cache4RowsArgs) - _ROWS_LENGTHS == _ROWS_TAIL.size
_AT_Q, _AT_HEADS, _AT_LENGTHS = (getattr(_native.Cache4AttendArgs, f).offset for f in ("q", "heads", "lengths"))
_AT_QO = struct.Struct("=3Q")  # q, o, lse
_AT_TAIL = struct.Struct("=QqqQQfiQQ")  # lengths, length, max_length, counts, pos_start, sm_scale, accumulate, workspace, its bytes
assert _AT_HEADS - _AT_Q == _AT_QO.size and ctypes.sizeof(_native.Cache4AttendArgs) - _AT_LENGTHS == _AT_TAIL.size
_EVICT_LENGTHS = _native.Cache4EvictArgs.lengths.offset
_EVICT_TAIL = struct.Struct("=QqqqqqQQQ")  # lengths, length, n, budget, recent, sinks, out, workspace, its bytes
assert ctypes.sizeof(_native.Cache4EvictArgs) - _EVICT_LENGTHS == _EVICT_TAIL.size
_FUNCTIONS = {}


def _function(name):
    """An entry point that takes its argument struct's bytes."""
    fn = _FUNCTIONS.get(name)
    if fn is None:
        fn = _FUNCTIONS[name] = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_char_p, ctypes.c_void_p)((name, _native.lib()))
    return fn


def _is_int(x):
    return isinstance(x, int) and not isinstance(x, bool)


def _no_gradient(*tensors):
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise RuntimeError("a Cache4 keeps no gradients: call it under torch.no_grad()")
    if _has_tangent(*tensors):
        raise RuntimeError("a Cache4 keeps no gradients, those of forward mode neither: call it with the tensors' primals")


class Cache4:
    """``Cache4(Z, H, capacity, head_dim, dtype=torch.float16, device="cuda", weights=True)``

    ``dtype``: of the rows that are written and read and of q and o.  Without
    ``weights`` the cache keeps no attention weights (no accumulate, claim or evict).
    The buffers are attributes: k_codes, v_codes (uint8 [Z, H, capacity, D / 2]), k_scales,
    v_scales (uint8 [Z, H, capacity, D / 32]), positions (int32) and weights (float32,
    both [Z, H, capacity]).  Programs may write into them (``cache.weights.zero_()``), but
    not put others in their places: the kernels hold their addresses.
    """

    def __setattr__(self, name, value):
        # (cache.weights *= 0.5 works in place, and assigns the same tensor)
        if name in _FIXED and name in self.__dict__ and value is not self.__dict__[name]:
            raise AttributeError(f"{name} of a Cache4 is fixed: the kernels hold the buffers' addresses and sizes "
                                 f"(write into a buffer, as cache.weights.copy_(...), or take from_buffers)")
        object.__setattr__(self, name, value)

    def __delattr__(self, name):
        raise AttributeError(f"{name} of a Cache4 is fixed")

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
            if t.requires_grad:
                raise ValueError(f"{name} must not require a gradient")
            if not t.is_cuda or t.device != kc.device:
                raise ValueError(f"{name} must be a GPU tensor on the device of k_codes")
            # strides of dims of size 1 mean nothing
            st = [s if n > 1 else 0 for s, n in zip(t.stride(), t.shape)]
            row = shape[3] if len(shape) == 4 else 1
            if (C > 1 and st[2] != row) or (row > 1 and st[3] != 1):
                raise ValueError(f"{name}: the rows of a sequence and head must lie densely")
            if _overlap.meets_itself(t, t.dim() - 2):
                raise ValueError(f"{name}: its sequences and heads must not share memory")
            strides.append(tuple(st[:2]))
        for a, b in ((0, 1), (2, 3)) + (((4, 5),) if weights is not None else ()):
            if strides[a] != strides[b]:
                raise ValueError(f"{named[a][0]} and {named[b][0]} must have the same strides")
        if any(s % 16 for s in strides[0]) or (kc.data_ptr() | vc.data_ptr()) % 16:
            raise ValueError("codes must be 16-byte aligned, with strides that are multiples of 16")
        width = D // 32
        if any(s % width for s in strides[2]) or (ks.data_ptr() | vs.data_ptr()) % width:
            raise ValueError(f"scales must be {width}-byte aligned, with strides that are multiples of {width}")
        spans = [(t, *_overlap.span(t)) for _, t, _, _ in named]
        for i, (a, a0, a1) in enumerate(spans):
            for j, (b, b0, b1) in enumerate(spans[:i]):
                if a0 < b1 and b0 < a1 and _overlap.meet(a, b, a.dim() - 2, b.dim() - 2):
                    raise ValueError(f"{named[j][0]} and {named[i][0]} must not share memory")
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
        self._z = torch.Size((Z,))
        self._spans = spans
        self._buffers = tuple(t for _, t, _, _ in named)
        self._kept = {}

    def _keep(self, key, parts):
        if len(self._kept) > 1024:
            self._kept.clear()
        self._kept[key] = parts
        return parts

    # -- arguments ----------------------------------------------------------
    def _vector(self, t, name):
        """The address of an int32 GPU tensor [Z] (None: NULL)."""
        if t is None:
            return 0
        if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.shape != self._z:
            raise TypeError(f"{name} must be an int32 tensor [{self.Z}]")
        if t.device != self.device:
            raise ValueError(f"{name} must be on the cache's device")
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
        return t.data_ptr()

    def _lengths(self, lengths, extra=0):
        """(address, value) of lengths."""
        if _is_int(lengths):
            if lengths < 0 or lengths + extra > self.capacity:
                raise ValueError(f"{lengths} + {extra} slots do not fit the capacity of {self.capacity}")
            return 0, lengths
        return self._vector(lengths, "lengths (an int, or a tensor)"), 0

    def _rows(self, x, name):
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

    def _call(self, name, args):
        _raise_for(self._on_device(_function(name), args, torch._C._cuda_getCurrentRawStream(self.device.index)))

    def _rows_parts(self, k, v, T):
        args = _native.Cache4RowsArgs()
        args.struct_size = ctypes.sizeof(args)
        args.cache, args.t = self._c, T
        args.k_stride[:], args.v_stride[:] = k.stride(), v.stride()
        b = bytes(args)
        return b[:_ROWS_K], b[_ROWS_T:_ROWS_LENGTHS]

    # -- rows ---------------------------------------------------------------
    def append(self, k, v, lengths, *, positions=None, counts=None, slots=None):
        """Writes the rows of k, v [Z, H, T, D] (float16 / bfloat16, the cache's dtype).

        Token i of sequence z goes to slot ``lengths[z] + i``, or with ``slots`` (int32
        [Z, H, T], as ``claim`` gives) to ``slots[z, h, i]``; its position is
        ``positions[z] + i`` (int32 [Z]; None: ``lengths[z] + i``), its weight 0.
        Not written: tokens ``i >= counts[z]`` and slots outside the cache
        (-1, say).  A slot that ``slots`` names twice holds the last of its tokens.
        """
        _no_gradient(k, v)
        key = ("append", k.shape, v.shape, k.stride(), v.stride(), k.dtype, v.dtype, k.device, v.device)
        parts = self._kept.get(key)
        if parts is None or (k.data_ptr() | v.data_ptr()) & 15:
            if k.shape != v.shape or k.dim() != 4 or k.shape[1] != self.H:
                raise ValueError(f"k and v must share one shape [{self.Z}, {self.H}, T, {self.head_dim}]; "
                                 f"got {tuple(k.shape)} and {tuple(v.shape)}")
            k_, v_ = self._rows(k, "k"), self._rows(v, "v")
            parts = self._rows_parts(k_, v_, k.shape[2])
            if k_ is k and v_ is v:
                self._keep(key, parts)
            k, v = k_, v_
        T = k.shape[2]
        at, length = self._lengths(lengths, 0 if slots is not None or counts is not None else T)
        counts, positions = self._vector(counts, "counts"), self._vector(positions, "positions")
        if slots is not None:
            slots = self._slots(slots, T)
        if T:
            self._call("rsfa_cache4_append", b"".join((parts[0], _ROWS_KV.pack(k.data_ptr(), v.data_ptr()), parts[1], _ROWS_TAIL.pack(
                at, length, 0 if slots is None else slots.data_ptr(), counts, positions))))
            increment_version(self._buffers)  # (an earlier operation may have kept them for its gradient)

    def read(self, start=0, count=None, *, slots=None):
        """(k, v): the values of slots ``start[z] .. start[z] + count - 1`` (an int or an
        int32 tensor [Z]; ``count=None``: to the capacity, for an int), or of ``slots``
        (int32 [Z, H, n]); slots outside the cache read as 0."""
        at = length = 0
        if slots is not None:
            slots = self._slots(slots)
            count = slots.shape[2]
        elif _is_int(start):
            if count is None:
                count = self.capacity - start
            if start < 0 or count < 0 or start + count > self.capacity:
                raise ValueError(f"slots {start} .. {start + count - 1} are not within the capacity of {self.capacity}")
            length = start
        else:
            if not _is_int(count) or count < 0:
                raise ValueError("read needs a count with a tensor of first slots")
            at = self._vector(start, "start (an int, or a tensor)")
        k = torch.empty((self.Z, self.H, count, self.head_dim), dtype=self.dtype, device=self.device)
        v = torch.empty_like(k)
        if count:
            key = ("read", count)
            parts = self._kept.get(key) or self._keep(key, self._rows_parts(k, v, count))
            self._call("rsfa_cache4_read", b"".join((parts[0], _ROWS_KV.pack(k.data_ptr(), v.data_ptr()), parts[1], _ROWS_TAIL.pack(
                at, length, 0 if slots is None else slots.data_ptr(), 0, 0))))
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
        ``i >= counts[z]``, and tokens that see no slot, give 0 (lse -inf); so do tokens whose
        visible scores are all -inf (an infinite q), as hidden scores are.  Sums are in 32 bits;
        softmax weights are rounded to the dtype for the product with v, as o is.

        ``accumulate`` adds to each slot's weight the attention that it received: the sum of
        its softmax weights over all tokens and the query heads of its group.
        ``max_length``: a bound on the lengths (longer ones are cut to it), which
        sizes the call's workspace and its division of the work; the capacity without one.
        (With ``accumulate`` and at most 32 rows a key head, tokens times group, the workspace
        holds 4 bytes for each row and slot, up to 4 GiB.)
        ``lse``: the natural logarithm of each row's sum of exponentials, float32 [Z, Hq, T].
        """
        _no_gradient(q) if out is None else _no_gradient(q, out)
        key = ("attend", q.shape, q.stride(), q.dtype, q.device, bool(causal), None if out is None else out.stride())
        parts = self._kept.get(key)
        if parts is None or out is not None or q.data_ptr() & 15:
            q_ = self._rows(q, "q")
            if q.shape[1] == 0 or q.shape[1] % self.H:
                raise ValueError(f"query heads ({q.shape[1]}) must be a multiple of the cache's ({self.H})")
            if out is None:
                o = torch.empty_like(q_)
                if not _meets_contract(o):
                    o = torch.empty(q_.shape, dtype=q_.dtype, device=q_.device)
            else:
                o = out
                if o.shape != q.shape or o.dtype != q.dtype or o.device != q.device or not _meets_contract(o):
                    raise ValueError("out must match q's shape, dtype and device and have a unit-stride head dim")
                if o.numel() and _overlap.meets_itself(o):
                    raise ValueError("the rows of out must not share memory")
                if o.numel() and _overlap.meet(o, q_):  # (a copy of q meets nothing)
                    raise ValueError("out must not share memory with q")
            args = _native.Cache4AttendArgs()
            args.struct_size = ctypes.sizeof(args)
            args.cache, args.causal = self._c, int(bool(causal))
            args.heads, args.t = q.shape[1], q.shape[2]
            args.q_stride[:], args.o_stride[:] = q_.stride(), o.stride()
            b = bytes(args)
            parts = (b[:_AT_Q], b[_AT_HEADS:_AT_LENGTHS], {})
            if q_ is q and out is None:
                self._keep(key, parts)
        else:
            q_ = q
            o = torch.empty_like(q)
        lse = torch.empty(q.shape[:3], dtype=torch.float32, device=self.device) if return_lse else None
        if accumulate and self.weights is None:
            raise ValueError("this cache keeps no weights")
        at, length = self._lengths(lengths)
        if max_length is not None:
            if not _is_int(max_length) or not 1 <= max_length <= self.capacity:
                raise ValueError(f"max_length must be within 1 .. {self.capacity}; got {max_length}")
            if length > max_length:
                raise ValueError(f"length {length} is more than max_length {max_length}")
        else:
            max_length = 0 if at else max(1, length)
        counts, positions = self._vector(counts, "counts"), self._vector(positions, "positions")
        scale = float(sm_scale)
        if math.isnan(scale):
            raise ValueError("sm_scale is NaN")
        if q.numel() == 0:
            return (o, lse) if return_lse else o
        accumulate = int(bool(accumulate))
        head = b"".join((parts[0], _AT_QO.pack(q_.data_ptr(), o.data_ptr(), lse.data_ptr() if return_lse else 0), parts[1]))
        nbytes = parts[2].get((max_length, accumulate))
        if nbytes is None:
            tail = _AT_TAIL.pack(at, length, max_length, counts, positions, 0.0, accumulate, 0, 0)
            args = _native.Cache4AttendArgs.from_buffer_copy(head + tail)
            nbytes = self._on_device(_native.lib().rsfa_cache4_attend_workspace_bytes, ctypes.byref(args))
            if at:  # (an int's bound changes from call to call)
                parts[2][max_length, accumulate] = nbytes
        ws = torch.empty(nbytes, dtype=torch.uint8, device=self.device) if nbytes else None
        self._call("rsfa_cache4_attend", head + _AT_TAIL.pack(at, length, max_length, counts, positions, scale, accumulate,
                                                              ws.data_ptr() if nbytes else 0, nbytes))
        if out is not None:
            increment_version(out)
        if accumulate:
            increment_version(self.weights)
        return (o, lse) if return_lse else o

    # -- eviction -----------------------------------------------------------
    def _evict_call(self, name, into, lengths, n, budget, recent, sinks, out):
        if self.weights is None:
            raise ValueError("this cache keeps no weights")
        for what, x in (("budget", budget), ("recent", recent), ("sinks", sinks)):
            if not _is_int(x) or x < 0:
                raise ValueError(f"{what} must be an int of at least 0; got {x!r}")
        limit = self.capacity if into is None else into.capacity
        if not 1 <= budget <= limit:
            raise ValueError(f"budget must be within 1 .. {limit}; got {budget}")
        if recent + sinks > budget:
            raise ValueError(f"recent ({recent}) and sinks ({sinks}) are more than the budget of {budget}")
        at, length = self._lengths(lengths)
        parts = self._kept.get("claim") if into is None else None
        if parts is None:
            args = _native.Cache4EvictArgs()
            args.struct_size = ctypes.sizeof(args)
            args.cache = self._c
            if into is not None:
                args.into = into._c
            parts = (bytes(args)[:_EVICT_LENGTHS], {})
            if into is None:
                self._keep("claim", parts)
        head, sizes = parts
        nbytes = sizes.get(budget)
        if nbytes is None:
            args = _native.Cache4EvictArgs.from_buffer_copy(head + _EVICT_TAIL.pack(0, 0, 1, budget, 0, 0, 0, 0, 0))
            nbytes = sizes[budget] = _native.lib().rsfa_cache4_evict_workspace_bytes(ctypes.byref(args), 0 if into is None else 1)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=self.device) if nbytes else None
        self._call(name, head + _EVICT_TAIL.pack(at, length, n, budget, recent, sinks, out, ws.data_ptr() if nbytes else 0, nbytes))

    def claim(self, lengths, n, *, budget=None, recent=0, sinks=0):
        """Slots for the next n tokens of each sequence and head: int32 [Z, H, n].

        First the slots ``lengths[z], lengths[z] + 1, ...`` below ``budget`` (None: the
        capacity), then the slots of least weight among those in use (ties: the lowest slot),
        in order of slot; -1 where there is none.  Not given away: slots whose
        position is below ``sinks``, or among the ``recent`` last up to the largest
        position of their sequence and head.  For ``append(..., slots=...)``; the length becomes
        ``min(lengths + n, budget)``.
        """
        if not _is_int(n) or n < 1:
            raise ValueError(f"n must be an int of at least 1; got {n!r}")
        if n > 1 << 30:
            raise ValueError(f"n must be at most 2^30; got {n}")
        slots = torch.empty((self.Z, self.H, n), dtype=torch.int32, device=self.device)
        self._evict_call("rsfa_cache4_claim", None, lengths, n, self.capacity if budget is None else budget, recent, sinks,
                         slots.data_ptr())
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
        for a, a0, a1 in self._spans:
            for b, b0, b1 in into._spans:
                if a0 < b1 and b0 < a1 and _overlap.meet(a, b, a.dim() - 2, b.dim() - 2):
                    raise ValueError("into must not share memory with this cache")
        self._evict_call("rsfa_cache4_evict", into, lengths, 1, into.capacity if budget is None else budget, recent, sinks, 0)
        increment_version(into._buffers)
