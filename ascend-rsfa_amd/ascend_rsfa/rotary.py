"""Rotary positions on q and k, forward and backward, on MI355X (gfx950).

``rotary_plan`` holds a model's frequencies; ``rotary`` turns q and k (in one
launch) by the angles of their tokens' positions, ahead of ``attention`` or of
a ``Cache4``; ``rotary_`` does it in place.  Pair i of a head at position p is
turned by ``p * plan.frequencies[i]`` radians and scaled by ``plan.amplitude``:

==================  =========================================================
``layout``          pairs of the first R = ``rotary_dim`` values of a head
==================  =========================================================
``"half"``          (x[i], x[i + R/2])
``"interleaved"``   (x[2i], x[2i + 1])
==================  =========================================================

Values from R on are copied.  Angles are reduced in 64 bits, so positions may
be as large as a text gets; each output is rounded once.  All arithmetic runs in
``lib/librsfa.so`` (``rsfa_rotary`` in ``include/rsfa.h``), on the current
stream of the tensors' device; there is no other path.
"""
import ctypes
import functools
import math
import struct
import threading

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from . import _native, _overlap
from .flash_attention_forward import _raise_for

__all__ = ["RotaryPlan", "rotary_plan", "rotary", "rotary_"]

_DTYPES = {torch.float16: _native.DTYPE_F16, torch.bfloat16: _native.DTYPE_BF16, torch.float32: _native.DTYPE_F32}
_LAYOUTS = ("half", "interleaved")

# A call's argument struct is joined from parts that its tensors' shapes settle, kept with
# the plan, and packed addresses.
_X, _Z, _POS, _POS_STRIDE, _START, _TURNS = (
    getattr(_native.RotaryArgs, f).offset for f in ("x", "z", "positions", "pos_stride", "start", "turns"))
_XY, _ONE, _NUMBER = struct.Struct("=4Q"), struct.Struct("=Q"), struct.Struct("=q")
assert _Z - _X == _XY.size and _POS_STRIDE - _POS == _ONE.size and _TURNS - _START == _NUMBER.size
_FUNCTION = None

# Frequencies on devices whose plans are gone: launches on any stream may still read them, and freed
# memory is given out again on the stream of the plan's first call. They wait for many, and then for the devices.
_DEAD, _DEAD_MOST, _DEAD_LOCK = [], 256, threading.Lock()


def _bury():
    with _DEAD_LOCK:
        n = len(_DEAD)
        if n >= _DEAD_MOST:
            for device in {t.device for t in _DEAD[:n]}:
                torch.cuda.synchronize(device)
            del _DEAD[:n]


def _function():
    """rsfa_rotary, taking its argument struct's bytes."""
    global _FUNCTION
    if _FUNCTION is None:
        _FUNCTION = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_char_p, ctypes.c_void_p)(("rsfa_rotary", _native.lib()))
    return _FUNCTION


def _has_tangent(*xs):
    """Whether a tensor carries a derivative of forward mode (no grad mode hides it)."""
    return getattr(forward_ad, "_current_level", 0) >= 0 and any(
        x is not None and forward_ad.unpack_dual(x).tangent is not None for x in xs)


class RotaryPlan:
    """Frequencies (float64, radians a position, [R/2], on the CPU), amplitude and layout.

    A plan stays as it was made (rotary_plan gives one plan to all callers of the same
    arguments): its attributes are read-only, ``frequencies`` is a copy.  Programs keep a plan
    as long as a captured graph that uses it, as they keep the graph's tensors."""

    def __init__(self, frequencies, layout="half", amplitude=1.0):
        f = torch.as_tensor(frequencies, dtype=torch.float64, device="cpu")
        if (f.requires_grad and torch.is_grad_enabled()) or _has_tangent(f):
            raise RuntimeError("a plan's frequencies are constants: no gradient reaches them (detach them)")
        f = f.detach().contiguous().clone()
        if f.dim() != 1 or f.numel() < 1 or not bool(torch.isfinite(f).all()):
            raise ValueError("frequencies must be a vector of finite numbers, one for each pair")
        if layout not in _LAYOUTS:
            raise ValueError(f"layout must be one of {_LAYOUTS}; got {layout!r}")
        if not math.isfinite(amplitude):
            raise ValueError("amplitude must be finite")
        self._frequencies = f
        self._layout = layout
        self._amplitude = float(amplitude)
        self._rotary_dim = 2 * f.numel()
        self._turns = {}
        self._kept = {}

    def __reduce__(self):  # (what is kept holds addresses of this process, of memory that a copy does not keep alive)
        return type(self), (self.frequencies, self.layout, self.amplitude)

    frequencies = property(lambda self: self._frequencies.clone())
    layout = property(lambda self: self._layout)
    amplitude = property(lambda self: self._amplitude)
    rotary_dim = property(lambda self: self._rotary_dim)

    def __del__(self, dead=_DEAD):
        dead.extend(self.__dict__.get("_turns", {}).values())

    def turns(self, device):
        """Turns a position of each pair, on `device` ("cuda": the current one)."""
        device = torch.device(device)
        if device.type == "cuda" and device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        t = self._turns.get(device)
        if t is None:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("call plan.turns(device) (or rotary) once before capturing a graph")
            _bury()
            t = (self._frequencies / (2.0 * math.pi)).to(device)
            # (other streams may use it at once)
            torch.cuda.current_stream(device).synchronize()
            self._turns[device] = t
        return t


def rotary_plan(rotary_dim, *, base=10000.0, layout="half", scaling=None, factor=1.0, original_length=None,
                low=1.0, high=32.0, amplitude=1.0):
    """A ``RotaryPlan`` of frequencies base^(-2i/R), scaled for long contexts:

    ``scaling=None``: as they are.  ``"linear"``: divided by ``factor``.  ``"ntk"``: the base times
    factor^(R/(R-2)), which divides the slowest frequency by ``factor`` and keeps
    the fastest.  ``"by_parts"``: pairs that turn less than ``low`` times within
    ``original_length`` positions are divided by ``factor``, those that turn more than
    ``high`` times kept, with a linear ramp between.  ``amplitude`` scales the
    turned values (by_parts plans often take 0.1 ln(factor) + 1).
    """
    # (plans are constants: the same arguments give the same one; tensors and the like by what they hold now)
    dim, *numbers = (x if x is None or type(x) in (int, float) else float(x)
                     for x in (rotary_dim, base, factor, original_length, low, high, amplitude))
    return _plan(dim, layout, scaling, *numbers)


@functools.lru_cache(maxsize=64)
def _plan(rotary_dim, layout, scaling, base, factor, original_length, low, high, amplitude):
    R = int(rotary_dim)
    if R != rotary_dim or R < 2 or R % 2:
        raise ValueError(f"rotary_dim must be an even number of at least 2; got {rotary_dim}")
    if not (base > 0 and math.isfinite(base)):
        raise ValueError("base must be positive")
    if not (factor > 0 and math.isfinite(factor)):
        raise ValueError("factor must be positive")
    if scaling not in (None, "linear", "ntk", "by_parts"):
        raise ValueError(f"scaling must be None, 'linear', 'ntk' or 'by_parts'; got {scaling!r}")
    if scaling == "ntk":
        if R == 2:
            raise ValueError("ntk scaling needs rotary_dim of at least 4")
        base = base * factor ** (R / (R - 2.0))
    f = base ** (-2.0 * torch.arange(R // 2, dtype=torch.float64, device="cpu") / R)
    if scaling == "linear":
        f = f / factor
    elif scaling == "by_parts":
        if original_length is None or original_length < 1 or not low < high:
            raise ValueError("by_parts scaling needs original_length >= 1 and low < high")
        turns = original_length * f / (2.0 * math.pi)
        keep = ((turns - low) / (high - low)).clamp(0.0, 1.0)
        f = (1.0 - keep) * f / factor + keep * f
    return RotaryPlan(f, layout, amplitude)


def _check(x, name):
    if x.dim() != 4:
        raise ValueError(f"{name} must be 4-D [Z, H, N, D]; got {tuple(x.shape)}")
    if x.dtype not in _DTYPES:
        raise TypeError(f"unsupported dtype {x.dtype}; float16, bfloat16 and float32 are supported")
    if not x.is_cuda:
        raise ValueError(f"{name} must be a GPU tensor")


def _like(x):
    """An output for x: in x's layout where that is dense, or contiguous."""
    y = torch.empty_like(x)
    return y if y.stride(3) == 1 else torch.empty(x.shape, dtype=x.dtype, device=x.device)


def _key(q, k, positions, inverse):
    """What a call's argument struct depends on, but for addresses."""
    return (q.shape, q.stride(), q.dtype, q.device, None if k is None else (k.shape, k.stride(), k.dtype, k.device),
            None if isinstance(positions, int) else (positions.shape, positions.stride(), positions.dtype, positions.device),
            inverse)


def _parts(xs, ys, positions, plan, inverse):
    x = xs[0]
    Z, _, N, D = x.shape
    args = _native.RotaryArgs()
    args.struct_size = ctypes.sizeof(_native.RotaryArgs)
    args.dtype = _DTYPES[x.dtype]
    args.z, args.n, args.head_dim, args.rotary_dim = Z, N, D, plan.rotary_dim
    for i, (a, b) in enumerate(zip(xs, ys)):
        args.heads[i] = a.shape[1]
        args.x_stride[i][:] = a.stride()
        args.y_stride[i][:] = b.stride()
    flags = (_native.ROTARY_INTERLEAVED if plan.layout == "interleaved" else 0) | (
        _native.ROTARY_INVERSE if inverse else 0)
    if not isinstance(positions, int):
        st = positions.stride()
        args.pos_stride[:] = (st[0] if positions.dim() == 2 and positions.shape[0] > 1 else 0, st[-1])
        if positions.dtype == torch.int64:
            flags |= _native.ROTARY_POS64
    args.turns = plan.turns(x.device).data_ptr()
    args.amplitude = plan.amplitude
    args.flags = flags
    b = bytes(args)
    return b[:_X], b[_Z:_POS], b[_POS_STRIDE:_START], b[_TURNS:]


def _launch(parts, xs, ys, positions):
    """ys[i] = xs[i] turned; xs: one or two tensors."""
    head, sizes, strides, tail = parts
    two = len(xs) > 1
    start = isinstance(positions, int)
    args = b"".join((head, _XY.pack(xs[0].data_ptr(), xs[1].data_ptr() if two else 0, ys[0].data_ptr(), ys[1].data_ptr() if two else 0),
                     sizes, _ONE.pack(0 if start else positions.data_ptr()), strides, _NUMBER.pack(positions if start else 0), tail))
    dev = xs[0].device.index
    stream = torch._C._cuda_getCurrentRawStream(dev)
    if dev == torch.cuda.current_device():
        st = _function()(args, stream)
    else:
        with torch.cuda.device(dev):
            st = _function()(args, stream)
    _raise_for(st)


def _unit(x):
    return x if x.stride(3) == 1 else x.contiguous()


class _Rotary(torch.autograd.Function):

    @staticmethod
    def forward(ctx, q, k, positions, plan, inverse):
        ctx.plan, ctx.positions, ctx.inverse = plan, positions, inverse
        # positions may be changed by the program before the backward pass
        if not isinstance(positions, int):
            ctx.positions = None
            ctx.save_for_backward(positions)
            ctx.save_for_forward(positions)
        return _forward(q, k, positions, plan, inverse)

    @staticmethod
    def jvp(ctx, tq, tk, *_):  # linear: tangents turn as values do
        positions = ctx.saved_tensors[0] if ctx.positions is None else ctx.positions
        return _turn(tq, tk, positions, ctx.plan, ctx.inverse)

    @staticmethod
    def backward(ctx, gq, gk=None):
        positions = ctx.saved_tensors[0] if ctx.positions is None else ctx.positions
        if not ctx.needs_input_grad[0]:
            gq = None
        if not ctx.needs_input_grad[1]:
            gk = None
        if gq is not None and gk is not None:
            gq, gk = _turn(gq, gk, positions, ctx.plan, not ctx.inverse)
        elif gq is not None:
            gq = _turn(gq, None, positions, ctx.plan, not ctx.inverse)
        elif gk is not None:
            gk = _turn(gk, None, positions, ctx.plan, not ctx.inverse)
        return gq, gk, None, None, None


def _turn(q, k, positions, plan, inverse):
    if (torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad))) or _has_tangent(q, k):
        return _Rotary.apply(q, k, positions, plan, inverse)
    return _forward(q, k, positions, plan, inverse)


def _forward(q, k, positions, plan, inverse):
    key = _key(q, k, positions, inverse)
    parts = plan._kept.get(key)
    if parts is not None:  # (tensors of this key were taken as they are)
        y = torch.empty_like(q)
        if k is None:
            _launch(parts, (q,), (y,), positions)
            return y
        w = torch.empty_like(k)
        _launch(parts, (q, k), (y, w), positions)
        return y, w
    _checked(q, k, positions, plan)
    xs = [_unit(q)] if k is None else [_unit(q), _unit(k)]
    ys = [_like(x) for x in xs]
    some = [(x, y) for x, y in zip(xs, ys) if x.numel()]
    if some:
        parts = _parts([x for x, _ in some], [y for _, y in some], positions, plan, inverse)
        # kept where q and k go in as they are and empty_like gives their outputs
        if len(some) == len(xs) and xs[0] is q and xs[-1] is (q if k is None else k) and all(
                y.stride() == torch.empty_like(x, device="meta").stride() for x, y in some):
            if len(plan._kept) > 1024:
                plan._kept.clear()
            plan._kept[key] = parts
        _launch(parts, [x for x, _ in some], [y for _, y in some], positions)
    return ys[0] if k is None else tuple(ys)


def _checked(q, k, positions, plan):
    if not isinstance(plan, RotaryPlan):
        raise TypeError("plan must be a RotaryPlan (rotary_plan(...))")
    _check(q, "q")
    if k is not None:
        _check(k, "k")
        if k.dtype != q.dtype or k.device != q.device:
            raise TypeError("q and k must have one dtype and device")
        if k.shape[0] != q.shape[0] or k.shape[2:] != q.shape[2:]:
            raise ValueError(f"q and k must share Z, N and D; got {tuple(q.shape)} and {tuple(k.shape)}")
    if plan.rotary_dim > q.shape[3]:
        raise ValueError(f"the plan turns {plan.rotary_dim} values of a head; the head dim is {q.shape[3]}")
    if isinstance(positions, bool) or not isinstance(positions, (int, torch.Tensor)):
        raise TypeError("positions must be an int (the first token's) or an int32/int64 tensor [N] or [Z, N]")
    if isinstance(positions, int) and abs(positions) >= 1 << 53:
        raise ValueError("positions must be below 2^53")
    if isinstance(positions, torch.Tensor):
        Z, N = q.shape[0], q.shape[2]
        if positions.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"positions must be int32 or int64; got {positions.dtype}")
        if positions.device != q.device:
            raise ValueError("positions must be on q's device")
        if tuple(positions.shape) not in ((N,), (Z, N), (1, N)):
            raise ValueError(f"positions must be [N] or [Z, N]; got {tuple(positions.shape)}")


def rotary(q, k, positions, plan):
    """(q', k') turned by their positions; ``k=None``: q' alone.

    q [Z, Hq, N, D] and k [Z, Hk, N, D] (float16, bfloat16 or float32, any
    strides); ``positions``: the first token's position (an int), or a tensor [N]
    or [Z, N] of int32 or int64.  Differentiable in q and k, in reverse and in
    forward mode: the gradient is the same turn backwards, a tangent turns as its value does.
    """
    if not isinstance(plan, RotaryPlan):
        raise TypeError("plan must be a RotaryPlan (rotary_plan(...))")
    if isinstance(positions, bool) or not isinstance(positions, (int, torch.Tensor)):
        raise TypeError("positions must be an int (the first token's) or an int32/int64 tensor [N] or [Z, N]")
    if isinstance(positions, int) and abs(positions) >= 1 << 53:
        raise ValueError("positions must be below 2^53")
    return _turn(q, k, positions, plan, False)


def rotary_(q, k, positions, plan):
    """``rotary`` in place (inference); the values beyond ``rotary_dim`` are not touched.  q and k (parts of one
    fused tensor, say) must not share elements."""
    _checked(q, k, positions, plan)
    for x in (q, k):
        if x is None:
            continue
        if (x.requires_grad and torch.is_grad_enabled()) or _has_tangent(x):
            raise RuntimeError("rotary_ works in place and keeps no gradient; use rotary")
        if x.stride(3) != 1 and x.shape[3] > 1:
            raise ValueError("rotary_ needs a unit stride in the head dim")
        if x.numel() and _overlap.meets_itself(x):
            raise ValueError("rotary_ cannot write to a tensor whose rows share memory, as an expanded one's do")
    xs = [x for x in (q, k) if x is not None and x.numel()]
    if len(xs) == 2 and _overlap.meet(q, k):
        raise ValueError("q and k must not share memory")
    if xs:
        _launch(_parts(xs, xs, positions, plan, False), xs, xs, positions)
        increment_version(xs)  # (an earlier operation may have kept them for its gradient)
    return q if k is None else (q, k)
