"""Cross attention on MI355X (gfx950): queries over keys of another length, an encoder's states say.

``cross_attention(q, k, v, sm_scale, lengths)`` is ``softmax(q k^T sm_scale) v`` without a mask
but for the lengths of a padded batch.  A training step differentiates it; a decoding step calls it with one
token or a few.

All arithmetic runs in ``lib/librsfa.so`` (``rsfa_cross_*`` in ``include/rsfa.h``), enqueued on the
current stream of the tensors' device; there is no other path.
"""
import ctypes
import math
import struct

import torch
from torch.autograd.function import once_differentiable

from . import _native
from .flash_attention_forward import _as_kernel_layout, _meets_contract, _raise_for
from .rotary import _has_tangent

__all__ = ["cross_attention"]

_DTYPES = {torch.float16: _native.DTYPE_F16, torch.bfloat16: _native.DTYPE_BF16}
_HEAD_DIMS = (32, 64, 128, 256)

# What a call does is settled by its tensors' shapes, strides, types and devices, and kept by them: a _Plan holds the
# argument structs but for their addresses, so that a call is one lookup and a struct joined from bytes (a training step's
# two passes run in two threads, each of which finds the other's objects far away).
_F, _B = _native.CrossArgs, _native.CrossBwdArgs
_FWD_PTRS = struct.Struct("=5Q")  # q, k, v, o, lse
_BWD_PTRS = struct.Struct("=10Q")  # q, k, v, o, lse, grad_o, grad_lse, grad_q, grad_k, grad_v
_TAIL = struct.Struct("=QfIQQ")  # lengths, sm_scale, reserved, workspace, its bytes
assert _F.z.offset - _F.q.offset == _FWD_PTRS.size and ctypes.sizeof(_F) - _F.lengths.offset == _TAIL.size
assert _B.z.offset - _B.q.offset == _BWD_PTRS.size and ctypes.sizeof(_B) - _B.lengths.offset == _TAIL.size
_PLANS = {}
_FUNCTIONS = {}


def _function(name):
    """An entry point that takes its argument struct's bytes."""
    fn = _FUNCTIONS.get(name)
    if fn is None:
        fn = _FUNCTIONS[name] = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_char_p, ctypes.c_void_p)((name, _native.lib()))
    return fn


def _on_device(index, fn, *args):
    if index == torch.cuda.current_device():
        return fn(*args)
    with torch.cuda.device(index):
        return fn(*args)


def _launch(index, name, args):
    fn, stream = _FUNCTIONS.get(name) or _function(name), torch._C._cuda_getCurrentRawStream(index)
    status = fn(args, stream) if index == torch.cuda.current_device() else _on_device(index, fn, args, stream)
    if status:
        _raise_for(status)


def _empty_rows(t):
    """(an output like t, whose rows the kernels can write, whether empty_like gives it)."""
    o = torch.empty_like(t)
    return (o, True) if _meets_contract(o) else (torch.empty(t.shape, dtype=t.dtype, device=t.device), False)


def _struct(kind, tensors, q, k, workspace):
    """(the struct's bytes before and after its addresses, workspace bytes) for {name: tensor}."""
    args = kind()
    args.struct_size, args.dtype = ctypes.sizeof(args), _DTYPES[q.dtype]
    args.z, args.heads, args.t, args.head_dim = q.shape
    args.key_heads, args.n = k.shape[1], k.shape[2]
    for name, t in tensors.items():
        if t is not None:
            getattr(args, name + "_stride")[:] = t.stride()
    nbytes = _on_device(q.device.index, getattr(_native.lib(), workspace), ctypes.byref(args))
    b = bytes(args)
    return b[:kind.q.offset], b[kind.z.offset:kind.lengths.offset], nbytes


class _Plan:
    """A call's argument structs, for tensors in the kernels' layout that are not empty."""

    __slots__ = ("index", "head", "sizes", "nbytes", "like", "kinds", "backward")

    def __init__(self, q, k, v):
        o, self.like = _empty_rows(q)
        self.index = q.device.index
        self.kinds = tuple((t.shape, t.dtype, t.device) for t in (q, k, v, q, q))  # of q, k, v, o and the gradient of o
        self.head, self.sizes, self.nbytes = _struct(_F, {"q": q, "k": k, "v": v, "o": o}, q, k, "rsfa_cross_fwd_workspace_bytes")
        self.backward = {}


def _forward(plan, q, k, v, scale, lengths, want_lse):
    """(o, lse or None)."""
    o = torch.empty_like(q) if plan.like else torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty(q.shape[:3], dtype=torch.float32, device=q.device) if want_lse else None
    nbytes = plan.nbytes
    ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
    _launch(plan.index, "rsfa_cross_fwd", b"".join((
        plan.head, _FWD_PTRS.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), lse.data_ptr() if want_lse else 0), plan.sizes,
        _TAIL.pack(0 if lengths is None else lengths.data_ptr(), scale, 0, ws.data_ptr() if nbytes else 0, nbytes))))
    return o, lse


def _check_saved(plan, rows, stats, lengths):
    """q, k, v, o and the gradient of o; lse and its gradient; lengths: of the shapes, types and device that the kernels are told."""
    shape, _, device = plan.kinds[0]
    want = plan.kinds + (((shape[:3], torch.float32, device),) * 2) + ((shape[:1], torch.int32, device),)
    for t, (of, dtype, on) in zip((*rows, *stats, lengths), want):
        if t is not None and (t.shape != of or t.dtype != dtype or t.device != on):
            raise RuntimeError(f"a saved tensor or a gradient of {dtype} {tuple(of)} on {on} came back as {t.dtype} {tuple(t.shape)} on {t.device}")


def _backward(plan, q, k, v, o, lse, go, glse, scale, lengths, needs):
    """The gradients of q, k and v, those that ``needs`` names (None for the others)."""
    if go is None:
        go = torch.zeros_like(o)
    if glse is not None:
        glse = glse.contiguous()
    # Saved tensors need not be those that were saved: a hook (one that offloads them, say) may bring back others, of other
    # strides.  So all that the struct says of them is looked at, and tensors whose key is kept differ in their addresses only.
    key = (needs, q.stride(), k.stride(), v.stride(), o.stride(), go.stride(), lse.stride(), q.shape, k.shape, v.shape, o.shape, go.shape,
           lse.shape, q.dtype, k.dtype, v.dtype, o.dtype, go.dtype, lse.dtype, q.device, k.device, v.device, o.device, go.device, lse.device,
           None if glse is None else (glse.shape, glse.dtype, glse.device),
           None if lengths is None else (lengths.shape, lengths.stride(), lengths.dtype, lengths.device))
    kept = plan.backward.get(key)
    if kept is None or (q.data_ptr() | k.data_ptr() | v.data_ptr() | o.data_ptr() | go.data_ptr()) & 15:
        came = (q, k, v, o, go, lse, lengths)
        _check_saved(plan, came[:5], (lse, glse), lengths)
        q, k, v, o, go = (_as_kernel_layout(t) for t in came[:5])
        lse, lengths = lse.contiguous(), None if lengths is None else lengths.contiguous()
        grads = [_empty_rows(t) if need else (None, True) for t, need in zip((q, k, v), needs)]
        like = all(x for _, x in grads)
        grads = [g for g, _ in grads]
        kept = _struct(_B, {"q": q, "k": k, "v": v, "o": o, "grad_o": go, "grad_q": grads[0], "grad_k": grads[1], "grad_v": grads[2]},
                       q, k, "rsfa_cross_bwd_workspace_bytes")
        if like and all(a is b for a, b in zip(came, (q, k, v, o, go, lse, lengths))):
            if len(plan.backward) > 64:
                plan.backward.clear()
            plan.backward[key] = kept
    else:
        grads = [torch.empty_like(t) if need else None for t, need in zip((q, k, v), needs)]
    head, sizes, nbytes = kept
    ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
    ptrs = [0 if t is None else t.data_ptr() for t in (q, k, v, o, lse, go, glse, *grads)]
    _launch(plan.index, "rsfa_cross_bwd", b"".join((
        head, _BWD_PTRS.pack(*ptrs), sizes, _TAIL.pack(0 if lengths is None else lengths.data_ptr(), scale, 0, ws.data_ptr(), nbytes))))
    return grads


def _check(q, k, v, lengths):
    if q.dim() != 4 or k.dim() != 4 or v.shape != k.shape or k.shape[0] != q.shape[0] or k.shape[3] != q.shape[3]:
        raise ValueError(f"q must be [Z, heads, T, D], k and v [Z, key heads, N, D]; got {tuple(q.shape)}, {tuple(k.shape)}, "
                         f"{tuple(v.shape)}")
    if q.shape[3] not in _HEAD_DIMS:
        raise ValueError(f"the head dim must be one of {_HEAD_DIMS}; got {q.shape[3]}")
    if k.shape[1] == 0 or q.shape[1] % k.shape[1]:
        raise ValueError(f"query heads ({q.shape[1]}) must be a multiple of the key heads ({k.shape[1]})")
    if not (q.dtype == k.dtype == v.dtype):
        raise TypeError("q, k and v must have the same dtype")
    if q.dtype not in _DTYPES:
        raise TypeError(f"unsupported dtype {q.dtype}; float16 and bfloat16 are supported")
    if not q.is_cuda or not (q.device == k.device == v.device):
        raise ValueError("q, k and v must be GPU tensors on one device")
    if lengths is not None:
        if not isinstance(lengths, torch.Tensor) or lengths.dtype != torch.int32 or lengths.shape != q.shape[:1]:
            raise TypeError(f"lengths must be an int32 tensor [{q.shape[0]}]")
        if lengths.device != q.device:
            raise ValueError("lengths must be on the device of q")


class _CrossAttention(torch.autograd.Function):

    @staticmethod
    def forward(ctx, q, k, v, plan, sm_scale, lengths, return_lse):
        if plan is None:
            o, lse = _nothing(q)
        else:
            o, lse = _forward(plan, q, k, v, sm_scale, lengths, True)
        ctx.save_for_backward(q, k, v, o, lse, lengths)
        ctx.plan, ctx.sm_scale = plan, sm_scale
        if not return_lse:
            return o
        ctx.set_materialize_grads(False)
        return o, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, go, glse=None):
        q, k, v, o, lse, lengths = ctx.saved_tensors
        if go is None and glse is None:
            return (None,) * 7
        needs = ctx.needs_input_grad[:3]
        if ctx.plan is None:
            grads = [torch.zeros_like(t) if need else None for t, need in zip((q, k, v), needs)]
        else:
            grads = _backward(ctx.plan, q, k, v, o, lse, go, glse, ctx.sm_scale, lengths, needs)
        return (*grads, None, None, None, None)


def _nothing(q):
    """(o, lse) of rows that see no key, or of no rows."""
    return torch.zeros(q.shape, dtype=q.dtype, device=q.device), torch.full(q.shape[:3], -math.inf, dtype=torch.float32, device=q.device)


def cross_attention(q, k, v, sm_scale, lengths=None, *, return_lse=False):
    """softmax(q k^T sm_scale) v: ``o``, or ``(o, lse)``.

    q [Z, heads, T, D]; k, v [Z, key heads, N, D] of the same dtype, float16 or bfloat16; D is 32, 64, 128
    or 256, heads a multiple of the key heads: query head i reads key head ``i // (heads // key heads)``.
    Any strides (rows that are not 16-byte aligned with a unit last stride are copied first; strides of 0, as
    ``expand`` gives them, are fine).  ``lengths`` (int32 [Z] on the GPU; None: N of all): the keys of each
    sequence, its first ones; values outside [0, N] are taken as its ends, and what lies behind them is not read.  A
    sequence without keys gives 0 (lse -inf).

    Sums are in 32 bits; softmax weights are rounded to the dtype for the product with v, as o is.
    ``lse``: the natural logarithm of each row's sum of exponentials, float32 [Z, heads, T].

    Differentiable once in q, k and v, through o and lse; gradients do not change from call to call (no atomics).
    For the gradients' products softmax weights and their gradients are rounded to the dtype, in float16 scaled by
    powers of two first that keep them within the type, whatever the sizes of v and of o's gradient.  Keys
    past a length have gradients of 0.
    """
    sm_scale = float(sm_scale)
    if math.isnan(sm_scale):
        raise ValueError("sm_scale is NaN")
    # tensors with a key that is kept have passed the checks, and only their addresses may differ
    key = (q.shape, k.shape, v.shape, q.stride(), k.stride(), v.stride(), q.dtype, k.dtype, v.dtype, q.device, k.device, v.device,
           (lengths.shape, lengths.stride(), lengths.dtype, lengths.device) if isinstance(lengths, torch.Tensor) else lengths is None)
    plan = _PLANS.get(key)
    if plan is None or (q.data_ptr() | k.data_ptr() | v.data_ptr()) & 15:
        _check(q, k, v, lengths)
        if lengths is not None:
            lengths = lengths.contiguous()
        if q.numel() and k.numel():
            tensors = [_as_kernel_layout(t) for t in (q, k, v)]
            plan = _Plan(*tensors)
            if tensors[0] is q and tensors[1] is k and tensors[2] is v and (lengths is None or lengths.stride() == key[-1][1]):
                if len(_PLANS) > 4096:
                    _PLANS.clear()
                _PLANS[key] = plan
            q, k, v = tensors
    if (torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)) or _has_tangent(q, k, v):
        return _CrossAttention.apply(q, k, v, plan, sm_scale, lengths, bool(return_lse))
    if plan is None:
        o, lse = _nothing(q)
    else:
        o, lse = _forward(plan, q, k, v, sm_scale, lengths, return_lse)
    return (o, lse) if return_lse else o
