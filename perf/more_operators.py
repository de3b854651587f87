"""Attention outside of a sequence's own keys, as it is measured.

What a decoder runs next to its causal attention: cross attention to an
encoder's states of another length (one token, a prompt, a training step with
its gradients), and speculative decoding over the 4-bit cache: attention of a
tree of drafted tokens, each of which sees the context and its ancestors, and
keeping the tokens that were accepted.

``run`` computes each in elementary torch operations, or with ``own`` through
the framework.  A cache row holds the head dim in blocks of 32: a scale byte
b (2^(b - 127); 255: the block is NaN) and 32 codes of 4 bits, sign and
magnitude index into 0, 0.5, 1, 1.5, 2, 3, 4, 6; byte j of a row has dim 2j in its
low and dim 2j + 1 in its high bits.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _framework():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ascend-rsfa_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    from ascend_rsfa import cache4, cross, draft
    return cache4, cross, draft


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def _cross(Z, Hq, H, T, N, D, dtype, layout, lengths, lse=False, train=False):
    """lengths: "none" (all N states), "ragged" (a padded batch) or "empty" (padded, one sequence without states)."""
    return {"op": "cross", "Z": Z, "Hq": Hq, "H": H, "T": T, "N": N, "D": D, "dtype": dtype, "layout": layout,
            "lengths": lengths, "lse": lse, "train": train}


def _tree(Z, Hq, H, T, N, D, dtype, layout, ragged, dynamic, lse=False):
    """dynamic: every sequence drafts a tree of its own, of its own size, in each step; otherwise one fixed tree."""
    return {"op": "tree", "Z": Z, "Hq": Hq, "H": H, "T": T, "N": N, "D": D, "dtype": dtype, "layout": layout,
            "ragged": ragged, "dynamic": dynamic, "lse": lse}


def _keep(Z, H, T, n, C, D, dtype, ragged):
    return {"op": "keep", "Z": Z, "H": H, "T": T, "n": n, "C": C, "D": D, "dtype": dtype, "ragged": ragged}


def listed():
    return [
        # one sequence's next token over a long source: all latency
        dict(_cross(1, 32, 8, 1, 8192, 128, "bf16", "bhsd", "none"), name="cross-token"),
        # the next token of every sequence of a padded batch, one key head per query head
        dict(_cross(32, 16, 16, 1, 1531, 64, "f16", "bshd", "ragged"), name="cross-token-batch"),
        # prompts of a decoder over its encoder's states; the caller merges parts by the logsumexp
        dict(_cross(8, 16, 16, 1024, 4096, 128, "bf16", "bshd", "none", lse=True), name="cross-prompt"),
        # a training step of a few short targets over short sources: all latency
        dict(_cross(2, 8, 8, 64, 197, 32, "f16", "bhsd", "none", train=True), name="cross-train-short"),
        # a training step of an image's positions over a short text
        dict(_cross(8, 8, 8, 4096, 77, 64, "f16", "bshd", "ragged", train=True), name="cross-train-text"),
        # a training step of ragged sources and targets of no round length
        dict(_cross(16, 16, 16, 447, 1531, 64, "bf16", "bshd", "ragged", train=True), name="cross-train-ragged"),
        # a training step over long sources, several query heads to a key head: the largest
        dict(_cross(8, 32, 8, 2048, 4096, 128, "bf16", "bhsd", "none", train=True), name="cross-train-long"),
        # seven drafted tokens of each of a few short sequences, the same tree for all: all latency
        dict(_tree(8, 16, 16, 7, 511, 64, "f16", "bhsd", True, False), name="tree-short"),
        # a batch, trees of its own for each sequence, up to 25 tokens
        dict(_tree(32, 32, 8, 25, 4096, 128, "bf16", "bshd", True, True), name="tree-batch"),
        # one sequence, a wide tree of 64 tokens over a long text
        dict(_tree(1, 32, 8, 64, 32768, 128, "f16", "bhsd", False, False, lse=True), name="tree-long"),
        # the accepted path of one sequence
        dict(_keep(1, 8, 25, 5, 4096, 128, "bf16", False), name="keep-one"),
        # the accepted paths of a large batch
        dict(_keep(64, 8, 64, 17, 2048, 256, "f16", True), name="keep-batch"),
    ]


# products of the largest listed case, and the elements a case may hold
_MAX_PRODUCTS = 8 * 32 * 2048 * 4096 * 128
_MAX_ROWS = 1 << 27


def _log_int(rng, lo, hi):
    n = min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))
    return n + 1 if n % 2 == 0 and n < hi and rng.random() < 0.4 else n


def draw(rng):
    op = rng.choice(["cross", "cross", "cross", "cross", "tree", "tree", "tree", "keep"])
    D = rng.choice([32, 64, 64, 128, 128, 128, 256])
    H = rng.choice([2, 4, 8, 8, 16])
    group = rng.choice([1, 1, 2, 4, 8])
    Z = _log_int(rng, 1, 64)
    dtype = rng.choice(["f16", "bf16"])
    layout = rng.choice(["bhsd", "bshd"])
    if op == "cross":
        train = rng.random() < 0.5
        T = rng.choice([1, 1, _log_int(rng, 2, 64), _log_int(rng, 65, 4096)]) if not train else _log_int(rng, 16, 4096)
        N = _log_int(rng, 17, 8192)
        Z = max(1, min(Z, _MAX_ROWS // (H * N * D), _MAX_ROWS // (H * group * T * D),
                       _MAX_PRODUCTS // (H * group * T * N * max(D, 64) * (1 if train else 2))))
        return _cross(Z, H * group, H, T, N, D, dtype, layout, rng.choice(["none", "ragged", "ragged", "empty"]),
                      rng.random() < 0.3 and not train, train)
    if op == "tree":
        T = _log_int(rng, 2, 128)
        N = _log_int(rng, max(T, 33), 32768)
        Z = max(1, min(Z, _MAX_ROWS // (N * H * D), (1 << 29) // (H * group * T * N)))
        return _tree(Z, H * group, H, T, N, D, dtype, layout, rng.random() < 0.6, rng.random() < 0.5, rng.random() < 0.3)
    T = _log_int(rng, 2, 256)
    C = T + _log_int(rng, 64, 4096)
    Z = max(1, min(Z, _MAX_ROWS // (C * H * D)))
    return _keep(Z, H, T, _log_int(rng, 1, min(T, 32)), C, D, dtype, rng.random() < 0.6)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _normal(shape, g, std=1.0):
    return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(0.0, std, generator=g)


def _heads(Z, H, N, D, dtype, layout, g, std=1.0):
    """[Z, H, N, D], in that order in memory or seen through a transpose of [Z, N, H, D]."""
    if layout == "bshd":
        return _normal((Z, N, H, D), g, std).to(DTYPES[dtype]).transpose(1, 2)
    return _normal((Z, H, N, D), g, std).to(DTYPES[dtype])


def _spread(Z, N, least):
    """Lengths from `least` to N, in no order."""
    return [N - (N - least) * (z * 7 % Z) // Z for z in range(Z)]


def _states(case):
    """Encoder states of each sequence."""
    Z, N = case["Z"], case["N"]
    lengths = [N] * Z if case["lengths"] == "none" else _spread(Z, N, max(1, N // 4))
    if case["lengths"] == "empty":
        lengths[-1] = 0
    return lengths


def _slots(case):
    """Slots in use of each sequence, its drafted tokens included."""
    Z, N, T = case["Z"], case["N"], case["T"]
    return [max(T, n) for n in _spread(Z, N, max(1, N // 4))] if case["ragged"] else [N] * Z


def _drafted(case):
    """Drafted tokens of each sequence."""
    Z, T = case["Z"], case["T"]
    return _spread(Z, T, max(1, T // 2)) if case["dynamic"] else [T] * Z


def _accepted(case):
    Z, n = case["Z"], case["n"]
    return _spread(Z, n, 0) if case["ragged"] else [n] * Z


def _pow2(e):
    """2^e of whole numbers -126 .. 127, exactly."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _packed(Z, H, N, D, g, std):
    """A filled cache's codes and scales: rows of a projection, a few dims larger than the rest."""
    codes = torch.empty((Z, H, N, D // 2), dtype=torch.uint8, device="cuda")
    scales = torch.empty((Z, H, N, D // 32), dtype=torch.uint8, device="cuda")
    gain = 1.0 + 3.0 * (torch.rand((H, 1, D), device="cuda", generator=g) < 0.03)
    for z in range(Z):
        b = (_normal((H, N, D), g, std) * gain).unflatten(-1, (-1, 32))
        mantissa, exponent = torch.frexp(b.abs().amax(-1))
        e = (exponent - 3 + (mantissa > 0.875)).clamp(-20, 13)
        y = b * _pow2(-e)[..., None]
        a = y.abs()
        m = sum((a > edge).int() for edge in (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0))
        m = torch.where(torch.signbit(y), m + 8, m).flatten(-2)
        codes[z], scales[z] = (m[..., 0::2] | (m[..., 1::2] << 4)).to(torch.uint8), (e + 127).to(torch.uint8)
    return codes, scales


def _values(codes, scales):
    """float32 values of packed rows."""
    table = torch.tensor(GRID + tuple(-v for v in GRID), dtype=torch.float32, device=codes.device)
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()
    s = _pow2((scales.int() - 127).clamp(max=127)).masked_fill(scales == 255, math.nan)
    return (table[c].unflatten(-1, (-1, 32)) * s[..., None]).flatten(-2)


def _cache_buffers(case, C, g):
    Z, H, D = case["Z"], case["H"], case["D"]
    kc, ks = _packed(Z, H, C, D, g, 0.7)
    vc, vs = _packed(Z, H, C, D, g, 1.0)
    positions = torch.arange(C, dtype=torch.int32, device="cuda").expand(Z, H, C).contiguous()
    weights = _normal((Z, H, C), g).exp_()
    return {"k_codes": kc, "k_scales": ks, "v_codes": vc, "v_scales": vs, "positions": positions, "weights": weights}


def _parents(Z, T, g):
    """Drafted trees: a token's parent is an earlier token, or -1, the context's last token; wide near the root."""
    i = torch.arange(T, device="cuda")
    u = torch.rand((Z, T), device="cuda", generator=g) ** 2
    return ((u * (i + 1)).floor().long() - 1).clamp(max=i - 1).int()


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": dict(case)}
    op, Z, H, D = case["op"], case["Z"], case["H"], case["D"]
    if op == "cross":
        T, N, Hq = case["T"], case["N"], case["Hq"]
        s["q"] = _heads(Z, Hq, T, D, case["dtype"], case["layout"], g)
        s["k"] = _heads(Z, H, N, D, case["dtype"], case["layout"], g)
        s["v"] = _heads(Z, H, N, D, case["dtype"], case["layout"], g)
        s["lengths"] = None if case["lengths"] == "none" else _int(_states(case))
        s["scale"] = D ** -0.5
        if case["train"]:
            for x in "qkv":
                s[x].requires_grad_()
            s["go"] = _heads(Z, Hq, T, D, case["dtype"], case["layout"], g, 0.05)
        return s
    if op == "tree":
        T, N = case["T"], case["N"]
        s["q"] = _heads(Z, case["Hq"], T, D, case["dtype"], case["layout"], g)
        b = _cache_buffers(case, N, g)
        s["lengths"] = _int(_slots(case))
        s["parents"] = _parents(Z, T, g) if case["dynamic"] else _parents(1, T, g)[0]
        s["counts"] = _int(_drafted(case)) if case["dynamic"] else None
        s["scale"] = D ** -0.5
    else:
        T, n, C = case["T"], case["n"], case["C"]
        b = _cache_buffers(case, C, g)
        s["lengths"] = torch.randint(0, C - T + 1, (Z,), device="cuda", generator=g).int()  # the contexts
        # a path: tokens in ascending order
        s["tokens"] = torch.rand((Z, T), device="cuda", generator=g).argsort(-1)[:, :n].sort(-1)[0].int()
        s["counts"] = _int(_accepted(case)) if case["ragged"] else None
    s["buffers"] = b
    if own:
        cache4, _, draft = _framework()
        s["cache"] = cache4.Cache4.from_buffers(**b, dtype=DTYPES[case["dtype"]])
        if op == "tree" and not case["dynamic"]:
            s["tree"] = draft.draft_tree(s["parents"])  # a fixed tree is made once
    return s


# ---------------------------------------------------------------------------
# Cross attention
# ---------------------------------------------------------------------------
def _cross_plain(q, k, v, lengths, scale, go):
    """(o, lse), and with go (dq, dk, dv), in float32, of some sequences."""
    Z, Hq, T, D = q.shape
    H, N = k.shape[1], k.shape[2]
    qf, kf, vf = q.float().reshape(Z, H, -1, D), k.float(), v.float()
    x = torch.matmul(qf, kf.transpose(-1, -2)).mul_(scale)
    if lengths is not None:
        hidden = torch.arange(N, device="cuda") >= lengths[:, None]
        x = x.masked_fill_(hidden[:, None, None, :], -math.inf)
    top = x.amax(-1, keepdim=True)
    p = x.sub_(top.clamp(min=-1e30)).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(total.masked_fill(total == 0, 1.0))
    o = torch.matmul(p, vf)
    lse = top + total.log()
    if go is None:
        return o.reshape(q.shape), lse.reshape(Z, Hq, T), None
    gf = go.float().reshape(Z, H, -1, D)
    dv = torch.matmul(p.transpose(-1, -2), gf)
    ds = torch.matmul(gf, vf.transpose(-1, -2))
    ds = ds.sub_((gf * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    return o.reshape(q.shape), None, (torch.matmul(ds, kf).reshape(q.shape), torch.matmul(ds.transpose(-1, -2), qf), dv)


def _run_cross(s):
    case, q, k, v = s["case"], s["q"], s["k"], s["v"]
    if own:
        _, cross, _ = _framework()
        if case["train"]:
            o = cross.cross_attention(q, k, v, s["scale"], s["lengths"])
            return [o, *torch.autograd.grad(o, (q, k, v), s["go"])]
        r = cross.cross_attention(q, k, v, s["scale"], s["lengths"], return_lse=case["lse"])
        return list(r) if case["lse"] else [r]
    Z, Hq, T, _ = q.shape
    step = max(1, (1 << 30) // (Hq * T * case["N"]))  # sequences at once, within memory
    parts = []
    with torch.no_grad():
        for z in range(0, Z, step):
            at = slice(z, z + step)
            lengths = None if s["lengths"] is None else s["lengths"][at]
            o, lse, grads = _cross_plain(q[at], k[at], v[at], lengths, s["scale"], s["go"][at] if case["train"] else None)
            part = [o.to(q.dtype)]
            if case["lse"]:
                part.append(lse)
            if case["train"]:
                part += [x.to(q.dtype) for x in grads]
            parts.append(part)
        return parts[0] if len(parts) == 1 else [torch.cat(x) for x in zip(*parts)]


# ---------------------------------------------------------------------------
# A tree of drafted tokens over the cache
# ---------------------------------------------------------------------------
def _seen(parents):
    """[Z, T, T]: whether token i sees drafted token j, itself or an ancestor."""
    p = parents.long().reshape(-1, parents.shape[-1])
    T = p.shape[-1]
    step = torch.nn.functional.one_hot(p + 1, T + 1)[..., 1:].float()  # row i: its parent
    seen = torch.eye(T, device="cuda") + step
    for _ in range(max(1, T - 1).bit_length()):  # paths of twice the length each time
        seen = torch.matmul(seen, seen).clamp_(max=1.0)
    return seen > 0


def _run_tree(s):
    case, b, q = s["case"], s["buffers"], s["q"]
    if own:
        tree = s["tree"] if not case["dynamic"] else _framework()[2].draft_tree(s["parents"])
        r = s["cache"].attend(q, s["lengths"], True, s["scale"], counts=s["counts"], return_lse=case["lse"], tree=tree)
        return list(r) if case["lse"] else [r]
    Z, Hq, T, D = q.shape
    H, N = case["H"], case["N"]
    k, v = _values(b["k_codes"], b["k_scales"]), _values(b["v_codes"], b["v_scales"])
    counts = s["counts"] if s["counts"] is not None else torch.full((Z,), T, device="cuda", dtype=torch.int32)
    context = (s["lengths"] - counts)[:, None]
    slot = torch.arange(N, device="cuda")
    token = slot - context  # [Z, N]: the drafted token of a slot
    drafted = (token >= 0) & (token < counts[:, None])
    seen = _seen(s["parents"]).expand(Z, T, T)
    seen = seen.gather(2, token.clamp(0, T - 1)[:, None, :].expand(Z, T, N)) & drafted[:, None, :]
    seen = seen | (slot < context)[:, None, :]
    x = torch.matmul(q.float().reshape(Z, H, -1, D), k.transpose(-1, -2)).mul_(s["scale"]).view(Z, H, Hq // H, T, N)
    x = x.masked_fill_(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    p = x.sub_(top.clamp(min=-1e30)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(Z, H, -1, N), v).view(Z, H, Hq // H, T, D)
    there = (torch.arange(T, device="cuda") < counts[:, None])[:, None, None, :, None] & (total > 0)
    o = torch.where(there, o / total, torch.zeros_like(o)).reshape(q.shape).to(q.dtype)
    if not case["lse"]:
        return [o]
    return [o, torch.where(there, top + total.log(), torch.full_like(top, -math.inf)).reshape(Z, Hq, T)]


# ---------------------------------------------------------------------------
# Keeping the accepted tokens
# ---------------------------------------------------------------------------
def _run_keep(s):
    case, b = s["case"], s["buffers"]
    if own:
        s["cache"].keep(s["tokens"], s["lengths"], counts=s["counts"])
        return dict(b)
    n = case["n"]
    i = torch.arange(n, device="cuda")
    start = s["lengths"][:, None].long()
    taken = (i < (s["counts"][:, None] if s["counts"] is not None else n)).expand(start.shape[0], n)
    to = (start + i)[:, None, :].expand(-1, case["H"], -1)
    source = torch.where(taken, start + s["tokens"].long(), start + i)[:, None, :].expand(-1, case["H"], -1)
    for name, t in b.items():
        shape = to.shape + (1,) * (t.dim() - 3)
        rows = t.gather(2, source.reshape(shape).expand(to.shape + t.shape[3:]))
        if name == "positions":
            rows = torch.where(taken[:, None, :], to, t.gather(2, to).long()).int()
        t.scatter_(2, to.reshape(shape).expand(to.shape + t.shape[3:]), rows)
    # bytes that are moved as they are: codes and scales are compared as whole numbers
    return dict(b)


def run(state):
    return {"cross": _run_cross, "tree": _run_tree, "keep": _run_keep}[state["case"]["op"]](state)


# ---------------------------------------------------------------------------
# Work, and the definition in 64 bits
# ---------------------------------------------------------------------------
def work(case):
    op, Z, H, D = case["op"], case["Z"], case["H"], case["D"]
    if op == "cross":
        T, Hq, states = case["T"], case["Hq"], sum(_states(case))
        rows, keys = Z * Hq * T * D * 2, states * H * D * 2
        padded = Z * case["N"] * H * D * 2
        # q, k, v, o; the gradients of all four, those of padded states among them
        nbytes = 2 * rows + 2 * keys + (2 * rows + 2 * padded if case["train"] else 0) + (4 * Z * Hq * T if case["lse"] else 0)
        # q k^T and p v; and go v^T, p^T go, ds k, ds^T q
        return {"bytes": nbytes, "flops": (12 if case["train"] else 4) * Hq * D * T * states}
    if op == "tree":
        T, Hq = case["T"], case["Hq"]
        live, pairs = sum(_slots(case)), sum(n * t for n, t in zip(_slots(case), _drafted(case)))
        nbytes = live * H * 2 * (D // 2 + D // 32) + 4 * Z * Hq * T * D + (4 * Z * Hq * T if case["lse"] else 0)
        return {"bytes": nbytes + 4 * T * (Z if case["dynamic"] else 1), "flops": 4 * Hq * D * pairs}
    rows = sum(_accepted(case)) * H
    return {"bytes": 2 * rows * (2 * (D // 2 + D // 32) + 8) + 4 * Z * case["n"], "flops": rows}


def _decoded(codes, scales):
    """float64 values of packed rows, from the fields of each code: sign, two exponent bits, one fraction bit."""
    c = torch.cat(((codes & 15)[..., None], (codes >> 4)[..., None]), -1).reshape(codes.shape[:-1] + (-1,)).double()
    sign = torch.where(c >= 8, -1.0, 1.0).double()
    c = torch.where(c >= 8, c - 8, c)
    exponent, fraction = torch.div(c, 2, rounding_mode="floor"), c.remainder(2.0)
    value = torch.where(exponent == 0, 0.5 * fraction, (1.0 + 0.5 * fraction) * 2.0 ** (exponent - 1.0))
    step = (2.0 ** (scales.double() - 127.0)).repeat_interleave(32, -1)
    return sign * value * step


def _exact_cross(case, s):
    q, k, v = (s[x].detach() for x in "qkv")
    Z, Hq, T, D = q.shape
    group = Hq // case["H"]
    lengths = _states(case)
    double = {"dtype": torch.float64, "device": "cuda"}
    o, lse = torch.zeros(q.shape, **double), torch.full((Z, Hq, T), -math.inf, **double)
    dq, dk, dv = torch.zeros(q.shape, **double), torch.zeros(k.shape, **double), torch.zeros(v.shape, **double)
    for z in range(Z):
        n = lengths[z]
        if n == 0:
            continue
        for i in range(Hq):
            h = i // group
            a, b, c = q[z, i].double(), k[z, h, :n].double(), v[z, h, :n].double()
            x = (a @ b.T) * s["scale"]
            lse[z, i] = torch.logsumexp(x, -1)
            p = torch.exp(x - lse[z, i, :, None])
            o[z, i] = p @ c
            if case["train"]:
                d = s["go"][z, i].double()
                dv[z, h, :n] += p.T @ d
                e = d @ c.T
                e = p * (e - (p * e).sum(-1, keepdim=True)) * s["scale"]
                dq[z, i] = e @ b
                dk[z, h, :n] += e.T @ a
    return [o] + ([lse] if case["lse"] else []) + ([dq, dk, dv] if case["train"] else [])


def _exact_tree(case, s):
    b, q = s["buffers"], s["q"]
    Z, Hq, T, D = q.shape
    group = Hq // case["H"]
    parents = s["parents"].reshape(-1, T).tolist()
    o = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    lse = torch.full((Z, Hq, T), -math.inf, dtype=torch.float64, device="cuda")
    for z, (n, count) in enumerate(zip(_slots(case), _drafted(case))):
        up = parents[z if case["dynamic"] else 0]
        bias = torch.zeros((count, n), dtype=torch.float64)
        bias[:, n - count:] = -math.inf
        for i in range(count):
            j = i
            while j >= 0:
                bias[i, n - count + j] = 0.0
                j = up[j]
        bias = bias.cuda().repeat(group, 1)
        for h in range(case["H"]):
            k = _decoded(b["k_codes"][z, h, :n], b["k_scales"][z, h, :n])
            v = _decoded(b["v_codes"][z, h, :n], b["v_scales"][z, h, :n])
            heads = slice(h * group, (h + 1) * group)
            x = q[z, heads, :count].double().reshape(group * count, D) @ k.T * s["scale"] + bias
            m = torch.logsumexp(x, -1)
            o[z, heads, :count] = (torch.exp(x - m[:, None]) @ v).reshape(group, count, D)
            lse[z, heads, :count] = m.reshape(group, count)
    return [o, lse] if case["lse"] else [o]


def exact(case, seed):
    if case["op"] == "keep":
        return None  # whole numbers, and moved bytes
    s = prepare(case, seed)
    return _exact_cross(case, s) if case["op"] == "cross" else _exact_tree(case, s)
