"""A decoder's layers with an encoder, served with drafts: rotary positions, a drafted tree over the 4-bit cache, cross
attention to the encoder's states, the accepted path kept."""
import pytest
import torch

from ascend_rsfa.cache4 import Cache4
from ascend_rsfa.cross import cross_attention
from ascend_rsfa.draft import draft_tree
from ascend_rsfa.rotary import rotary, rotary_plan
from oracle import cross as X64
from oracle import draft as D64
from oracle import serving as S

pytestmark = pytest.mark.gpu

BF16, HALF = torch.bfloat16, 2.0 ** -8
BUFFERS = ("k_codes", "k_scales", "v_codes", "v_scales", "positions", "weights")


def _randn(shape, seed, dtype):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def _ints(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


def _parents(T, seed):
    g = torch.Generator().manual_seed(seed)
    return [int(torch.randint(-1, i, (1,), generator=g)) if i else -1 for i in range(T)]


def _decode(keys, values, plan, prompts, steps, T, draft, group=2):
    """A decoder's steps over its text and an encoder's states: a tree of drafted tokens, its attention, the
    accepted path kept; returns each step's outputs of the accepted tokens."""
    Z, H, _, D = prompts[0].shape
    cache = Cache4(Z, H, 400, D, BF16)
    lengths = _ints([0] * Z)
    q, k = rotary(prompts[0], prompts[0], 0, plan)
    cache.append(k, prompts[1], lengths)
    lengths += prompts[0].shape[2]
    out = []
    for step in range(steps):
        x, v = draft(step)
        parents = _parents(T, 100 + step)
        path = []
        i = T - 1
        while i >= 0:
            path, i = [i] + path, parents[i]
        tree = draft_tree(_ints(parents))
        q, k = rotary(x, x[:, ::group].contiguous(), lengths[:, None] + tree.depths, plan)
        cache.append(k, v, lengths)
        o = cache.attend(q, lengths + T, True, D ** -0.5, tree=tree)
        o = o + cross_attention(x, keys, values, D ** -0.5)
        out.append(o[:, :, path])
        cache.keep(_ints([path] * Z), lengths)
        lengths += len(path)
    return cache, lengths, out


def test_drafted_decoding_equals_decoding_token_by_token():
    # the accepted tokens alone, one by one, give the same rows and (but for roundings of the sums' order) outputs
    Z, H, D, T, group = 2, 2, 64, 9, 2
    plan = rotary_plan(D)
    keys, values = _randn((Z, H, 77, D), 1, BF16), _randn((Z, H, 77, D), 2, BF16)
    prompts = [_randn((Z, H, 130, D), 3, BF16), _randn((Z, H, 130, D), 4, BF16)]
    drafts = [(_randn((Z, H * group, T, D), 10 + i, BF16), _randn((Z, H, T, D), 20 + i, BF16)) for i in range(6)]
    cache, lengths, out = _decode(keys, values, plan, prompts, 6, T, lambda i: drafts[i], group)
    # each side of an attention is off by a weight's rounding, at most half a step of all |v|, and o's own, no more;
    # the sum of both rounds once more: per side (2 + 1) half steps (2^-8) of each largest |v|, and 2 % for the rest
    largest = max(float(values.abs().max()), 1e-9) + max(float(S.values(cache.v_codes, cache.v_scales).abs().max()), 1e-9)
    tol = 2 * 3 * 2.0 ** -8 * largest * 1.02
    one = Cache4(Z, H, 400, D, BF16)
    at = _ints([0] * Z)
    _, k = rotary(prompts[0], prompts[0], 0, plan)
    one.append(k, prompts[1], at)
    at += 130
    for step in range(6):
        parents = _parents(T, 100 + step)
        path, i = [], T - 1
        while i >= 0:
            path, i = [i] + path, parents[i]
        for j, t in enumerate(path):
            x, v = drafts[step][0][:, :, t:t + 1], drafts[step][1][:, :, t:t + 1]
            q, k = rotary(x, x[:, ::group].contiguous(), at[:, None], plan)
            one.append(k, v, at)
            at += 1
            o = one.attend(q, at, True, D ** -0.5)
            o = o + cross_attention(x, keys, values, D ** -0.5)
            assert ((o - out[step][:, :, j:j + 1]).double().abs() <= tol).all()
    n = int(lengths[0])
    assert torch.equal(lengths, at)
    for name in BUFFERS[:5]:
        assert torch.equal(getattr(one, name)[:, :, :n], getattr(cache, name)[:, :, :n]), name


def _bounded(q, k, v, see, scale):
    """Attention of drafted tokens in float64, and what the kernel may be off by: the tolerance of tests/test_draft_gpu.py for bfloat16."""
    o, _, total, reach = D64.attend(q, k, v, see, scale)
    r, sums = (q.shape[3] + 4) * 2.0 ** -24 * reach, (int(see.sum(-1).max()) + 16) * 2.0 ** -23
    return o, total * (HALF + (2 * r + sums)[..., None]) * (1 + HALF) + o.abs() * HALF


def test_drafted_decoding_equals_decoding_token_by_token_where_ancestors_weigh():
    # Drafted tokens share a direction in the dims that rotary turns least, so that each token's weight lies on its ancestors and
    # itself; outputs are held to the bounds of their own elements, which a tree that hides or shows other tokens is far outside of.
    Z, H, D, T, group, steps, scale = 2, 2, 64, 9, 2, 5, 64 ** -0.5
    plan = rotary_plan(D)
    keys, values = _randn((Z, H, 77, D), 1, BF16), _randn((Z, H, 77, D), 2, BF16)
    prompts = [_randn((Z, H, 130, D), 3, BF16), _randn((Z, H, 130, D), 4, BF16)]
    way = torch.zeros(D)
    way[[28, 29, 30, 31, 60, 61, 62, 63]] = 2.5
    drafted, one = Cache4(Z, H, 300, D, BF16), Cache4(Z, H, 300, D, BF16)
    lengths, at = _ints([0] * Z), _ints([0] * Z)
    for c, n in ((drafted, lengths), (one, at)):
        _, k = rotary(prompts[0], prompts[0], 0, plan)
        c.append(k, prompts[1], n)
        n += 130
    told_apart = 0
    for step in range(steps):
        x = (0.5 * _randn((Z, H * group, T, D), 10 + step, torch.float32) + way.cuda()).to(BF16)
        v = _randn((Z, H, T, D), 20 + step, BF16)
        g = torch.Generator().manual_seed(step)
        parents = [max(-1, i - 1 - int(torch.randint(0, 2, (1,), generator=g))) for i in range(T)]
        path, i = [], T - 1
        while i >= 0:
            path, i = [i] + path, parents[i]
        tree = draft_tree(_ints(parents))
        q, k = rotary(x, x[:, ::group].contiguous(), lengths[:, None] + tree.depths, plan)
        drafted.append(k, v, lengths)
        got = (drafted.attend(q, lengths + T, True, scale, tree=tree) + cross_attention(x, keys, values, scale))[:, :, path]
        # what it is, and what it would be if tokens saw themselves and the context alone, or all drafted tokens up to themselves
        rows = S.values(drafted.k_codes, drafted.k_scales), S.values(drafted.v_codes, drafted.v_scales)
        tables = D64.seen(parents), torch.eye(T, dtype=torch.bool), torch.ones((T, T), dtype=torch.bool).tril()
        o, wrong, more = (_bounded(q, *rows, D64.visible(t.expand(Z, T, T), (lengths + T).tolist(), None, 300), scale) for t in tables)
        c, bound = X64.expect(x, keys, values, None, scale)["o"]
        off = 2 * ((o[1] + bound) * (1 + HALF) + HALF * (o[0] + c).abs())[:, :, path]
        for other in (wrong, more):
            told_apart += int(((other[0] - o[0])[:, :, path].abs() > off).sum())
        for j, t in enumerate(path):
            y = x[:, :, t:t + 1]
            q, k = rotary(y, y[:, ::group].contiguous(), at[:, None], plan)
            one.append(k, v[:, :, t:t + 1], at)
            at += 1
            want = one.attend(q, at, True, scale) + cross_attention(y, keys, values, scale)
            assert ((want - got[:, :, j:j + 1]).double().abs() <= off[:, :, j:j + 1]).all(), (step, t)
            assert ((want.double() - (o[0] + c)[:, :, t:t + 1]).abs() <= off[:, :, j:j + 1] / 2).all(), (step, t)
        drafted.keep(_ints([path] * Z), lengths)
        lengths += len(path)
    compared = 2 * Z * H * group * D * int((lengths - 130)[0])
    assert told_apart > compared // 2, (told_apart, compared)
