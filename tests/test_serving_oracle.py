"""Known answers that pin the float64 definitions of the serving operators (oracle/serving.py)."""
import math

import long_rows
import pytest
import torch

from oracle import serving as S


def test_quantiser_known_answers():
    # every code's value, every midpoint (ties to the even index), and beyond the last
    x = torch.zeros(1, 32, dtype=torch.float64)
    row = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, 0.24, 0.26, 5.01, 4.99]
    want = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 6.0, 0.0, 0.5, 6.0, 4.0]
    for sign in (1.0, -1.0):
        for e in (-3, 0, 5):
            x[0, :len(row)] = sign * torch.tensor(row, dtype=torch.float64) * 2.0 ** e
            codes, scales = S.quantise(x, torch.float16)
            assert scales.item() == 127 + e  # 7 * 2^e is the largest value that scale holds
            got = S.values(codes, scales)[0, :len(row)]
            assert torch.equal(got, sign * torch.tensor(want, dtype=torch.float64) * 2.0 ** e)


def test_quantiser_scales_end_at_the_types_range():
    x = torch.zeros(3, 32, dtype=torch.float64)
    x[1, 3] = 2.0 ** -24
    x[2, 3] = 65504.0
    codes, scales = S.quantise(x, torch.float16)
    assert scales[:, 0].tolist() == [127 - 23, 127 - 23, 127 + 13]
    v = S.values(codes, scales)
    assert v[1, 3] == 2.0 ** -24 and v[2, 3] == 6.0 * 2.0 ** 13
    x[1, 3] = math.inf
    x[2, 3] = math.nan
    _, scales = S.quantise(x, torch.bfloat16)
    assert scales[:, 0].tolist() == [2, 255, 255]


def test_attend_against_softmax():
    g = torch.Generator().manual_seed(3)
    q = torch.randn(2, 4, 3, 32, generator=g, dtype=torch.float64)
    k, v = (torch.randn(2, 2, 7, 32, generator=g, dtype=torch.float64) for _ in range(2))
    pos = torch.arange(7).expand(2, 2, 7)
    o, lse, w, total, _ = S.attend(q, k, v, [7, 0], 0.2, pos, [4, 0])
    kk, vv = (t.repeat_interleave(2, 1) for t in (k, v))
    s = torch.matmul(q, kk.transpose(-1, -2)) * 0.2
    s = s.masked_fill(torch.ones(3, 7, dtype=torch.bool).triu(5), -math.inf)
    assert torch.allclose(o[0], torch.matmul(s.softmax(-1), vv)[0], rtol=0, atol=1e-14)
    assert torch.allclose(lse[0], s.logsumexp(-1)[0], rtol=0, atol=1e-14)
    assert torch.allclose(w[0], s.softmax(-1)[0].reshape(2, 6, 7).sum(1), rtol=0, atol=1e-14)
    assert (o[1] == 0).all() and (lse[1] == -math.inf).all() and (w[1] == 0).all()
    assert (total >= o.abs() - 1e-15).all()


def test_rotary_known_answers():
    f = torch.tensor([math.pi / 2, math.pi], dtype=torch.float64)
    x = torch.tensor([1.0, 2.0, 3.0, 4.0, 9.0]).reshape(1, 1, 1, 5)
    half = S.rotary(x, torch.tensor([1]), f, 1.0, "half")
    # pairs (1, 3) by a quarter turn, (2, 4) by a half
    assert torch.allclose(half.flatten(), torch.tensor([-3.0, -2.0, 1.0, -4.0, 9.0], dtype=torch.float64), atol=1e-15)
    inter = S.rotary(x, torch.tensor([1]), f, 2.0, "interleaved")
    assert torch.allclose(inter.flatten(), torch.tensor([-4.0, 2.0, -6.0, -8.0, 9.0], dtype=torch.float64), atol=1e-14)
    back = S.rotary(half, torch.tensor([1]), f, 1.0, "half", inverse=True)
    assert torch.allclose(back, x.double(), atol=1e-14)


def test_eviction_known_answers():
    w = torch.tensor([[[3.0, 1.0, math.nan, 1.0, -0.0, 0.0, 9.0, 5.0]]])
    pos = torch.arange(8).reshape(1, 1, 8)
    assert S.claim(w, pos, [8], 3, 8)[0, 0].tolist() == [1, 4, 5]
    assert S.claim(w, pos, [6], 3, 8)[0, 0].tolist() == [6, 7, 4]
    assert S.claim(w, pos, [8], 4, 8, recent=4, sinks=2)[0, 0].tolist() == [2, 3, -1, -1]
    assert S.evict(w, pos, [8], 3)[0][0] == [2, 6, 7]
    assert S.evict(w, pos, [8], 3, recent=2, sinks=1)[0][0] == [0, 6, 7]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_long_rows_show_what_is_lost(dtype):
    # the values that the GPU tests of long rows expect follow from the definition, and a mistake in V alone shows
    for n, D, C in ((19999, 128, 20000), (16000, 64, 16000), (8130, 256, 9000), (3977, 32, 4000)):
        k, q = torch.zeros((1, 1, C, D), dtype=torch.float64), torch.zeros((1, 1, 1, D), dtype=torch.float64)
        steps = {step: long_rows.marked(n, C, D, dtype, step) for step in (1, 32, 512)}

        def holds(spoil):
            found = []
            for step, v in steps.items():
                bad = v.double()
                spoil(bad[0, 0])
                found.append(long_rows.marks_hold(S.attend(q, k, bad, [n], 1.0)[0].to(dtype), n, v))
            return all(found)

        def shift(v):
            v[512:1024] = v[513:1025].clone()

        def twice(v):
            v[64:96] += v[96:128]

        def unseen(v):
            v[n - 1] = 1.0

        assert holds(lambda v: None)
        one = (lambda v: v[5].zero_(), lambda v: v[n - 1].zero_(), unseen) if dtype == torch.float16 or n <= 2 ** 7 * D else ()
        for spoil in (lambda v: v[:512].zero_(), lambda v: v[n // 2:n // 2 + 32].zero_(), lambda v: v[n - n % 32 - 32:].zero_(),
                      lambda v: v[1024:1536].zero_(), shift, twice, *one):
            assert not holds(spoil)
        slots = [0, n - 1, n // 2, 31]
        k, v, q = long_rows.peaks(slots, n, C, D, dtype, 1)
        codes, scales = S.quantise(v, dtype)
        assert torch.equal(S.values(codes, scales), v.double())
        o = S.attend(q[None, None].double(), k.double(), v.double(), [n], 1.0)[0]
        assert torch.equal(o[0, 0].to(dtype), v[0, 0, slots])
