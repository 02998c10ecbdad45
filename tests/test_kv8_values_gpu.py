"""Attention over 8-bit pages where numbers of very different size meet, or that are none."""
import pytest
import torch

from tests.kv8_reference import FMTS, Cache
from tests.test_kv8_gpu import _attend, _check_attend, _groups, bf

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("hq,hkv,hd", [(16, 2, 128), (8, 2, 64)])
@pytest.mark.parametrize("factor", [30.0, 200.0])
@pytest.mark.parametrize("rows", [1, 5])
def test_channels_of_very_different_size(hq, hkv, hd, fmt, factor, rows):
    """One channel of q `factor` times the others; another one of K as much larger, q as much smaller there, so that it counts as any
    other.  A score has to come from all digits of q: the bound takes its error as 2^-17 of sum |q k|, no part of the largest channel."""
    n = 700
    g = torch.Generator().manual_seed(int(factor) + hd)
    k = torch.randn(n, hkv, hd, generator=g)
    v = torch.randn(n, hkv, hd, generator=g)
    q = torch.randn(rows, hq, hd, generator=g)
    k[..., 9] *= factor
    q[..., 9] /= factor
    q[..., 40] *= factor
    k[..., 40] *= 0.02                                        # codes of 0 to 3 where the large channel is: the others decide
    c = Cache([n], hkv, hd, fmt, k=[k], v=[v])
    pos, seq, g0, gc = _groups([n], [rows])
    q = bf(q.reshape(rows, hq * hd))
    out = _attend(c, q, hq, pos, seq, g0, gc)
    _check_attend(c, q, hq, out, pos, seq, g0, gc)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_rows_that_see_nothing_are_zeros_whatever_their_q_holds(fmt, bad):
    """Padded rows (position -1) and rows with an empty mask, of one split and of two, with q that is no number: zeros, and their
    neighbours do not notice."""
    hq, hkv, hd = 8, 2, 64
    lens, new = [24, 40, 9], [24, 1, 9]
    c = Cache(lens, hkv, hd, fmt, seed=3)
    pos, seq, g0, gc = _groups(lens, new)
    pos[24] = -1
    mask = [(1 << r + 1) - 1 for cnt in new for r in range(cnt)]
    empty = [0, 7, 20, 23, 24, 25, 33]                        # 20 and 23 lie in the second split of sixteen keys
    for t in empty:
        mask[t] = 0
    q = bf(torch.randn(len(pos), hq * hd))
    out = _attend(c, q, hq, pos, seq, g0, gc, mask, split_keys=16)
    assert bool((out[empty] == 0).all())
    q[empty] = bad
    again = _attend(c, q, hq, pos, seq, g0, gc, mask, split_keys=16)
    assert bool((again[empty] == 0).all())
    assert torch.equal(again, out)
    _check_attend(c, q, hq, out, pos, seq, g0, gc, mask)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("big", [1.0, 1e15, 1e25])
@pytest.mark.parametrize("split", [128, 768])
def test_rows_of_zeros_beside_large_values_keep_their_weight(fmt, big, split):
    """Some pages' V are zeros (the least scale there is), the others' are as large as `big`: what the zeros weigh stays in the sum,
    whichever warp or split has them, and in whichever order they come."""
    hq, hkv, hd = 8, 2, 64
    n = 640
    g = torch.Generator().manual_seed(8)
    k = [torch.randn(n, hkv, hd, generator=g) for _ in range(3)]
    v = [torch.randn(n, hkv, hd, generator=g) * big for _ in range(3)]
    page = torch.arange(n) // 16
    v[0][page % 4 == 1] = 0                                   # all of one warp's
    v[1][(page >= 8) & (page < 24)] = 0                       # whole splits
    v[2][page < 20] = 0                                       # zeros first, then large ones
    c = Cache([n] * 3, hkv, hd, fmt, k=k, v=v)
    pos, seq, g0, gc = _groups([n] * 3, [1, 4, 1])
    q = bf(torch.randn(len(pos), hq * hd))
    out = _attend(c, q, hq, pos, seq, g0, gc, split_keys=split)
    _check_attend(c, q, hq, out, pos, seq, g0, gc)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("power", [98, 40, -50])
def test_scores_of_large_times_small(fmt, power):
    """K of 2^98 against q of 2^-98 and the other way round: the scores are ordinary numbers, and nothing on the way to them is not."""
    hq, hkv, hd = 8, 2, 128
    g = torch.Generator().manual_seed(abs(power))
    n = 300
    k = torch.randn(n, hkv, hd, generator=g) * 2.0 ** power
    v = torch.randn(n, hkv, hd, generator=g)
    c = Cache([n], hkv, hd, fmt, k=[k], v=[v])
    pos, seq, g0, gc = _groups([n], [3])
    q = bf(torch.randn(3, hq * hd, generator=g) * 2.0 ** -power)
    out = _attend(c, q, hq, pos, seq, g0, gc)
    _check_attend(c, q, hq, out, pos, seq, g0, gc)
