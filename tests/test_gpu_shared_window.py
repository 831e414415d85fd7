"""Attention behind shared prefixes with windows that leave enough of a prefix to be read
once (paged.attention_shared), against plain 64-bit attention over each sequence's whole table."""

import math

import pytest
import torch

import oracle.ref_paged as R
from tests.test_gpu_paged_shared import Setup

pytestmark = pytest.mark.gpu


def _mb(s, window):
    """What sharing saves, as the tables' widths and the window have it."""
    Hk, page, D = s.k.shape[1:]
    left = window - max(0, (s.cols - s.ptable.shape[1]) * page)
    return (len(s.lens) - len(s.plens)) * min(left, s.ptable.shape[1] * page) * Hk * D * 4 / 1e6


def _compare(s, window, scale=0.1):
    from attention_nn_amd import paged
    kc, vc, table, starts, lens, gr, pt, pl = s.dev()
    got, lse = paged.attention_shared(s.q.cuda(), kc, vc, table, starts, lens, gr, pt, pl, scale, window, True)
    ref, rlse, tol, ltol = R.attention_whole(s.q, s.k, s.v, s.table, s.starts, s.lens, scale, window)
    got, lse = got.cpu().double(), lse.cpu().double()
    fine = torch.isfinite(ref)
    assert torch.equal(torch.isfinite(got), fine) and torch.equal(torch.isnan(got), torch.isnan(ref))
    assert ((got - ref).abs()[fine] <= tol[fine]).all()
    same = lse == rlse      # -inf of rows that see nothing
    assert ((lse - rlse).abs() <= ltol)[~same].all()
    return got


SHAPES = [
    # prefix, [(new, own)], heads, window
    (5000, [(1, 1 + 7 * i) for i in range(8)], (12, 12, 128), 4000),
    (5000, [(1 + i % 16, 20 + 70 * i) for i in range(9)], (12, 12, 128), 4300),
    (4000, [(1 + i % 3, 3 + i) for i in range(24)], (16, 8, 64), 3600),
    (4100, [(40, 50), *[(1, 60 - i) for i in range(11)]], (12, 12, 128), 2600),
    (3000, [(16, 16)] * 11, (24, 12, 128), 2700),
]


@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_windows(i):
    prefix, members, (H, Hk, D), window = SHAPES[i]
    s = Setup([(prefix, members)], H=H, Hk=Hk, D=D, page=64, seed=i)
    assert _mb(s, window) >= 160 and s.N <= 16 * len(s.lens)
    _compare(s, window)


def test_tokens_inside_the_prefix():
    """Some sequences' tokens lie within the prefix, and see of it what the others do not."""
    s = Setup([(5000, [(1 + i % 4, 4 + i) for i in range(9)])], H=12, Hk=12, page=64, seed=7)
    window = 3700
    assert _mb(s, window) >= 160
    for i, n in ((0, 300), (3, 64), (5, 1), (8, 4999)):
        s.lens[i] = n
    got = _compare(s, window)
    a, b = s.starts[5], s.starts[6]         # two tokens, one entry: the first sees nothing
    assert b - a == 2 and (got[a] == 0).all() and not (got[a + 1] == 0).all()


@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_what_is_not_finite_in_front_of_the_windows(bad):
    """Of the prefix's entries that no window reaches, and that some do."""
    s = Setup([(5000, [(1, 1 + 40 * i) for i in range(9)])], H=12, Hk=12, page=64, seed=3)
    window = 4100
    assert _mb(s, window) >= 160
    for e in (0, 700, 1100):    # the first entries seen are 901 .. 1221
        s.v[s.ptable[0, e // 64], :, e % 64, 5] = bad
    s.k[s.ptable[0, 3], :, 2] = math.nan
    got = _compare(s, window)
    assert not torch.isfinite(got).all() and torch.isfinite(got[-1]).all()
