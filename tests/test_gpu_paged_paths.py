"""Paged attention and the weight of its entries at the sizes where other kernels
or other branches of them take a call: parts of few rows beside tiles of many, joined
together and by themselves, walks of more than 64 tiles, shared heads in parts.  Each
case names the kernels that it has to reach."""

import pytest
import torch

import oracle.ref_paged as R
from tests.test_gpu_paged import Setup, _gen

pytestmark = pytest.mark.gpu

# (new tokens, lengths), what differs from 6 x 128 heads, and the kernels that have to run
CASES = [
    # chunks beside decoding past 1024 entries: both kinds come in parts
    dict(new=[40, 1, 2], lens=[1300, 1250, 9], run=("many<128, 1>", "join<128, 1>")),
    dict(new=[40, 1, 2], lens=[1300, 1250, 9], Hk=3, run=("many<128, 1>", "join<128, 1>")),
    dict(new=[40, 1, 2], lens=[1300, 1250, 9], D=64, run=("many<64, 1>", "join<64, 1>")),
    dict(new=[40, 1, 2], lens=[1300, 1250, 9], H=12, Hk=6, D=64, window=1200, run=("many<64, 1>", "join<64, 1>")),
    dict(new=[1, 40, 8], lens=[1300, 1250, 700], H=4, Hk=2, window=1100, run=("many<128, 1>", "join<128, 1>")),
    # as much work as fills the tiles' places: only the few rows come in parts, and
    # the join goes by their sequences
    dict(new=[1300, 1, 2], lens=[1300, 1250, 1111], H=12, Hk=12, page=64, run=("many<128, 2>", "join<128, 1>")),
    dict(new=[1, 1300, 2], lens=[1250, 1300, 1111], H=8, Hk=8, D=64, page=64, run=("many<64, 1>", "join<64, 1>")),
    dict(new=[2, 1300, 1], lens=[1100, 1300, 3], H=8, Hk=4, D=64, page=64, window=1290, run=("many<64, 1>", "join<64, 1>")),
    # shared heads of few rows, in parts
    dict(new=[1], lens=[1280], H=8, Hk=2, D=64, run=("few<64, 4>", "join<64, 1>")),
    dict(new=[2], lens=[1280], H=8, Hk=2, run=("few<128, 4>", "join<128, 1>")),
    dict(new=[1, 2, 0, 3], lens=[3000, 2, 7, 1500], H=10, Hk=2, run=("many<128, 1>", "join<128, 1>")),
    # more than 64 steps a part
    dict(new=[1400], lens=[9000], page=64, run=("many<128, 2>", "join<128, 3>")),
    dict(new=[2000], lens=[10000], H=8, Hk=8, D=64, page=64, run=("many<64, 2>", "join<64, 1>")),
    # and more than 32 chunks a wave of few rows
    dict(new=[1], lens=[300000], H=1, Hk=1, D=64, page=1024, run=("few<64, 4>", "join<64, 1>")),
    dict(new=[1] * 64, lens=[4160] + [4100 - 9 * i for i in range(63)], H=4, Hk=4, D=64, window=4080, run=()),
    # two halves of the weights, where one would show
    dict(new=[1] * 9, lens=[2, 3, 4, 5, 7, 9, 12, 17, 30], D=64, run=("few<64, 8>",)),
    dict(new=[2, 3], lens=[9, 5], H=10, Hk=2, run=("many<128, 1>",)),
    dict(new=[30, 1, 1, 1, 5, 2], lens=[40, 9, 5, 3, 8, 12], run=("many<128, 1>",)),
]


@pytest.mark.parametrize("i", range(len(CASES)))
def test_attention_and_weight(i, traced):
    from attention_nn_amd import paged
    case = dict(CASES[i])
    window, run = case.pop("window", 0), case.pop("run")
    s = Setup(seed=i, **case)
    kc, vc, table, starts, lens = s.dev()
    q = s.q.cuda()
    ref, rlse, tol, ltol = R.attention_whole(s.q, s.k, s.v, s.table, s.starts, s.lens, 0.1, window)
    got = []
    names = traced(lambda: got.append(paged.attention(q, kc, vc, table, starts, lens, 0.1, window, True)))
    for n in run:
        assert any("k_paged_" + n in x for x in names), (n, names)
    for y, lse in got:
        assert ((y.cpu().double() - ref).abs() <= tol).all()
        assert ((lse.cpu().double() - rlse).abs() <= ltol).all()
    y, lse = paged.attention(q, kc, vc, table, starts, lens, 0.1, window, True)
    assert torch.equal(y, got[0][0]) and torch.equal(lse, got[0][1])
    w = torch.rand((len(s.lens), s.cols * s.page), generator=_gen(i))
    out = paged.attention_weight(q, lse, kc, table, starts, lens, w.cuda(), 0.1, window).cpu().double()
    want, bound = R.weight_whole(s.q, lse.cpu(), s.k, s.table, s.starts, s.lens, w, 0.1, window)
    assert ((out - want).abs() <= bound).all()
