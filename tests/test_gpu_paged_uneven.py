"""Paged attention of calls with no more tokens than sequences whose tokens are not
spread evenly: a captured step of many slots, replayed with a chunk in one of them."""

import statistics

import pytest
import torch

import oracle.ref_paged as R
from tests.test_gpu_paged import Setup

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new,lens,kw", [
    ([0] * 7 + [60] + [0] * 60, [5] * 7 + [90] + [0] * 60, dict(H=2, Hk=2)),
    ([1, 0, 1, 37, 2, 0, 18, 1] + [0] * 70, [9, 3, 200, 1500, 40, 0, 18, 77] + [11] * 70, dict(H=4, Hk=2, D=64)),
    ([3, 17] + [0] * 20, [300, 290] + [4] * 20, dict(H=6, Hk=1, window=50)),
    ([1], [700], dict(H=40, Hk=1, D=64)),
    ([1, 1, 0, 2, 1], [70, 1300, 2, 33, 5], dict(H=34, Hk=2, D=64)),
    ([20] + [0] * 19, [12] + [0] * 19, dict(H=2, Hk=2)),   # the first tokens see nothing
])
def test_uneven(new, lens, kw):
    from attention_nn_amd import paged
    kw = dict(kw)
    window = kw.pop("window", 0)
    s = Setup(new, lens, **kw)
    kc, vc, table, starts, ln = s.dev()
    ref, rlse, tol, ltol = R.attention_whole(s.q, s.k, s.v, s.table, s.starts, s.lens, 0.1, window)
    got, lse = paged.attention(s.q.cuda(), kc, vc, table, starts, ln, 0.1, window, True)
    assert ((got.cpu().double() - ref).abs() <= tol).all()
    seen = rlse > -float("inf")
    assert torch.equal(lse.cpu() > -float("inf"), seen)
    assert ((lse.cpu().double() - rlse).abs()[seen] <= ltol[seen]).all()


def test_a_chunk_among_empty_sequences_is_shared_out():
    """512 tokens of one sequence beside 511 empty ones: within five times the chunk by
    itself (one work-group for a sequence's rows takes more than twenty times)."""
    from attention_nn_amd import paged

    def us(empty):
        s = Setup([512] + [0] * empty, [2000] + [0] * empty, garbage=False)
        q, (kc, vc, table, starts, lens) = s.q.cuda(), s.dev()
        times = []
        for _ in range(9):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            for _ in range(5):
                paged.attention(q, kc, vc, table, starts, lens, 0.1)
            b.record()
            b.synchronize()
            times.append(a.elapsed_time(b) * 200)
        return statistics.median(times)

    assert us(511) < 5 * us(0)
