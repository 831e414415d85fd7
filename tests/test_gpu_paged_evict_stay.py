"""Eviction in place: what stays where it is, is not written again."""

import statistics

import pytest
import torch

import oracle.ref_paged as R
from tests.test_gpu_paged import I32, Setup, _gen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens,keep,first", [
    # sequences' lengths, entries kept, and from which entry on weights are such that some go
    ([40, 64, 17], 64, 0), ([1300, 2100, 5], 1024, 1000), ([1300, 2100, 5], 1024, 1023), ([1300], 1024, 1024),
    ([1300], 1024, 0), ([5000, 4100, 4096], 4096, 4095), ([5000, 4100], 4096, 1), ([5000, 3000], 3000, 2999),
    ([9000], 5000, 4321), ([33], 32, 31), ([2], 1, 0), ([2], 1, 1), ([1], 1, 0), ([0, 3], 1, 0)])
def test_prefixes_that_stay(lens, keep, first):
    """Entries before `first` outweigh the others, so the prefix that does not move
    ends there or behind, at every place that the search for its end may miss."""
    from attention_nn_amd import paged
    s = Setup([0] * len(lens), lens, H=1, Hk=1, D=64, page=32, garbage=False, more_cols=-(-keep // 32))
    w = torch.rand((len(lens), s.cols * 32), generator=_gen(first))
    w[:, :first] += 2.0
    kc, vc, table, _, n = s.dev()
    ref = R.evict(s.k, s.v, s.table, lens, w, keep, 0, s.table)
    got = paged.evict(kc, vc, table, n, w.cuda(), keep)
    for a, b in zip((*got, kc, vc), ref):
        assert torch.equal(a.cpu(), b)


def test_what_stays_is_not_copied():
    """Sequences that are short enough cost less than a third of those that move."""
    from attention_nn_amd import paged
    k = torch.zeros((64 * 128 + 1, 6, 32, 128), dtype=torch.bfloat16, device="cuda")
    v = k.clone()
    table = torch.arange(64 * 128, dtype=I32, device="cuda").view(64, 128)
    w = torch.rand((64, 4096), device="cuda")
    w[:, 0] = -1.0

    def us(entries, keep):
        lens = torch.full((64,), entries, dtype=I32, device="cuda")
        times = []
        for _ in range(9):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            for _ in range(5):
                paged.evict(k, v, table, lens, w, keep)
            b.record()
            b.synchronize()
            times.append(a.elapsed_time(b) * 200)
        return statistics.median(times)

    assert us(4095, 4095) < us(4096, 4095) / 3
