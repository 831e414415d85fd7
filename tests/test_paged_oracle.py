"""The oracle's paged attention and weights of whole sequences against those formed
token by token, and its bounds: what they must not let pass."""

import math

import pytest
import torch

import oracle.ref_paged as R

BF = torch.bfloat16


def _inputs(new, lens, H, Hk, D, page, seed=0):
    g = torch.Generator().manual_seed(seed)
    S, cols = len(lens), -(-max(max(lens), 1) // page)
    order = torch.randperm(S * cols + 2, generator=g).to(torch.int32)
    k = torch.randn((S * cols + 2, Hk, page, D), generator=g)
    k = (k / torch.sqrt((k * k).mean(-1, keepdim=True))).to(BF)
    v = torch.randn(k.shape, generator=g).to(BF)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    q = torch.randn((starts[-1], H, D), generator=g).to(BF)
    w = torch.rand((S, cols * page), generator=g)
    return q, k, v, order[:S * cols].view(S, cols), starts, w


@pytest.mark.parametrize("window", [0, 5])
@pytest.mark.parametrize("new,lens,H,Hk,D", [([3, 0, 2], [20, 4, 2], 4, 2, 64), ([5, 4], [3, 0], 2, 2, 64),
                                             ([17], [40], 3, 1, 128)])
def test_whole_sequences(new, lens, H, Hk, D, window):
    q, k, v, table, starts, w = _inputs(new, lens, H, Hk, D, 16)
    a = R.attention(q, k, v, table, starts, lens, 0.1, window)
    b = R.attention_whole(q, k, v, table, starts, lens, 0.1, window)
    assert torch.allclose(a[0], b[0], rtol=1e-12, atol=1e-12)
    seen = a[1] > -math.inf
    assert torch.equal(seen, b[1] > -math.inf) and torch.allclose(a[1][seen], b[1][seen], rtol=1e-12)
    assert (b[2] <= a[2] * (1 + 1e-9) + 1e-30).all() and torch.allclose(a[3][seen], b[3][seen])
    lse = torch.where(seen, a[1], 0.0).float()
    for x, y in zip(R.weight(q, lse, k, table, starts, lens, w, 0.1, window),
                    R.weight_whole(q, lse, k, table, starts, lens, w, 0.1, window)):
        assert torch.allclose(x, y, rtol=1e-9, atol=1e-12)


def test_infinities_stay_with_what_sees_them():
    q, k, v, table, starts, _ = _inputs([4], [20], 2, 2, 64, 16)
    v[int(table[0, 1]), 0, 2, 7] = math.inf   # entry 18: seen by the last two tokens
    out, _, tol, _ = R.attention_whole(q, k, v, table, starts, [20], 0.1, 0)
    assert torch.isfinite(tol[:2]).all() and int((~torch.isfinite(tol)).sum()) == 2
    bad = ~torch.isfinite(out)
    assert (out[2:, 0, 7] == math.inf).all() and int(bad.sum()) == 2


def test_one_half_of_the_weights_passes_the_bound_of_two():
    """Weights rounded to bf16 once are outside the bounds that rows of short
    sequences are held to."""
    q, k, v, table, starts, _ = _inputs([1] * 6, [2, 3, 5, 9, 17, 30], 6, 6, 64, 16)
    ref, _, tol, _ = R.attention_whole(q, k, v, table, starts, [2, 3, 5, 9, 17, 30], 0.1, 0)
    outside = 0
    for n, s, e in R.tokens(starts, [2, 3, 5, 9, 17, 30], 32):
        for h in range(6):
            x = 0.1 * (R.entries(k, table[s], e + 1)[:, h] @ q[n, h].double())
            p = torch.exp(x - x.max())
            got = (p.to(BF).double() @ R.entries(v, table[s], e + 1)[:, h]) / p.sum()
            outside += int(((got.to(BF).double() - ref[n, h]).abs() > tol[n, h]).sum())
    assert outside > 20
