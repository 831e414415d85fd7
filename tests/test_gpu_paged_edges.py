"""The paged cache's operators where values leave the ordinary: infinities that a
token sees, alone in its sequence or beside others."""

import math

import pytest
import torch

import oracle.ref_paged as R
from tests.test_gpu_paged import Setup

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("H,Hk,D", [(2, 2, 128), (2, 1, 64)])
@pytest.mark.parametrize("new,length", [(1, 1), (1, 5), (1, 33), (1, 777), (1, 3000), (2, 40), (2, 3000), (40, 100),
                                        (40, 3000)])
def test_infinities_that_a_token_sees(new, length, H, Hk, D):
    """An infinite value makes its dimension infinite for the tokens that see it, two
    of unlike sign or a NaN make it NaN, as the sum of the products does; the other
    dimensions are as they were."""
    from attention_nn_amd import paged
    s = Setup([new], [length], H=H, Hk=Hk, D=D, garbage=False)
    first, last = max(0, length - new - 2), length - 1
    for e, dim, value in ((first, 3, math.inf), (last, 60, -math.inf), (first, 17, math.inf), (last, 17, -math.inf),
                          (first, 33, math.nan)):
        s.v[int(s.table[0, e // 16]), :, e % 16, dim] = value
    if first == last:
        s.v[int(s.table[0, 0]), :, last % 16, 17] = math.nan
    kc, vc, table, starts, lens = s.dev()
    ref, rlse, tol, ltol = R.attention_whole(s.q, s.k, s.v, s.table, s.starts, s.lens, 0.1, 0)
    got, lse = paged.attention(s.q.cuda(), kc, vc, table, starts, lens, 0.1, want_lse=True)
    got = got.cpu().double()
    fine = torch.isfinite(ref)
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    assert torch.equal(got[got.abs() == math.inf], ref[ref.abs() == math.inf])
    assert ((got - ref).abs()[fine] <= tol[fine]).all()
    assert ((lse.cpu().double() - rlse).abs() <= ltol).all()


def test_a_result_in_the_queries_gaps():
    """Rows of queries far enough apart hold the result between them; on one of them
    it is refused."""
    from attention_nn_amd import paged
    s = Setup([2, 1], [20, 30], H=4, Hk=2, D=64, garbage=False)
    kc, vc, table, starts, lens = s.dev()
    want = paged.attention(s.q.cuda(), kc, vc, table, starts, lens, 0.1)
    buf = torch.zeros(3 * 2048, dtype=torch.bfloat16, device="cuda")
    q = buf.as_strided((3, 4, 64), (2048, 64, 1))
    q.copy_(s.q)
    at = lambda i: buf[i:i + 3 * 4 * 64].view(3, 4, 64)
    for i in (2048 + 256, 4096 - 768, 5120):
        assert torch.equal(paged.attention(q, kc, vc, table, starts, lens, 0.1, out=at(i)), want)
        assert torch.equal(q.cpu(), s.q)
    for i in (0, 2048, 2048 + 248, 4096 - 760):
        with pytest.raises(ValueError, match="overlaps"):
            paged.attention(q, kc, vc, table, starts, lens, 0.1, out=at(i))


def test_weights_beside_the_new_ones():
    """Old and new weights as column halves of one tensor, and a broadcast row of old
    ones; what shares some of the rows is refused."""
    from attention_nn_amd import paged
    s = Setup([2, 1], [20, 30], H=4, Hk=2, D=64, garbage=False)
    kc, vc, table, starts, lens = s.dev()
    q, cap = s.q.cuda(), s.cols * 16
    lse = paged.attention(q, kc, vc, table, starts, lens, 0.1, want_lse=True)[1]
    both = torch.rand((2, 2 * cap), device="cuda")
    old, new = both[:, :cap], both[:, cap:]
    was = old.clone()
    want = paged.attention_weight(q, lse, kc, table, starts, lens, was, 0.1)
    assert paged.attention_weight(q, lse, kc, table, starts, lens, old, 0.1, out=new) is new
    assert torch.equal(new, want) and torch.equal(old, was)
    one = was[:1].expand(2, -1)
    assert torch.equal(paged.attention_weight(q, lse, kc, table, starts, lens, one, 0.1),
                       paged.attention_weight(q, lse, kc, table, starts, lens, one.contiguous(), 0.1))
    rows = torch.rand((3, cap), device="cuda")
    for w, out in ((rows[:2], rows[1:]), (rows[1:], rows[:2]), (old, both[:, cap - 1:-1]), (one, was)):
        with pytest.raises(ValueError, match="overlaps|in place"):
            paged.attention_weight(q, lse, kc, table, starts, lens, w, 0.1, out=out)


def test_more_rows_than_a_launch_takes():
    """2^26 and some tokens of one sequence, of which the last ones have entries: the
    tokens around each 2^25th and the last ones are turned, stored and answered."""
    from attention_nn_amd import kernels, paged
    n, cap = (1 << 26) + 5, 48
    if torch.cuda.mem_get_info()[0] < 4 * n * 128:
        pytest.skip("not enough memory")
    x = torch.zeros((n, 1, 64), dtype=torch.bfloat16, device="cuda")
    at = [i for c in (4, 1 << 25, (1 << 26) - cap) for i in range(c - 4, c + 4)] + list(range(n - cap, n))
    rows = torch.randn((len(at), 1, 64), generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).cuda()
    x[at] = rows
    a = torch.rand((1, 16), generator=torch.Generator().manual_seed(1)).cuda()
    cs, sn = a.cos(), a.sin()
    kc, vc = (torch.zeros((3, 1, 16, 64), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    table, starts, lens = (torch.tensor(t, dtype=torch.int32, device="cuda") for t in ([[2, 0, 1]], [0, n], [n]))
    q = paged.append(x, x, x, cs, sn, kc, vc, table, starts, lens)
    want = kernels.qk_norm_rope(rows[None], rows[None], cs, sn, torch.zeros((1, len(at)), dtype=torch.int32, device="cuda"))
    assert torch.equal(q[at], want[0][0])
    k, v = (c[table[0].long()].transpose(1, 2).reshape(cap, 1, 64) for c in (kc, vc))
    assert torch.equal(k, want[1][0, -cap:]) and torch.equal(v, rows[-cap:])
    del x
    y, lse = paged.attention(q, kc, vc, table, starts, lens, 0.1, want_lse=True, out=q.clone())
    last = torch.tensor([0, cap], dtype=torch.int32, device="cuda")
    few, flse = paged.attention(q[-cap:], kc, vc, table, last, last[1:], 0.1, want_lse=True)
    assert torch.equal(lse[-cap:] > -math.inf, flse > -math.inf)
    assert ((lse[-cap:] - flse).abs() <= 1e-5).all()
    # either form rounds the weights to bf16 once, and the result
    assert ((y[-cap:].float() - few.float()).abs() <= 2.0 ** -6 * v.float().abs().amax()).all()
    none = [i for i in at if i < n - cap]
    assert (y[none] == 0).all() and (lse[none] == -math.inf).all()
