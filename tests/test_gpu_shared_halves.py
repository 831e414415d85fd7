"""Weights of attention behind a shared prefix (paged.attention_shared): as two bf16 halves
for all sequences of up to 16 new tokens, of the prefix's entries and of their own."""

import pytest
import torch

from tests.test_shared_halves import SCALE, SHAPES, Halves

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", SHAPES + [(2, 16, 16, 2000, (2, 1, 128)), (40, 1, 20, 900, (4, 4, 128)),
                                            (9, 7, 25, 1500, (12, 3, 64))])
def test_weights_in_two_halves(shape):
    from attention_nn_amd import paged
    S, n, own, prefix, (H, Hk, D) = shape
    s = Halves(S, n, own, prefix, H, Hk, D).widened()
    ref, rlse, tol, ltol = s.expected()

    def i(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")
    got, lse = paged.attention_shared(s.q.cuda(), s.k.cuda(), s.v.cuda(), s.table.cuda(), i(s.starts), i(s.lens),
                                      i(s.groups), s.ptable.cuda(), i(s.plens), SCALE, want_lse=True)
    assert ((got.cpu().double() - ref).abs() <= tol).all()
    assert ((lse.cpu().double() - rlse).abs() <= ltol).all()
