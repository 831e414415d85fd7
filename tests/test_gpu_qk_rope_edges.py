"""qk_norm_rope at the ends of what its arguments may be."""

import pytest
import torch

pytestmark = pytest.mark.gpu

INT_MAX = (1 << 31) - 1


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 20])
def test_starts_at_the_ends_of_32_bits(D, dtype):
    """A start from which a token's position passes 32 bits takes the tables' last
    row, as every position past them does."""
    from attention_nn_amd import kernels as K
    a = torch.rand((9, D // 4), generator=torch.Generator().manual_seed(1)) * 6.28
    cs, sn = a.cos().cuda(), a.sin().cuda()
    g = torch.Generator().manual_seed(2)
    q, k = (torch.randn((5, 4, n, D), generator=g).to(dtype).cuda() for n in (3, 1))
    starts = torch.tensor([INT_MAX, INT_MAX - 1, INT_MAX - 3, -INT_MAX - 1, -2], dtype=torch.int32, device="cuda")
    each = torch.tensor([[8] * 4, [8] * 4, [8] * 4, [0] * 4, [0, 0, 0, 1]], dtype=torch.int32, device="cuda")
    for x, y in zip(K.qk_norm_rope(q, k, cs, sn, starts) + K.qk_norm_rope_bwd(q, k, q, k, cs, sn, starts),
                    K.qk_norm_rope(q, k, cs, sn, each) + K.qk_norm_rope_bwd(q, k, q, k, cs, sn, each)):
        assert torch.equal(x, y)
