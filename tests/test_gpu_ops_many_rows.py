"""Row operators on more rows than one launch's grid holds: 2^32 threads, of which a
row takes 64 or 256."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _rows(n, per, dim, dtype):
    """Zeros but for rows around the ends and each `per` rows: all, and those."""
    if torch.cuda.mem_get_info()[0] < 4 * n * dim * dtype.itemsize:
        pytest.skip("not enough memory")
    at = sorted({i for c in (2, *range(per, n, per), n) for i in range(max(0, c - 2), min(n, c + 2))})
    x = torch.zeros((n, dim), dtype=dtype, device="cuda")
    some = torch.randn((len(at), dim), generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    x[at] = some
    return x, some, at


@pytest.mark.parametrize("n,dim,dtype", [((1 << 24) + 5, 6, torch.float32), ((1 << 26) + 5, 8, torch.bfloat16)])
def test_rms(n, dim, dtype):
    from attention_nn_amd import kernels as K
    x, some, at = _rows(n, 1 << 23, dim, dtype)
    assert torch.equal(K.rms(x)[at], K.rms(some))


@pytest.mark.parametrize("offset", [0, 1])
def test_rope(offset):
    from attention_nn_amd import kernels as K
    n = (1 << 26) + 5
    x, some, at = _rows(n, 1 << 25, 4, torch.bfloat16)
    if offset:   # not aligned to a pair
        buf = torch.empty(n * 4 + 1, dtype=x.dtype, device="cuda")[1:].view(n, 4)
        buf.copy_(x)
        x = buf
    a = torch.rand((1, 1), generator=torch.Generator().manual_seed(1)).cuda()
    got = K.rope_ht(x.view(n, 1, 1, 4), a.cos(), a.sin())
    want = K.rope_ht(some.view(-1, 1, 1, 4), a.cos(), a.sin())
    assert torch.equal(got.view(n, 4)[at], want.view(-1, 4))
