"""Tokens of rows whose thresholds lie beside zero (kernels.sample_logits): zeros of both
signs and subnormal numbers below them, at temperatures that leave them all about one weight."""

import math

import pytest
import torch

from tests.test_gpu_sample_logits import _check

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32

# the least magnitude below a normal number's of each type, and a few others
TINY = {F32: [-1e-45, -3e-45, -2e-42, -1.1e-38], BF: [-9.2e-41, -1.9e-40, -5e-39, -1.1e-38]}


def _rows(zeros, others, dtype, seed):
    """Four rows of 0, -0 and negative subnormals, shuffled: of one, of all values, beside a few
    larger entries, and masked in part."""
    g = torch.Generator().manual_seed(seed)
    n = zeros + others
    x = torch.zeros((4, n))
    x[:, :zeros // 2] = -0.0
    x[:, zeros:] = TINY[dtype][0]
    x[1, zeros:] = torch.tensor(TINY[dtype])[torch.randint(0, 4, (others,), generator=g)]
    x[2, :3] = torch.tensor([2.0, 1e-30, 1.0])[:min(3, n)]
    x[3, ::7] = -math.inf
    x[3, 5::11] = math.nan
    return torch.stack([r[torch.randperm(n, generator=g)] for r in x]).to(dtype)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("zeros,others", [(100, 200), (200, 100), (700, 1400), (6000, 3000), (10000, 20000), (20000, 10000),
                                          (30000, 40000)])
def test_zeros_beside_subnormals(zeros, others, dtype):
    from attention_nn_amd import kernels
    x = _rows(zeros, others, dtype, zeros)
    n = zeros + others
    for j, kw in enumerate([dict(temperature=math.inf, top_p=0.5), dict(temperature=1.2e37, top_p=0.9),
                            dict(temperature=3e38, top_p=0.2, top_k=n - 1), dict(temperature=math.inf, top_k=zeros + others // 2),
                            dict(temperature=math.inf, top_k=zeros // 2, top_p=0.6), dict(temperature=1.0, top_p=0.4),
                            dict(temperature=math.inf, min_p=1.0, top_p=0.99)]):
        u = torch.rand(4, generator=torch.Generator().manual_seed(31 * n + j))
        _check(x, u, kernels.sample_logits(x.cuda(), u.cuda(), want_logprob=True, **kw), kw)
