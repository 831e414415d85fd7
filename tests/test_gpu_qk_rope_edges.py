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


def _inputs(dtype, B=2, T=5, H=4, Hk=2, D=64):
    g = torch.Generator().manual_seed(3)
    a = torch.rand((T + 3, D // 4), generator=g) * 6.28
    x = [torch.randn((B, T, n, D), generator=g).to(dtype).cuda() for n in (H, Hk, H, Hk)]
    return (*x, a.cos().cuda(), a.sin().cuda())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_autograd_passes_through(dtype):
    """The gradient that autograd finds is qk_norm_rope_bwd's, for positions of either
    kind; the results are those without it."""
    from attention_nn_amd import kernels as K
    q, k, gq, gk, cs, sn = _inputs(dtype)
    for pos in (3, torch.tensor([0, 2], dtype=torch.int32, device="cuda")):
        want = K.qk_norm_rope(q, k, cs, sn, pos)
        a, b = q.clone().requires_grad_(), k.clone().requires_grad_()
        y = K.qk_norm_rope(a, b, cs, sn, pos)
        assert all(torch.equal(x, w) and x.requires_grad for x, w in zip(y, want))
        d = torch.autograd.grad(y, (a, b), (gq, gk))
        back = K.qk_norm_rope_bwd(gq, gk, q, k, cs, sn, pos)
        assert all(torch.equal(x, w) for x, w in zip(d, back))
        with torch.no_grad():
            assert not any(x.requires_grad for x in K.qk_norm_rope(a, b, cs, sn, pos))


def test_autograd_of_views_and_parts():
    """Gradients of a fused projection's memory, of a broadcast head, of one output
    alone, and of one input alone."""
    from attention_nn_amd import kernels as K
    q, k, gq, gk, cs, sn = _inputs(torch.float32)
    dq, dk = K.qk_norm_rope_bwd(gq, gk, q, k, cs, sn)
    fused = torch.cat((q, k, k), 2).requires_grad_()
    y = K.qk_norm_rope(fused[:, :, :4], fused[:, :, 4:6], cs, sn)
    ((y[0] * gq).sum() + (y[1] * gk).sum()).backward()
    assert torch.equal(fused.grad, torch.cat((dq, dk, torch.zeros_like(k)), 2))
    one = q[:, :, :1].clone().requires_grad_()
    y = K.qk_norm_rope(one.expand(-1, -1, 4, -1), k, cs, sn)
    got, = torch.autograd.grad((y[0] * gq).sum(), one)
    parts = K.qk_norm_rope_bwd(gq, gk, q[:, :, :1].expand(-1, -1, 4, -1), k, cs, sn)[0]
    assert torch.allclose(got, parts.sum(2, keepdim=True), rtol=0, atol=4 * 2.0 ** -23 * float(parts.abs().sum(2).max()))
    a, b = q.clone().requires_grad_(), k.clone().requires_grad_()
    y = K.qk_norm_rope(a, b, cs, sn)
    got = torch.autograd.grad((y[1] * gk).sum(), (a, b))
    assert (got[0] == 0).all() and torch.equal(got[1], dk)
    y = K.qk_norm_rope(a, k, cs, sn)
    got, = torch.autograd.grad(y[0], a, gq)
    assert torch.equal(got, dq) and not y[1].requires_grad
    y = K.qk_norm_rope(q, b, cs, sn)
    got, = torch.autograd.grad(y[1], b, gk)
    assert torch.equal(got, dk) and not y[0].requires_grad


def test_autograd_twice_or_captured_is_refused(monkeypatch):
    from attention_nn_amd import kernels as K
    q, k, gq, gk, cs, sn = _inputs(torch.float32)
    a = q.clone().requires_grad_()
    d, = torch.autograd.grad(K.qk_norm_rope(a, k, cs, sn)[0], a, gq.requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        d.sum().backward()
    y = K.qk_norm_rope(a, k, cs, sn)[0]
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="qk_norm_rope_bwd"):
        torch.autograd.grad(y, a, gq.detach())


@pytest.mark.parametrize("D,dtype", [(4, torch.float32), (64, torch.bfloat16)])
def test_more_rows_than_a_launch_takes(D, dtype):
    """2^26 and some rows, of 256 threads for every four: the first and the last ones,
    and those around each 2^25th."""
    from attention_nn_amd import kernels as K
    n = (1 << 26) + 5
    if torch.cuda.mem_get_info()[0] < 4 * n * D * dtype.itemsize:
        pytest.skip("not enough memory")
    x = torch.zeros((n, 1, 1, D), dtype=dtype, device="cuda")
    at = sorted({i for c in (4, 1 << 25, 1 << 26, n) for i in range(max(0, c - 4), min(n, c + 4))})
    rows = torch.randn((len(at), 1, 1, D), generator=torch.Generator().manual_seed(4)).to(dtype).cuda()
    x[at] = rows
    a = torch.rand((1, D // 4), generator=torch.Generator().manual_seed(1)).cuda()
    cs, sn = a.cos(), a.sin()
    y, _ = K.qk_norm_rope(x, x[:, :, :0], cs, sn)
    want, _ = K.qk_norm_rope(rows, rows[:, :, :0], cs, sn)
    assert torch.equal(y[at], want)
    del y
    y, _ = K.qk_norm_rope_bwd(x, x[:, :, :0], x, x[:, :, :0], cs, sn)
    want, _ = K.qk_norm_rope_bwd(rows, rows[:, :, :0], rows, rows[:, :, :0], cs, sn)
    assert torch.equal(y[at], want)
