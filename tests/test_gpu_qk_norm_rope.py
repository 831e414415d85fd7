"""qk_norm_rope and its gradient against the formula in 64 bits and against
differences, over types, head layouts, strides, positions and odd sizes."""

import pytest
import torch

import oracle.ref_paged as R

pytestmark = pytest.mark.gpu

DT = [torch.float32, torch.bfloat16]
STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def _tables(rows, D, seed=0):
    g = torch.Generator().manual_seed(seed)
    a = torch.rand((rows, D // 4), generator=g) * 6.28
    return torch.cos(a), torch.sin(a)


def _x(seed, dtype, *shape):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _bound(y, dtype, D):
    """One rounding to the type; fp32: the row's scale from a sum of D squares
    (half of D 2^-24 at most, whatever its order) and five operations a value,
    relative to the row's largest value (a turned pair mixes two)."""
    return STEP[dtype] * y.abs() + (D / 2 + 8) * 2.0 ** -24 * y.abs().amax(-1, keepdim=True) * 1.5


SHAPES = [(1, 1, 6, 6, 128), (2, 7, 3, 1, 64), (1, 5, 12, 12, 128), (3, 3, 8, 2, 64), (1, 2, 1, 1, 4),
          (2, 3, 5, 2, 20), (1, 9, 4, 2, 96), (1, 4, 3, 3, 36), (2, 2, 2, 1, 256), (1, 3, 2, 0, 128),
          (1, 2, 2, 1, 512), (1, 67, 2, 2, 64)]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("B,T,H,Hk,D", SHAPES)
def test_forward_and_gradient(dtype, B, T, H, Hk, D):
    from attention_nn_amd import kernels as K
    cs, sn = _tables(T + 5, D)
    q, k = _x(1, dtype, B, T, H, D), _x(2, dtype, B, T, Hk, D)
    gq, gk = _x(3, dtype, B, T, H, D), _x(4, dtype, B, T, Hk, D)
    c, s = cs[5:, None].double(), sn[5:, None].double()
    csg, sng = cs.cuda(), sn.cuda()
    got = K.qk_norm_rope(q.cuda(), k.cuda(), csg, sng, 5)
    for x, y in zip((q, k), got):
        ref = R.norm_rope(x.double(), c, s)
        assert y.dtype == dtype and y.is_contiguous()
        if y.numel():
            assert ((y.cpu().double() - ref).abs() <= _bound(ref, dtype, D)).all()
    dq, dk = K.qk_norm_rope_bwd(gq.cuda(), gk.cuda(), q.cuda(), k.cuda(), csg, sng, 5)
    for x, g, y in ((q, gq, dq), (k, gk, dk)):
        if not y.numel():
            continue
        leaf = x.double().requires_grad_()
        ref, = torch.autograd.grad(R.norm_rope(leaf, c, s), leaf, g.double())
        # r (g' - x f): both parts are as large as r times the gradient's row
        r = 1 / torch.sqrt((x.double() ** 2).mean(-1, keepdim=True) + R.EPS)
        size = r * g.double().abs().amax(-1, keepdim=True) * (1 + (x.double() * r).abs().amax(-1, keepdim=True))
        tol = STEP[dtype] * ref.abs() + (2 * D + 16) * 2.0 ** -24 * size
        assert ((y.cpu().double() - ref).abs() <= tol).all()


def test_gradient_against_differences():
    """The fp32 gradient against central differences of the formula in 64 bits:
    h^2 of them times a third derivative of the order of the gradient."""
    from attention_nn_amd import kernels as K
    q, g = _x(1, torch.float32, 1, 2, 1, 64), _x(2, torch.float32, 1, 2, 1, 64)
    cs, sn = _tables(2, 64)
    k = q.clone()
    dq, _ = K.qk_norm_rope_bwd(g.cuda(), g.cuda(), q.cuda(), k.cuda(), cs.cuda(), sn.cuda())
    h = 1e-4
    for i in range(64):
        up, down = q.double().clone(), q.double().clone()
        up[..., i] += h
        down[..., i] -= h
        c, s = cs[:, None].double(), sn[:, None].double()
        diff = ((R.norm_rope(up, c, s) - R.norm_rope(down, c, s)) * g.double()).sum(-1) / (2 * h)
        assert ((dq[..., i].cpu().double() - diff).abs() <= 1e-5 * g.abs().max()).all()


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("D", [64, 128, 20])
def test_views_and_alignment(dtype, D):
    """Views of a fused projection, a transposed batch, a broadcast head and
    rows that are not 16-byte aligned give the bits of contiguous copies."""
    from attention_nn_amd import kernels as K
    cs, sn = (t.cuda() for t in _tables(9, D))
    fused = _x(5, dtype, 2, 9, 7, D).cuda()
    shifted = torch.empty(2 * 9 * 3 * D + 1, dtype=dtype, device="cuda")[1:].view(2, 9, 3, D)
    shifted.copy_(fused[:, :, :3])
    assert shifted.data_ptr() % 16
    views = [(fused[:, :, :4], fused[:, :, 4:6]), (fused.transpose(0, 1)[:, :, :3], fused.transpose(0, 1)[:, :, 6:]),
             (fused[:, :, :1].expand(2, 9, 5, D), fused[:, :, 2:4]), (shifted, shifted[:, :, :1]),
             (fused[:, ::2, :3], fused[:, ::2, 5:])]
    for q, k in views:
        want = K.qk_norm_rope(q.contiguous(), k.contiguous(), cs, sn)
        back = K.qk_norm_rope_bwd(k[:, :, :1].expand_as(q), k, q, k, cs, sn)
        plain = K.qk_norm_rope_bwd(k[:, :, :1].expand_as(q).contiguous(), k.contiguous(), q.contiguous(),
                                   k.contiguous(), cs, sn)
        for a, b in zip((*K.qk_norm_rope(q, k, cs, sn), *back), (*want, *plain)):
            # rows that are not aligned take the form for any alignment, whose sums
            # run in another order: an fp32 rounding of the row's scale apart
            tol = (STEP[dtype] * 2 + D * 2.0 ** -23) * b.float().abs().amax(-1, keepdim=True) * 2
            assert ((a.float() - b.float()).abs() <= tol).all()


def test_positions():
    """A start for all, one for each batch row, one for each token; outside the
    tables the nearest row."""
    from attention_nn_amd import kernels as K
    cs, sn = (t.cuda() for t in _tables(32, 64))
    q, k = _x(1, torch.float32, 3, 4, 2, 64).cuda(), _x(2, torch.float32, 3, 4, 1, 64).cuda()
    for starts in ([7, 7, 7], [0, 3, 28]):
        p = torch.tensor(starts, dtype=torch.int32, device="cuda")
        each = (p[:, None] + torch.arange(4, device="cuda")).to(torch.int32)
        a, b = K.qk_norm_rope(q, k, cs, sn, p), K.qk_norm_rope(q, k, cs, sn, each)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        for i, s in enumerate(starts):
            one = K.qk_norm_rope(q[i:i + 1], k[i:i + 1], cs, sn, s)
            assert torch.equal(one[0], a[0][i:i + 1]) and torch.equal(one[1], a[1][i:i + 1])
    far = torch.tensor([[-5, 0, 31, 1000]] * 3, dtype=torch.int32, device="cuda")
    near = far.clamp(0, 31)
    assert torch.equal(K.qk_norm_rope(q, k, cs, sn, far)[0], K.qk_norm_rope(q, k, cs, sn, near)[0])


def test_extremes():
    """A row of zeros gives zeros, a huge one stays finite where its squares do,
    an infinity or a NaN stays in its own row."""
    from attention_nn_amd import kernels as K
    cs, sn = (t.cuda() for t in _tables(4, 128))
    q = _x(1, torch.float32, 1, 4, 3, 128)
    q[0, 0, 0] = 0.0
    q[0, 1, 1] *= 1e17
    q[0, 2, 2, 5] = float("nan")
    q[0, 3, 0, 70] = float("inf")
    y, _ = K.qk_norm_rope(q.cuda(), q.cuda(), cs, sn)
    y = y.cpu()
    assert (y[0, 0, 0] == 0).all() and torch.isfinite(y[0, 1]).all()
    good = torch.ones(1, 4, 3, dtype=torch.bool)
    good[0, 2, 2] = good[0, 3, 0] = False
    assert torch.isfinite(y[good]).all() and torch.isnan(y[0, 2, 2]).any()


def test_empty():
    from attention_nn_amd import kernels as K
    cs, sn = (t.cuda() for t in _tables(4, 64))
    for B, T in ((0, 3), (2, 0)):
        q = torch.empty(B, T, 2, 64, device="cuda")
        a, b = K.qk_norm_rope(q, q, cs, sn)
        assert a.shape == q.shape and b.shape == q.shape


def test_gradient_replayed_from_a_graph():
    from attention_nn_amd import kernels as K
    cs, sn = (t.cuda() for t in _tables(8, 128))
    q, k = (_x(i, torch.bfloat16, 2, 8, n, 128).cuda() for i, n in ((1, 6), (2, 2)))
    gq, gk = torch.empty_like(q), torch.empty_like(k)
    K.qk_norm_rope_bwd(gq, gk, q, k, cs, sn)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = K.qk_norm_rope(q, k, cs, sn)
        d = K.qk_norm_rope_bwd(gq, gk, q, k, cs, sn)
    for i in range(4):
        for x in (q, k, gq, gk):
            x.copy_(_x(10 + i, torch.bfloat16, *x.shape))
        graph.replay()
        want = (*K.qk_norm_rope(q, k, cs, sn), *K.qk_norm_rope_bwd(gq, gk, q, k, cs, sn))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((*y, *d), want))
