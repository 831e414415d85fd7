"""A token of each row of logits (kernels.sample_logits) against the definition in
64 bits and more.

The tokens have to be equal: the random numbers below lie no nearer to a border
than the sums are exact.  A logarithm is rounded once to fp32, 2^-24 of its size,
and its two parts are formed in 64 bits; the sum of the weights is off by at most
half of 2^-F an entry, F = 62 - log2(entries): below 2^-26 of the largest weight,
which is one, for the 2^17 entries of the widest row here."""

import math

import pytest
import torch

import oracle.ref_serve as R

pytestmark = pytest.mark.gpu
BF, F32, I32 = torch.bfloat16, torch.float32, torch.int32


def _check(x, u, got, each):
    ids, lp = (t.cpu() for t in got)
    assert ids.dtype is I32 and lp.dtype is F32
    for r in range(x.shape[0]):
        kw = {k: (v[r].item() if isinstance(v, torch.Tensor) else v) for k, v in each.items()}
        i, ref = R.sample(x[r].float().numpy(), u[r].item(), **kw)
        assert ids[r].item() == i, (r, kw, u[r].item(), i, ids[r].item())
        if ref == -math.inf:
            assert lp[r].item() == ref
        else:
            assert abs(lp[r].item() - ref) <= abs(ref) * 2.0 ** -24 + 2.0 ** -26, (r, kw)


def _logits(rows, cols, seed, dtype, kind="model"):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((rows, cols), generator=g) * 2.0
    if kind == "model":
        x += torch.where(torch.rand((rows, cols), generator=g) < 0.003, 6.0 * torch.rand((rows, cols), generator=g), 0.0)
        x = 23.0 * torch.sigmoid((x + 5.0) / 7.5)
    elif kind == "flat":
        x = x * 0.01
    elif kind == "coarse":      # a handful of values, many times each
        x = torch.floor(x)
    elif kind == "masked":      # most entries forbidden, some by the type's lowest value
        x = torch.where(torch.rand((rows, cols), generator=g) < 0.9, -math.inf, x)
        x = torch.where(torch.rand((rows, cols), generator=g) < 0.3, torch.finfo(dtype).min, x)
    elif kind == "wide":        # both signs, from tiny to large
        x = x * 10.0 ** torch.randint(-6, 2, (rows, cols), generator=g)
    return x.to(dtype), torch.rand(rows, generator=g)


SETTINGS = [
    dict(), dict(temperature=0.0), dict(temperature=0.8, top_k=50), dict(top_p=0.9), dict(min_p=0.05),
    dict(temperature=0.3, top_k=1), dict(top_k=7, top_p=0.5), dict(temperature=1.7, top_p=0.999),
    dict(temperature=0.7, top_k=1000, top_p=0.8, min_p=0.001), dict(top_p=0.0), dict(top_p=1e-9), dict(min_p=1.0),
    dict(min_p=7.0, top_p=2.0), dict(temperature=40.0, top_k=100), dict(temperature=1e-6), dict(temperature=1e30, top_p=0.5),
]


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("kind", ["model", "flat", "coarse", "masked", "wide"])
@pytest.mark.parametrize("cols", [1, 2, 5, 63, 1009, 4097])
def test_settings(cols, kind, dtype):
    from attention_nn_amd import kernels
    x, _ = _logits(4, cols, cols, dtype, kind)
    xd = x.cuda()
    for j, kw in enumerate(SETTINGS):
        u = torch.rand(4, generator=torch.Generator().manual_seed(100 * cols + j))
        _check(x, u, kernels.sample_logits(xd, u.cuda(), want_logprob=True, **kw), kw)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("kind", ["model", "flat", "coarse", "masked", "wide"])
@pytest.mark.parametrize("cols", [9000, 50257, 70001])
def test_long_rows(cols, kind, dtype):
    from attention_nn_amd import kernels
    x, _ = _logits(2, cols, cols, dtype, kind)
    xd = x.cuda()
    for j, kw in enumerate([dict(), dict(temperature=0.8, top_k=50), dict(top_p=0.9), dict(top_k=5000, top_p=0.97),
                            dict(temperature=0.6, min_p=0.1), dict(top_k=cols - 1), dict(temperature=0.0),
                            dict(temperature=0.9, top_k=897, top_p=0.6, min_p=0.01)]):
        u = torch.rand(2, generator=torch.Generator().manual_seed(7 * cols + j))
        _check(x, u, kernels.sample_logits(xd, u.cuda(), want_logprob=True, **kw), kw)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_a_setting_for_each_row(dtype):
    from attention_nn_amd import kernels
    rows = 37
    x, u = _logits(rows, 6007, 5, dtype)
    g = torch.Generator().manual_seed(9)
    each = dict(temperature=torch.rand(rows, generator=g) * 1.5, top_k=torch.randint(-2, 6100, (rows,), generator=g).to(I32),
                top_p=torch.rand(rows, generator=g) * 1.2, min_p=torch.rand(rows, generator=g) * 0.2)
    each["temperature"][::5] = torch.tensor([0.0, -1.0, math.nan, 1e-40, 0.5, -0.0, 2.0, 1.0])
    each["top_p"][3], each["top_p"][4], each["min_p"][6], each["min_p"][7] = math.nan, -1.0, math.nan, -2.0
    got = kernels.sample_logits(x.cuda(), u.cuda(), want_logprob=True, **{k: v.cuda() for k, v in each.items()})
    plain = {**each, "min_p": torch.nan_to_num(each["min_p"], 0.0), "top_p": torch.nan_to_num(each["top_p"], 1.0)}
    _check(x, u, got, plain)
    only = kernels.sample_logits(x.cuda(), u.cuda(), **{k: v.cuda() for k, v in each.items()})
    assert torch.equal(only, got[0])


@pytest.mark.parametrize("u", [0.0, 1.0 - 2.0 ** -24, 1.0, 3.0, -1.0, math.nan, 0.5])
def test_random_numbers_at_and_past_the_ends(u):
    from attention_nn_amd import kernels
    for cols, kind in ((3, "model"), (777, "model"), (50257, "flat"), (50257, "model")):
        x, _ = _logits(2, cols, 3, F32, kind)
        uu = torch.full((2,), u)
        for kw in (dict(), dict(top_k=40), dict(top_p=0.7)):
            _check(x, uu, kernels.sample_logits(x.cuda(), uu.cuda(), want_logprob=True, **kw), kw)


def test_rows_without_a_choice():
    from attention_nn_amd import kernels
    inf, nan = math.inf, math.nan
    x = torch.tensor([[-inf] * 5, [nan] * 5, [nan, -inf, -2.0, nan, -inf], [inf, 1.0, inf, nan, -inf],
                      [-0.0, 0.0, -1e-45, 0.0, -0.0], [torch.finfo(F32).min] * 5, [torch.finfo(F32).max, 0, -inf, inf, 1]])
    for dtype in (F32, BF):
        y = x.to(dtype)
        for kw in (dict(), dict(temperature=0.0), dict(top_k=2), dict(top_p=0.6), dict(min_p=0.5, temperature=3.0)):
            for seed in range(4):
                u = torch.rand(7, generator=torch.Generator().manual_seed(seed))
                _check(y, u, kernels.sample_logits(y.cuda(), u.cuda(), want_logprob=True, **kw), kw)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_strides_and_alignment(dtype):
    from attention_nn_amd import kernels
    base, u = _logits(3, 9000, 11, dtype)
    for first in (0, 1, 3, 5):
        for width in (1, 6, 4099, 8990):
            view = base.cuda()[:, first:first + width]
            _check(base[:, first:first + width], u, kernels.sample_logits(view, u.cuda(), top_p=0.9, want_logprob=True),
                   dict(top_p=0.9))
    same = base[:1, :500].cuda().expand(3, 500)          # a row stride of 0
    _check(base[:1, :500].expand(3, 500), u, kernels.sample_logits(same, u.cuda(), top_k=9, want_logprob=True), dict(top_k=9))
    turned = base[:, :500].t().contiguous().cuda().t()   # entries apart
    _check(base[:, :500], u, kernels.sample_logits(turned, u.cuda(), want_logprob=True), dict())
    odd = torch.zeros(7, device="cuda")[1:].view(2, 3)[:, 1]    # random numbers apart
    assert kernels.sample_logits(base[:2].cuda(), odd).tolist() == [
        R.sample(base[r].float().numpy(), 0.0)[0] for r in range(2)]


def test_many_rows_and_none():
    from attention_nn_amd import kernels
    x, u = _logits(3000, 40, 1, F32)
    _check(x, u, kernels.sample_logits(x.cuda(), u.cuda(), top_p=0.8, want_logprob=True), dict(top_p=0.8))
    assert kernels.sample_logits(x.cuda()[:0], u.cuda()[:0]).shape == (0,)


def test_widest_row():
    from attention_nn_amd import kernels
    x, u = _logits(1, 1 << 20, 1, BF)
    for kw in (dict(), dict(top_k=100), dict(top_p=0.5)):
        ids, lp = kernels.sample_logits(x.cuda(), u.cuda(), want_logprob=True, **kw)
        i, ref = R.sample(x[0].float().numpy(), u[0].item(), **kw)
        # sums to half of 2^-42 an entry: 2^-23 of the largest weight at most
        assert ids.item() == i and abs(lp.item() - ref) <= abs(ref) * 2.0 ** -24 + 2.0 ** -23


def test_graph_and_other_stream():
    from attention_nn_amd import kernels
    x, u = _logits(5, 50257, 2, F32)
    xd, ud = x.cuda(), u.cuda()
    want = kernels.sample_logits(xd, ud, 0.9, 40, 0.95, want_logprob=True)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = kernels.sample_logits(xd, ud, 0.9, 40, 0.95, want_logprob=True)
    st.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ids, lp = kernels.sample_logits(xd, ud, 0.9, 40, 0.95, want_logprob=True)
    for seed in range(4):
        y, v = _logits(5, 50257, 30 + seed, F32)
        xd.copy_(y), ud.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        _check(y, v, (ids, lp), dict(temperature=0.9, top_k=40, top_p=0.95))
        eager = kernels.sample_logits(xd, ud, 0.9, 40, 0.95)
        assert torch.equal(eager, ids)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("peaks", [1, 5, 30, 90])
@pytest.mark.parametrize("cols", [9000, 50257, 53300, 70001, 131072])
def test_few_entries_hold_what_top_p_keeps(cols, peaks, dtype):
    """Far more entries weigh something than a list holds, and what top_p keeps of them
    lies with a few threads, of no particular wave or lane."""
    from attention_nn_amd import kernels
    g = torch.Generator().manual_seed(cols + peaks)
    x = 0.3 * torch.randn((6, cols), generator=g)
    for r in range(6):
        at = torch.randperm(cols, generator=g)[:peaks]
        if r == 4:
            at = cols - 1 - torch.arange(peaks)     # all with the last wave
        x[r, at] = 12.0 + torch.rand(peaks, generator=g)
    x = x.to(dtype)
    u = torch.rand(6, generator=g)
    for kw in (dict(top_p=0.3), dict(top_p=0.9 if peaks > 5 else 0.5), dict(top_p=0.6, top_k=cols - 1)):
        _check(x, u, kernels.sample_logits(x.cuda(), u.cuda(), want_logprob=True, **kw), kw)
