"""The paged cache's operators against plain 64-bit implementations: ragged
batches from one token to long chunks, empty sequences, windows, shared heads,
page sizes, strides, garbage behind the sequences, other streams and graphs."""

import math

import pytest
import torch

import oracle.ref_paged as R

pytestmark = pytest.mark.gpu
BF, I32 = torch.bfloat16, torch.int32


def _gen(seed):
    return torch.Generator().manual_seed(seed)


class Setup:
    """A pool of pages in random order; what no sequence uses is NaN in the keys
    and infinite in the values."""

    def __init__(self, new, lens, H=6, Hk=6, D=128, page=16, seed=0, more_cols=0, garbage=True,
                 layout="pages", spare_rows=0, out_cols=0):
        g = _gen(seed)
        S = len(lens)
        self.new, self.lens, self.H, self.Hk, self.D, self.page = new, lens, H, Hk, D, page
        self.cols = max(1, -(-max(max(lens), 1) // page)) + more_cols
        pages = S * (self.cols + out_cols) + 3
        order = torch.randperm(pages, generator=g).to(I32)
        self.table = order[:S * self.cols].view(S, self.cols).contiguous()
        self.out_table = order[S * self.cols:S * (self.cols + out_cols)].view(S, out_cols).contiguous()
        shape = (pages, Hk, page, D)
        k, v = torch.randn(shape, generator=g), torch.randn(shape, generator=g)
        k = k / torch.sqrt((k * k).mean(-1, keepdim=True))
        used = torch.zeros(pages, page, dtype=torch.bool)
        for s, n in enumerate(lens):
            for e in range(max(0, min(n, self.cols * page))):
                used[self.table[s, e // page], e % page] = True
        if garbage:
            k[~used[:, None, :].expand(pages, Hk, page)] = math.nan
            v[~used[:, None, :].expand(pages, Hk, page)] = math.inf
        self.k, self.v = k.to(BF), v.to(BF)
        self.starts = [0]
        for n in new:
            self.starts.append(self.starts[-1] + n)
        self.N = self.starts[-1] + spare_rows
        q = torch.randn((self.N, H, D), generator=g)
        self.q = (q / torch.sqrt((q * q).mean(-1, keepdim=True))).to(BF)
        self.layout = layout

    def cache(self, x):
        x = x.cuda()
        if self.layout == "slots":      # (pages, page, heads, dim) underneath
            x = x.transpose(1, 2).contiguous().transpose(1, 2)
        elif self.layout == "wide":     # a part of a wider pool
            y = torch.full((x.shape[0] * 2, *x.shape[1:3], x.shape[3] + 8), math.nan, dtype=BF, device="cuda")
            y = y[::2, :, :, 8:]
            y.copy_(x)
            x = y
        return x

    def dev(self):
        return (self.cache(self.k), self.cache(self.v), self.table.cuda(),
                torch.tensor(self.starts, dtype=I32, device="cuda"),
                torch.tensor(self.lens, dtype=I32, device="cuda"))


CASES = [
    # (new tokens, lengths), and what differs from 6 x 128 heads on pages of 16
    dict(new=[1], lens=[1]),
    dict(new=[1], lens=[777]),
    dict(new=[1, 1, 1, 1], lens=[5, 16, 17, 300]),
    dict(new=[3, 0, 1, 0], lens=[3, 9, 1, 0]),
    dict(new=[17, 1, 40], lens=[33, 64, 40], window=7),
    dict(new=[1, 1], lens=[500, 31], window=1),
    dict(new=[1, 1], lens=[500, 31], window=384),
    dict(new=[130], lens=[130], H=2, Hk=2),
    dict(new=[70], lens=[333], H=2, Hk=1, window=100),
    dict(new=[9, 33], lens=[200, 47], H=8, Hk=2, D=64, page=64),
    dict(new=[1, 1, 1], lens=[129, 1, 64], H=8, Hk=1, D=128, page=32),
    dict(new=[1, 2], lens=[129, 64], H=20, Hk=1, D=64),
    dict(new=[5, 1], lens=[70, 90], H=3, Hk=3, D=64, page=256, more_cols=2),
    dict(new=[2, 1], lens=[70, 90], H=6, Hk=3, layout="slots"),
    dict(new=[20, 1], lens=[70, 90], H=6, Hk=3, layout="wide", spare_rows=5),
    dict(new=[5, 4], lens=[3, 2], H=2, Hk=2),                 # more new tokens than entries
    dict(new=[2, 2], lens=[1000, -4], H=2, Hk=2, clip=True),   # lengths outside the table
    dict(new=[1], lens=[1100], H=1, Hk=1, page=1024),
    dict(new=[33], lens=[2100], H=1, Hk=1, D=64, page=128),
    dict(new=[150, 1, 200], lens=[150, 400, 260], H=2, Hk=1, window=64),
    dict(new=[300, 1], lens=[40, 40], H=2, Hk=2),              # tiles of rows that see nothing
]


def _setup(case, seed=0):
    kw = {k: v for k, v in case.items() if k not in ("window", "clip")}
    s = Setup(seed=seed, **{**kw, **({"lens": [48, 48]} if case.get("clip") else {})})
    s.lens = case["lens"]
    return s, case.get("window", 0)


@pytest.mark.parametrize("scale", [0.1, -1.5, 0.0])
@pytest.mark.parametrize("i", range(len(CASES)))
def test_attention(i, scale):
    from attention_nn_amd import paged
    s, window = _setup(CASES[i], seed=i)
    kc, vc, table, starts, lens = s.dev()
    ref, rlse, tol, ltol = R.attention(s.q, s.k, s.v, s.table, s.starts, s.lens, scale, window)
    out = torch.full((s.N, s.H, s.D), 7.0, dtype=BF, device="cuda")
    got, lse = paged.attention(s.q.cuda(), kc, vc, table, starts, lens, scale, window, True, out)
    assert got is out
    got, lse = got.cpu().double(), lse.cpu().double()
    end = s.starts[-1]
    assert (got[end:] == 7.0).all()
    assert ((got - ref).abs()[:end] <= tol[:end]).all()
    empty = rlse[:end] == -math.inf
    assert (lse[:end][empty] == -math.inf).all() and (got[:end][empty] == 0).all()
    assert ((lse[:end] - rlse[:end]).abs()[~empty] <= ltol[:end][~empty]).all()
    again = paged.attention(s.q.cuda(), kc, vc, table, starts, lens, scale, window)
    assert torch.equal(again[:end].cpu().double(), got[:end])


@pytest.mark.parametrize("i", range(len(CASES)))
def test_weight(i):
    from attention_nn_amd import paged
    s, window = _setup(CASES[i], seed=i)
    kc, vc, table, starts, lens = s.dev()
    rlse = R.attention(s.q, s.k, s.v, s.table, s.starts, s.lens, 0.1, window)[1]
    lse = rlse.float()
    w = torch.rand((len(s.lens), s.cols * s.page), generator=_gen(i))
    ref, tol = R.weight(s.q, lse, s.k, s.table, s.starts, s.lens, w, 0.1, window)
    got = paged.attention_weight(s.q.cuda(), lse.cuda(), kc, table, starts, lens, w.cuda(), 0.1, window)
    assert ((got.cpu().double() - ref).abs() <= tol).all()
    wg = w.cuda()
    assert paged.attention_weight(s.q.cuda(), lse.cuda(), kc, table, starts, lens, wg, 0.1, window, wg) is wg
    assert torch.equal(wg, got)
    # entries behind a sequence keep their weight
    for j, n in enumerate(s.lens):
        n = min(max(n, 0), w.shape[1])
        assert torch.equal(got[j, n:].cpu(), w[j, n:])


@pytest.mark.parametrize("i", range(len(CASES)))
def test_append(i):
    from attention_nn_amd import paged
    s, _ = _setup(CASES[i], seed=i)
    kc, vc, table, starts, lens = s.dev()
    g = _gen(100 + i)
    fused = torch.randn((s.N, s.H + 2 * s.Hk, s.D), generator=g).to(BF)
    q, k, v = fused[:, :s.H], fused[:, s.H:s.H + s.Hk], fused[:, s.H + s.Hk:]
    cap = s.cols * s.page
    ang = torch.rand((cap, s.D // 4), generator=g) * 6.28
    cs, sn = torch.cos(ang), torch.sin(ang)
    want_k, want_v = s.k.clone(), s.v.clone()
    qref = torch.full(q.shape, 7.0, dtype=torch.float64)
    touched = []
    for n, seq, e in R.tokens(s.starts, s.lens, cap):
        c, d = cs[max(e, 0)].double(), sn[max(e, 0)].double()
        qref[n] = R.norm_rope(q[n].double(), c, d)
        if e >= 0:
            slot = int(s.table[seq, e // s.page]), e % s.page
            want_k[slot[0], :, slot[1]] = 0
            want_v[slot[0], :, slot[1]] = v[n]
            touched.append((slot, R.norm_rope(k[n].double(), c, d)))
    out = torch.full(q.shape, 7.0, dtype=BF, device="cuda")
    f = fused.cuda()
    views = f[:, :s.H], f[:, s.H:s.H + s.Hk], f[:, s.H + s.Hk:]
    got = paged.append(*views, cs.cuda(), sn.cuda(), kc, vc, table, starts, lens, out=out)
    tol = (2.0 ** -8 + (s.D / 2 + 8) * 2.0 ** -23)

    def near(a, b):
        return ((a.double() - b).abs() <= tol * b.abs() + 2.0 ** -16 * b.abs().amax(-1, keepdim=True)).all()

    assert near(got.cpu(), qref)
    kh, vh = kc.cpu().clone(), vc.cpu()
    for (p, o), ref in touched:
        assert near(kh[p, :, o], ref)
        kh[p, :, o] = 0
    assert torch.equal(torch.nan_to_num(kh, 5.0), torch.nan_to_num(want_k, 5.0))
    assert torch.equal(vh, want_v)


def test_append_positions_and_bad_pages():
    """Positions of their own turn a token as its entry would; pages that are
    none, on the way into the cache, leave it as it was."""
    from attention_nn_amd import paged
    s = Setup([2, 3], [20, 30], H=2, Hk=2, D=64, garbage=False)
    kc, vc, table, starts, lens = s.dev()
    x = torch.randn((5, 2, 64), generator=_gen(1)).to(BF).cuda()
    ang = torch.rand((99, 16), generator=_gen(2)) * 6.28
    cs, sn = torch.cos(ang).cuda(), torch.sin(ang).cuda()
    a = paged.append(x, x, x, cs, sn, kc, vc, table, starts, lens)
    k1 = kc.clone()
    entry = torch.tensor([18, 19, 27, 28, 29], dtype=I32, device="cuda")
    assert torch.equal(a, paged.append(x, x, x, cs, sn, kc, vc, table, starts, lens, pos=entry))
    assert torch.equal(k1, kc)
    b = paged.append(x, x, x, cs, sn, kc, vc, table, starts, lens, pos=entry + 40)
    assert not torch.equal(a, b) and not torch.equal(k1, kc)
    far = paged.append(x, x, x, cs, sn, kc, vc, table, starts, lens, pos=entry + 4000)
    near = paged.append(x, x, x, cs, sn, kc, vc, table, starts, lens, pos=torch.full_like(entry, 98))
    assert torch.equal(far, near)
    for bad in (-1, kc.shape[0], 1 << 30):
        t = torch.full_like(table, bad)
        k2, v2 = kc.clone(), vc.clone()
        assert torch.equal(a, paged.append(x, x, x, cs, sn, kc, vc, t, starts, lens))
        assert torch.equal(k2, kc) and torch.equal(v2, vc)


def test_bad_pages_and_starts_are_read_as_documented():
    """An id that is no page reads page 0; starts outside the rows end at them."""
    from attention_nn_amd import paged
    s = Setup([2, 1], [60, 40], H=2, Hk=2, garbage=False)
    kc, vc, table, starts, lens = s.dev()
    q = s.q.cuda()
    bad, zero = table.clone(), table.clone()
    bad[0, 1], bad[1, 0], zero[0, 1], zero[1, 0] = -7, 1 << 30, 0, 0
    for window in (0, 20):
        a = paged.attention(q, kc, vc, bad, starts, lens, 0.1, window)
        assert torch.equal(a, paged.attention(q, kc, vc, zero, starts, lens, 0.1, window))
    w = torch.zeros((2, s.cols * 16), device="cuda")
    lse = paged.attention(q, kc, vc, zero, starts, lens, 0.1, want_lse=True)[1]
    assert torch.equal(paged.attention_weight(q, lse, kc, bad, starts, lens, w, 0.1),
                       paged.attention_weight(q, lse, kc, zero, starts, lens, w, 0.1))
    past = torch.tensor([0, 2, 1 << 30], dtype=I32, device="cuda")
    assert torch.equal(paged.attention(q, kc, vc, table, past, lens, 0.1),
                       paged.attention(q, kc, vc, table, starts, lens, 0.1))


def test_values_that_a_token_does_not_see():
    """NaN and infinities in later tokens' values and keys, and before the window,
    reach no token that does not see them."""
    from attention_nn_amd import paged
    for H, Hk, D, window, length, n in ((2, 2, 128, 0, 100, 40), (4, 2, 64, 24, 90, 50), (2, 1, 128, 5, 33, 33)):
        s = Setup([n], [length], H=H, Hk=Hk, D=D, garbage=False)
        clean = s.dev()
        q = s.q.cuda()
        want = paged.attention(q, *clean, 0.1, window, True)
        for e in (length - n + 3, length - 1, length - n - 1 - (window or 3)):
            if e < 0:
                continue
            p, o = int(s.table[0, e // 16]), e % 16
            for which, value in (("v", math.nan), ("v", math.inf), ("k", math.nan)):
                kc, vc = clean[0].clone(), clean[1].clone()
                (vc if which == "v" else kc)[p, :, o] = value
                got, lse = paged.attention(q, kc, vc, *clean[2:], 0.1, window, True)
                for t in range(n):
                    at = length - n + t
                    if not (e <= at and (not window or at - e < window)):
                        # the rows around it may take another path to the same sums
                        assert torch.isfinite(got[t]).all(), (e, at, which, value)
                        assert ((got[t] - want[0][t]).abs().float() <= 2.0 ** -6 * (1 + want[0][t].abs().float())).all()
                        assert ((lse[t] - want[1][t]).abs() <= 1e-5 * (1 + want[1][t].abs())).all()
                    else:
                        assert not torch.isfinite(got[t]).any()


def test_scores_of_any_size():
    """Large scores, all equal scores and scores that fall from entry to entry."""
    from attention_nn_amd import paged
    for mode in ("large", "equal", "falling", "rising"):
        s = Setup([40, 1], [300, 200], H=2, Hk=2, garbage=False, seed=3)
        if mode == "large":
            s.q = (s.q.float() * 30).to(BF)
        elif mode == "equal":
            s.k[:] = s.k[:1, :1, :1]
        else:
            u = s.q[0, 0].clone()
            s.q[:] = u
            for i in range(2):
                for e in range(s.lens[i]):
                    a = (300 - e if mode == "falling" else e) / 30
                    s.k[int(s.table[i, e // 16]), :, e % 16] = (u.float() * a).to(BF)
        kc, vc, table, starts, lens = s.dev()
        ref, rlse, tol, ltol = R.attention(s.q, s.k, s.v, s.table, s.starts, s.lens, 0.1, 0)
        got, lse = paged.attention(s.q.cuda(), kc, vc, table, starts, lens, 0.1, want_lse=True)
        assert ((got.cpu().double() - ref).abs() <= tol).all(), mode
        assert ((lse.cpu().double() - rlse).abs() <= ltol).all(), mode


EVICT = [dict(lens=[5], keep=3), dict(lens=[5], keep=5, recent=2), dict(lens=[5, 0, 16, 17], keep=16, recent=4),
         dict(lens=[700, 1500, 3], keep=600, recent=100), dict(lens=[300], keep=300, recent=300),
         dict(lens=[300], keep=200, recent=200), dict(lens=[40, 60], keep=1, recent=0),
         dict(lens=[2500, 1100], keep=1024, recent=1), dict(lens=[90, 64], keep=64, recent=9, page=64, D=64, Hk=3),
         dict(lens=[200, 130], keep=77, recent=30, page=32, layout="slots"),
         dict(lens=[200, 130], keep=77, recent=30, layout="wide", D=64),
         # longer than a work-group holds at once
         dict(lens=[9000, 12], keep=4000, recent=300, D=64, Hk=1, page=1024),
         dict(lens=[17000, 30000], keep=5000, recent=100, D=64, Hk=1, page=1024)]


@pytest.mark.parametrize("kind", ["spread", "ties", "few", "odd"])
@pytest.mark.parametrize("i", range(len(EVICT)))
def test_evict(i, kind):
    """Exact: the entries kept, their rows and weights, into other pages and in place."""
    from attention_nn_amd import paged
    case = {"recent": 0, "page": 16, "D": 128, "Hk": 2, **EVICT[i]}
    keep, recent = case.pop("keep"), case.pop("recent")
    page = case["page"]
    s = Setup(new=[0] * len(case["lens"]), H=case["Hk"], garbage=False, seed=i, out_cols=-(-keep // page), more_cols=1 + keep // page, **case)
    g = _gen(i)
    w = torch.randn((len(s.lens), s.cols * page), generator=g)
    if kind == "ties":
        w = torch.floor(w * 2) / 2
        w[w == 0] = -0.0
        w[:, ::3] = w[:, ::3].abs()
    elif kind == "few":
        w = (w > 1).float()
    elif kind == "odd":
        w[:, 1::4] = math.nan
        w[:, 2::4] = -math.inf
        w[:, 3::8] = math.inf
        w[:, 4::8] = w[:, 4::8] * 1e-40
    kc, vc, table, _, lens = s.dev()
    for out_table in (s.out_table, s.table):
        ref = R.evict(s.k, s.v, s.table, s.lens, w, keep, recent, out_table)
        k, v = kc.clone(), vc.clone()
        got = paged.evict(k, v, table, lens, w.cuda(), keep, recent,
                          None if out_table is s.table else out_table.cuda())
        assert torch.equal(got[0].cpu(), ref[0]) and torch.equal(got[1].cpu(), ref[1])
        assert torch.equal(torch.nan_to_num(got[2].cpu(), 9.0), torch.nan_to_num(ref[2], 9.0))
        assert torch.equal(k.cpu(), ref[3]) and torch.equal(v.cpu(), ref[4])


def test_long_offsets():
    """A pool whose entries lie past 2^31 elements from its start."""
    from attention_nn_amd import paged
    pages = (1 << 31) // (16 * 128) + 40
    if torch.cuda.mem_get_info()[0] < 3 * pages * 16 * 128 * 2:
        pytest.skip("not enough memory")
    kc = torch.empty((pages, 1, 16, 128), dtype=BF, device="cuda")
    vc = torch.empty_like(kc)
    s = Setup([3], [70], H=1, Hk=1, garbage=False, out_cols=3)
    high = torch.tensor([[pages - 1, pages - 9, 5, pages - 3, pages - 20]], dtype=I32, device="cuda")
    kc[high[0].long()] = s.k[s.table[0].long()].cuda()
    vc[high[0].long()] = s.v[s.table[0].long()].cuda()
    k0, v0, table, starts, lens = s.dev()
    q = s.q.cuda()
    a = paged.attention(q, k0, v0, table, starts, lens, 0.1, want_lse=True)
    b = paged.attention(q, kc, vc, high, starts, lens, 0.1, want_lse=True)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    w = torch.rand((1, 80), device="cuda")
    assert torch.equal(paged.attention_weight(q, a[1], k0, table, starts, lens, w, 0.1),
                       paged.attention_weight(q, a[1], kc, high, starts, lens, w, 0.1))
    ang = torch.rand((80, 32), device="cuda")
    args = (q, q, q, torch.cos(ang), torch.sin(ang))
    assert torch.equal(paged.append(*args, k0, v0, table, starts, lens), paged.append(*args, kc, vc, high, starts, lens))
    paged.evict(k0, v0, table, lens, w, 40, 5)
    paged.evict(kc, vc, high, lens, w, 40, 5)
    assert torch.equal(kc[high[0, :3].long()], k0[table[0, :3].long()])
    assert torch.equal(vc[high[0, :3].long()], v0[table[0, :3].long()])


def test_many_sequences():
    """More sequences than a wave looks at at once, empty ones among them."""
    from attention_nn_amd import paged
    S = 4200
    new = [(i * 7 % 3 == 0) * 1 + (i % 97 == 0) * 2 for i in range(S)]
    lens = [max(n, i % 23) for i, n in enumerate(new)]
    s = Setup(new, lens, H=1, Hk=1, D=64, page=32, garbage=False)
    kc, vc, table, starts, ln = s.dev()
    got = paged.attention(s.q.cuda(), kc, vc, table, starts, ln, 0.1).cpu().double()
    ref, _, tol, _ = R.attention(s.q, s.k, s.v, s.table, s.starts, s.lens, 0.1, 0)
    assert ((got - ref).abs() <= tol).all()


def _step(x, state, window=0, keep=0):
    """One layer's step as a serving loop makes it."""
    from attention_nn_amd import paged
    q, k, v = x
    kc, vc, table, starts, lens, cs, sn, w = state
    q = paged.append(q, k, v, cs, sn, kc, vc, table, starts, lens)
    y, lse = paged.attention(q, kc, vc, table, starts, lens, 0.1, window, True)
    w = paged.attention_weight(q, lse, kc, table, starts, lens, w, 0.1, window)
    if keep:
        return (y, *paged.evict(kc, vc, table, lens, w, keep, min(8, keep)))
    return y, w


def _serving(seed, new, lens, H=6, Hk=6, D=128, page=16):
    s = Setup(new, lens, H=H, Hk=Hk, D=D, page=page, seed=seed, garbage=False, more_cols=2)
    kc, vc, table, starts, ln = s.dev()
    ang = torch.rand((s.cols * page, D // 4), generator=_gen(seed)) * 6.28
    x = [torch.randn((s.N, n, D), generator=_gen(seed + i)).to(BF).cuda() for i, n in enumerate((H, Hk, Hk))]
    w = torch.zeros((len(lens), s.cols * page), device="cuda")
    return x, [kc, vc, table, starts, ln, torch.cos(ang).cuda(), torch.sin(ang).cuda(), w]


def test_replayed_from_graphs():
    """Two captured steps, replayed in turn with eager work between and with new
    tokens, lengths and tables, against the eager step."""
    graphs = []
    for n, (new, lens) in enumerate((([1, 1, 1], [40, 200, 90]), ([30, 1, 60], [70, 200, 90]))):
        x, st = _serving(n, new, lens)
        _step(x, st, 0, 32)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = _step(x, st, 0, 32)
        graphs.append((g, x, st, y, new))
    for i in range(4):
        for g, x, st, y, new in graphs:
            for j, t in enumerate(x):
                t.copy_(torch.randn(t.shape, generator=_gen(50 + i + j)).to(BF))
            st[4].copy_(torch.tensor([60 + 5 * i, 150 - i, 77 + i], dtype=I32))
            st[2].copy_(st[2].flip(0).clone())
            k0, v0 = st[0].clone(), st[1].clone()
            g.replay()
            want = _step(x, [k0, v0, *st[2:]], 0, 32)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(y, want))
            assert torch.equal(k0, st[0]) and torch.equal(v0, st[1])


def test_another_stream():
    x, st = _serving(7, [5, 1], [90, 300])
    x2, st2 = _serving(7, [5, 1], [90, 300])
    want = _step(x, st, 16, 40)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = _step(x2, st2, 16, 40)
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_chunks_join():
    """A prompt brought in chunks of any size ends as the prompt brought whole,
    within the bounds of one call; and it is the engine's attention."""
    from attention_nn_amd import paged
    H, D, T = 6, 128, 150
    x = [torch.randn((T, H, D), generator=_gen(i)).to(BF).cuda() for i in range(3)]
    ang = torch.rand((T, D // 4), generator=_gen(9)) * 6.28
    cs, sn = torch.cos(ang).cuda(), torch.sin(ang).cuda()
    table = torch.randperm(12, generator=_gen(4)).to(I32)[None, :10].contiguous().cuda()
    outs = []
    for chunks in ([150], [100, 50], [1] * 20 + [130], [37, 1, 64, 48]):
        kc = torch.zeros((12, H, 16, D), dtype=BF, device="cuda")
        vc = torch.zeros_like(kc)
        at, ys = 0, []
        for n in chunks:
            starts = torch.tensor([0, n], dtype=I32, device="cuda")
            lens = torch.tensor([at + n], dtype=I32, device="cuda")
            q = paged.append(*(t[at:at + n] for t in x), cs, sn, kc, vc, table, starts, lens)
            ys.append(paged.attention(q, kc, vc, table, starts, lens, 0.1, 48))
            at += n
        outs.append((torch.cat(ys).double().cpu(), kc, vc))
    q = R.norm_rope(x[0].double().cpu(), cs.cpu()[:, None].double(), sn.cpu()[:, None].double()).to(BF)
    ref, _, tol, _ = R.attention(q, outs[0][1].cpu(), outs[0][2].cpu(), table.cpu(), [0, T], [T], 0.1, 48)
    for y, kc, vc in outs:
        assert torch.equal(kc, outs[0][1]) and torch.equal(vc, outs[0][2])
        # the queries' own rounding lies half a step on either side of a tie
        assert ((y - ref).abs() <= 2 * tol + 2.0 ** -8).all()


def test_nothing_there():
    """No sequences, no rows, a table without pages, sequences without entries."""
    from attention_nn_amd import paged
    kc = torch.full((3, 2, 16, 64), 7.0, dtype=BF, device="cuda")
    vc = kc.clone()
    ang = torch.zeros((8, 16), device="cuda")

    def i32(*v, shape=None):
        t = torch.tensor(v, dtype=I32, device="cuda")
        return t if shape is None else t.view(shape)

    q = torch.ones((4, 2, 64), dtype=BF, device="cuda")
    for table, starts, lens in ((i32(shape=(0, 2)), i32(0), i32()), (i32(shape=(2, 0)), i32(0, 1, 4), i32(1, 3)),
                                (i32(0, 1, 2, 0, shape=(2, 2)), i32(0, 0, 0), i32(9, 0)),
                                (i32(0, 1, 2, 0, shape=(2, 2)), i32(0, 1, 4), i32(0, 0))):
        S, cap = table.shape[0], table.shape[1] * 16
        end = int(starts[-1])
        out = torch.full_like(q, 5.0)
        paged.append(q, q, q, ang, ang, kc, vc, table, starts, lens, out=out)
        assert (out[end:] == 5.0).all() and (kc == 7.0).all() and (vc == 7.0).all()
        out = torch.full_like(q, 5.0)
        lse = paged.attention(q, kc, vc, table, starts, lens, 0.1, 0, True, out)[1]
        assert (out[end:] == 5.0).all() and (out[:end] == 0).all() and (lse[:end] == -math.inf).all()
        w = torch.rand((S, cap), device="cuda")
        assert torch.equal(paged.attention_weight(q, lse, kc, table, starts, lens, w, 0.1), w)
        n = i32(*([0] * S))
        k, new, w2 = paged.evict(kc, vc, table, n, w, 5, 2, i32(*([1] * S), shape=(S, 1)))
        assert (k == -1).all() and (new == 0).all() and (w2 == 0).all() and (kc == 7.0).all()
    table, starts, lens = i32(0, 1, shape=(1, 2)), i32(0, 0), i32(20)
    none = q[:0]
    assert paged.append(none, none, none, ang, ang, kc, vc, table, starts, lens).shape == none.shape
    out, lse = paged.attention(none, kc, vc, table, starts, lens, 0.1, want_lse=True)
    assert out.shape == none.shape and lse.shape == (0, 2)
    w = torch.rand((1, 32), device="cuda")
    assert torch.equal(paged.attention_weight(none, lse, kc, table, starts, lens, w, 0.1), w)


@pytest.mark.parametrize("new,lens", [([1, 1], [900, 40]), ([1], [9000]), ([150, 1], [170, 60]),
                                      ([513], [5000])])
def test_out_is_the_queries(new, lens):
    """The result in the queries' own memory, in one part and in several."""
    from attention_nn_amd import paged
    s = Setup(new, lens, H=4, Hk=2, D=64, garbage=False)
    kc, vc, table, starts, ends = s.dev()
    q = s.q.cuda()
    want, wlse = paged.attention(q, kc, vc, table, starts, ends, 0.1, want_lse=True)
    x = q.clone()
    got, lse = paged.attention(x, kc, vc, table, starts, ends, 0.1, want_lse=True, out=x)
    assert got is x and torch.equal(got, want) and torch.equal(lse, wlse)
    ang = torch.rand((s.cols * 16, 16), generator=_gen(3)).cuda()
    k = torch.randn((s.N, 2, 64), generator=_gen(4)).to(BF).cuda()
    want = paged.append(q, k, k, ang.cos(), ang.sin(), kc, vc, table, starts, ends)
    x = q.clone()
    assert torch.equal(paged.append(x, k, k, ang.cos(), ang.sin(), kc, vc, table, starts, ends, out=x), want)


@pytest.mark.parametrize("far", [(1 << 25) + 8, 0])
def test_far_queries(far):
    """Queries whose rows (or heads) lie further apart than a tile's offsets reach."""
    from attention_nn_amd import paged
    s = Setup([1, 2], [60, 20], H=4, Hk=2, D=64, garbage=False)
    kc, vc, table, starts, lens = s.dev()
    q, w = s.q.cuda(), torch.zeros((2, s.cols * 16), device="cuda")
    buf = torch.empty(3 * (1 << 25) + 1024 if far else 3 * (1 << 26) + 1024, dtype=BF, device="cuda")
    x = buf.as_strided((3, 4, 64), (far, 64, 1) if far else (64, (1 << 26) + 8, 1))
    x.copy_(q)
    want, lse = paged.attention(q, kc, vc, table, starts, lens, 0.1, want_lse=True)
    assert torch.equal(paged.attention(x, kc, vc, table, starts, lens, 0.1), want)
    assert torch.equal(paged.attention_weight(x, lse, kc, table, starts, lens, w, 0.1),
                       paged.attention_weight(q, lse, kc, table, starts, lens, w, 0.1))


def test_windows_past_the_table():
    """A window of more entries than there are is none, in 32 bits and past them."""
    from attention_nn_amd import paged
    s = Setup([1, 30], [200, 90], H=2, Hk=1, D=64, garbage=False)
    kc, vc, table, starts, lens = s.dev()
    q, w = s.q.cuda(), torch.zeros((2, s.cols * 16), device="cuda")
    want, lse = paged.attention(q, kc, vc, table, starts, lens, 0.1, want_lse=True)
    seen = paged.attention_weight(q, lse, kc, table, starts, lens, w, 0.1)
    for window in (200, 1 << 30, (1 << 31) - 1, 1 << 31, (1 << 32) + 5):
        assert torch.equal(paged.attention(q, kc, vc, table, starts, lens, 0.1, window), want)
        assert torch.equal(paged.attention_weight(q, lse, kc, table, starts, lens, w, 0.1, window), seen)


def test_shared_pages():
    """A prefix that two sequences share, read by both; evicted to pages of their own."""
    from attention_nn_amd import paged
    s = Setup([1, 20], [100, 130], H=4, Hk=2, D=64, garbage=False, more_cols=1, out_cols=4)
    s.table[1, :5] = s.table[0, :5]
    kc, vc, table, starts, lens = s.dev()
    q = s.q.cuda()
    ref, _, tol, _ = R.attention(s.q, s.k, s.v, s.table, s.starts, s.lens, 0.1, 0)
    got, lse = paged.attention(q, kc, vc, table, starts, lens, 0.1, want_lse=True)
    assert ((got.double().cpu() - ref).abs() <= tol).all()
    w = paged.attention_weight(q, lse, kc, table, starts, lens, torch.zeros((2, s.cols * 16), device="cuda"), 0.1)
    ref = R.evict(s.k, s.v, s.table, s.lens, w.cpu(), 60, 20, s.out_table)
    got = paged.evict(kc, vc, table, lens, w, 60, 20, s.out_table.cuda())
    assert torch.equal(got[0].cpu(), ref[0])
    assert torch.equal(kc.cpu(), ref[3]) and torch.equal(vc.cpu(), ref[4])


def test_evict_within_a_larger_table():
    """Pages to go to that begin where the table does and go on elsewhere: the first
    sequence in place, the others not."""
    from attention_nn_amd import paged
    lens, keep = [1500, 1400, 1300], 1200
    s = Setup([0] * 3, lens, H=1, Hk=1, D=128, garbage=False, out_cols=80)
    n = s.cols
    both = torch.empty(4 * 2 * n, dtype=I32)   # rows 2 n apart, and n apart
    both[:2 * n].view(2, n)[0] = s.table[0]
    both[n:3 * n] = s.out_table.flatten()[:2 * n]
    both[2 * n:3 * n] = s.table[1]
    both[4 * n:5 * n] = s.table[2]
    dev = both.cuda()
    table = dev.as_strided((3, n), (2 * n, 1))
    for seqs, out in ((1, dev.as_strided((1, n), (n, 1))), (2, dev.as_strided((2, n), (n, 1)))):
        kc, vc = s.cache(s.k), s.cache(s.v)
        w = torch.rand((3, n * 16), generator=_gen(5))
        ref = R.evict(s.k, s.v, table[:seqs].cpu(), lens[:seqs], w[:seqs], keep, 100, out.cpu())
        paged.evict(kc, vc, table[:seqs], torch.tensor(lens[:seqs], dtype=I32, device="cuda"), w[:seqs].cuda(),
                    keep, 100, out)
        assert torch.equal(kc.cpu(), ref[3]) and torch.equal(vc.cpu(), ref[4])


def test_refusals():
    """Wrong types, shapes and sizes are refused before any launch."""
    from attention_nn_amd import paged
    s = Setup([2, 1], [20, 30], H=4, Hk=2, D=64, garbage=False)
    kc, vc, table, starts, lens = s.dev()
    q = s.q.cuda()
    w = torch.zeros((2, s.cols * 16), device="cuda")
    lse = torch.zeros((3, 4), device="cuda")

    def bad(error, fn, *args, **kw):
        with pytest.raises(error):
            fn(*args, **kw)

    at = paged.attention
    bad(TypeError, at, q.float(), kc, vc, table, starts, lens, 0.1)
    bad(TypeError, at, q, kc.half(), vc, table, starts, lens, 0.1)
    bad(TypeError, at, q, kc, vc, table.long(), starts, lens, 0.1)
    bad(TypeError, at, q, kc, vc, table, starts, lens.long(), 0.1)
    bad(ValueError, at, q, kc, vc[:-1], table, starts, lens, 0.1)
    bad(ValueError, at, q, kc, vc, table, starts[:-1], lens, 0.1)
    bad(ValueError, at, q, kc, vc, table, starts, lens[:1], 0.1)
    bad(ValueError, at, q[:, :3], kc, vc, table, starts, lens, 0.1)
    bad(ValueError, at, q.view(3, 2, 128), kc, vc, table, starts, lens, 0.1)
    bad(ValueError, at, q, kc, vc, table, starts, lens, 0.1, -1)
    bad(ValueError, at, q, kc, vc, table, starts, lens, math.nan)
    bad(ValueError, at, q, kc[:, :, :15], vc[:, :, :15], table, starts, lens, 0.1)
    bad(ValueError, at, q, kc, vc, table, starts, lens, 0.1, out=torch.empty_like(q)[:2])
    bad(ValueError, at, q, kc, vc, table.cpu(), starts, lens, 0.1)
    bad(ValueError, at, q, kc, vc, table, starts, lens, 3e38)
    bad(ValueError, at, q, kc, vc, table, starts, lens, 0.1, -(1 << 32) + 5)
    two = torch.zeros((4, 4, 64), dtype=BF, device="cuda")
    bad(ValueError, at, two[1:], kc, vc, table, starts, lens, 0.1, out=two[:-1])
    we = paged.attention_weight
    bad(ValueError, we, q, lse[:2], kc, table, starts, lens, w, 0.1)
    bad(ValueError, we, q, lse, kc, table, starts, lens, w[:, :-1], 0.1)
    bad(TypeError, we, q, lse, kc, table, starts, lens, w.double(), 0.1)
    bad(ValueError, we, q, lse, kc, table, starts, lens, w, 0.1, out=w[:1].expand(2, -1))
    ev = paged.evict
    bad(ValueError, ev, kc, vc, table, lens, w, 0)
    bad(ValueError, ev, kc, vc, table, lens, w, 8, 9)
    bad(ValueError, ev, kc, vc, table, lens, w, 8, 1 << 32)
    bad(ValueError, ev, kc, vc, table, lens, w, 1000)
    bad(ValueError, ev, kc, vc, table, lens, w[:1], 8)
    ang = torch.zeros((40, 16), device="cuda")
    ap = paged.append
    bad(ValueError, ap, q, q, q, ang, ang, kc, vc, table, starts, lens)
    bad(ValueError, ap, q, q[:, :2], q[:2, :2], ang, ang, kc, vc, table, starts, lens)
    bad(ValueError, ap, q, q[:, :2], q[:, :2], ang[:, :8], ang, kc, vc, table, starts, lens)
    bad(TypeError, ap, q, q[:, :2], q[:, :2], ang.double(), ang, kc, vc, table, starts, lens)
    ang, fused = torch.zeros((40, 16), device="cuda"), torch.zeros((3, 6, 64), dtype=BF, device="cuda")
    flat = fused.view(-1)[:3 * 4 * 64].view(3, 4, 64)   # the first rows of queries, keys and values
    bad(ValueError, ap, q, fused[:, 2:4], q[:, :2], ang, ang, kc, vc, table, starts, lens, out=flat)
    bad(ValueError, ap, fused[:, :4], q[:, :2], q[:, :2], ang, ang, kc, vc, table, starts, lens, out=flat)
