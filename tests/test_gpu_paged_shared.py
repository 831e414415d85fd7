"""Attention of sequences that begin with the same entries (paged.attention_shared)
against plain 64-bit attention over each sequence's whole table."""

import math

import pytest
import torch

import oracle.ref_paged as R

pytestmark = pytest.mark.gpu
BF, I32 = torch.bfloat16, torch.int32


class Setup:
    """groups: (prefix entries, [(new tokens, own entries with these), ...]) of each; a
    prefix of None: the sequences belong to no group (first and last groups only).  What
    no sequence uses is NaN in the keys and infinite in the values."""

    def __init__(self, groups, H=6, Hk=6, D=128, page=16, seed=0, layout="pages", spare_rows=0, more_cols=0):
        g = torch.Generator().manual_seed(seed)
        self.H, self.Hk, self.D, self.page = H, Hk, D, page
        seqs = [(p, i, n, m) for i, (p, members) in enumerate(groups) for n, m in members]
        self.new = [n for _, _, n, _ in seqs]
        self.lens = [(p or 0) + m for p, _, _, m in seqs]
        S = len(seqs)
        self.cols = max(1, -(-max(self.lens + [1]) // page)) + more_cols
        real = [(i, p) for i, (p, _) in enumerate(groups) if p is not None]
        self.pcols = max([1] + [-(-p // page) for _, p in real])
        pages = S * self.cols + len(groups) * (self.pcols + 1) + 3
        order = iter(torch.randperm(pages, generator=g).tolist())
        common = {i: [next(order) for _ in range(-(-p // page))] for i, p in real}
        self.ptable = torch.full((len(real), self.pcols), -1, dtype=I32)
        for r, (i, _) in enumerate(real):
            self.ptable[r, :len(common[i])] = torch.tensor(common[i], dtype=I32)
        self.plens = [p for _, p in real]
        at, self.groups = 0, []
        for i, (p, members) in enumerate(groups):
            if p is not None:
                self.groups.append(at)
            at += len(members)
            if p is not None:
                end = at
        self.groups.append(end if real else 0)
        self.table = torch.full((S, self.cols), -1, dtype=I32)
        shape = (pages, Hk, page, D)
        k, v = torch.randn(shape, generator=g), torch.randn(shape, generator=g)
        k = k / torch.sqrt((k * k).mean(-1, keepdim=True))
        used = torch.zeros(pages, page, dtype=torch.bool)
        for i, p in real:
            for e in range(p):
                used[common[i][e // page], e % page] = True
        for s, (p, i, n, m) in enumerate(seqs):
            full = (p or 0) // page
            for c in range(self.cols):
                self.table[s, c] = common[i][c] if c < full else next(order)
            if (p or 0) % page:     # the page that the prefix ends in is the sequence's own: a copy
                a, b = common[i][full], int(self.table[s, full])
                k[b, :, :p % page], v[b, :, :p % page] = k[a, :, :p % page], v[a, :, :p % page]
            for e in range(self.lens[s]):
                used[self.table[s, e // page], e % page] = True
        k[~used[:, None, :].expand(pages, Hk, page)] = math.nan
        v[~used[:, None, :].expand(pages, Hk, page)] = math.inf
        self.k, self.v = k.to(BF), v.to(BF)
        self.starts = [0]
        for n in self.new:
            self.starts.append(self.starts[-1] + n)
        self.N = self.starts[-1] + spare_rows
        q = torch.randn((self.N, H, D), generator=g)
        self.q = (q / torch.sqrt((q * q).mean(-1, keepdim=True))).to(BF)
        self.layout = layout

    def widened(self):
        """Tables of prefixes so wide that the call shares them, however short they are."""
        again = max(1, len(self.lens) - len(self.plens)) * self.Hk * self.D * 4
        cols = max(self.pcols, -(-48_100_000 // (again * self.page)))
        wide = torch.full((len(self.plens), cols), -1, dtype=I32)
        wide[:, :self.pcols] = self.ptable
        self.ptable = wide
        return self

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
        def i(x):
            return torch.tensor(x, dtype=I32, device="cuda")
        return (self.cache(self.k), self.cache(self.v), self.table.cuda(), i(self.starts), i(self.lens),
                i(self.groups), self.ptable.cuda(), i(self.plens))


def _one(n, *lens):
    return [(n, m) for m in lens]


CASES = [
    dict(groups=[(40, _one(1, 1, 2, 17))]),
    dict(groups=[(1, _one(1, 1))]),
    dict(groups=[(777, _one(1, 5, 60))]),
    dict(groups=[(64, _one(1, *range(1, 71)))], H=2, Hk=2),                    # more rows than a tile
    dict(groups=[(130, _one(1, *[3] * 140))], H=1, Hk=1, D=64),
    dict(groups=[(48, _one(3, 3, 9, 20)), (33, _one(2, 2, 40)), (0, _one(1, 5, 1))]),
    dict(groups=[(None, _one(1, 30, 4)), (100, _one(1, 7, 8)), (None, _one(2, 9))]),
    dict(groups=[(500, _one(1, 9, 12, 300))], window=7),
    dict(groups=[(500, [(1, 9), (5, 12), (1, 300)])], window=100),
    dict(groups=[(200, _one(1, 1, 20))], window=1),
    dict(groups=[(96, [(1, 5), (16, 16), (17, 20), (40, 90), (1, 1)])], H=2, Hk=2),   # many tokens beside few
    dict(groups=[(300, [(130, 130), (2, 5), (200, 260)])], H=2, Hk=1, window=64),
    dict(groups=[(150, _one(4, 4, 9, 50)), (70, _one(1, 1, 2, 3))], H=8, Hk=2, page=32),
    dict(groups=[(90, _one(16, 16, 30)), (90, [(17, 17), (3, 8)])], H=8, Hk=1, D=64, page=64),
    dict(groups=[(129, _one(1, 1, 64, 2))], H=20, Hk=1, D=64),
    dict(groups=[(257, _one(2, 70, 90))], H=6, Hk=3, layout="slots"),
    dict(groups=[(64, [(20, 70), (1, 90)])], H=6, Hk=3, layout="wide", spare_rows=5, more_cols=2),
    dict(groups=[(1100, _one(1, 1, 900))], H=1, Hk=1, page=1024),
    dict(groups=[(2100, _one(8, 33, 8))], H=1, Hk=1, D=64, page=128),
    dict(groups=[(None, [(3, 9), (0, 4)])], H=2, Hk=2),                        # no groups at all
    dict(groups=[(60, [(0, 5), (1, 1), (0, 0)]), (31, [(0, 3)])]),             # sequences without tokens
]


def _check(s, got, lse, scale, window, out=None):
    ref, rlse, tol, ltol = R.attention(s.q, s.k, s.v, s.table, s.starts, s.lens, scale, window)
    got, lse = got.cpu().double(), lse.cpu().double()
    end = s.starts[-1]
    if out is not None:
        assert (got[end:] == out).all()
    assert ((got - ref).abs()[:end] <= tol[:end]).all()
    empty = rlse[:end] == -math.inf
    assert (lse[:end][empty] == -math.inf).all() and (got[:end][empty] == 0).all()
    assert ((lse[:end] - rlse[:end]).abs()[~empty] <= ltol[:end][~empty]).all()


@pytest.mark.parametrize("wide,scale", [(True, 0.1), (True, -1.5), (True, 0.0), (False, 0.1)])
@pytest.mark.parametrize("i", range(len(CASES)))
def test_attention_shared(i, wide, scale):
    from attention_nn_amd import paged
    case = dict(CASES[i])
    window = case.pop("window", 0)
    s = Setup(seed=i, **case)
    if wide:
        s.widened()
    kc, vc, table, starts, lens, groups, pt, pl = s.dev()
    out = torch.full((s.N, s.H, s.D), 7.0, dtype=BF, device="cuda")
    got, lse = paged.attention_shared(s.q.cuda(), kc, vc, table, starts, lens, groups, pt, pl, scale, window, True, out)
    assert got is out
    _check(s, got, lse, scale, window, 7.0)
    q = s.q.cuda()      # in place of the queries, and the same bits again
    again = paged.attention_shared(q, kc, vc, table, starts, lens, groups, pt, pl, scale, window, out=q)
    assert again is q and torch.equal(again[:s.starts[-1]], got[:s.starts[-1]])


@pytest.mark.parametrize("window", [0, 384])
@pytest.mark.parametrize("shape", [
    # prefix, sequences, groups, new, own, heads
    (5000, 40, 1, 1, 300, (6, 6, 128)), (3001, 12, 4, 4, 333, (8, 2, 128)), (9000, 3, 2, 1, 1500, (12, 3, 64)),
    (2048, 8, 1, 40, 700, (8, 8, 64)), (700, 200, 1, 1, 20, (4, 4, 128)), (20000, 2, 1, 1, 5000, (2, 1, 128)),
])
def test_long_prefixes(shape, window):
    from attention_nn_amd import paged
    P, S, G, new, own, (H, Hk, D) = shape
    g = torch.Generator().manual_seed(P)
    groups = [(P, [(min(new, m), m) for m in torch.randint(1, own + 1, (S,), generator=g).tolist()]) for _ in range(G)]
    groups = [(p, [(1 if j % 3 == 0 else n, m) for j, (n, m) in enumerate(ms)]) for p, ms in groups]
    s = Setup(groups, H=H, Hk=Hk, D=D, page=64, seed=1)
    kc, vc, table, starts, lens, gr, pt, pl = s.dev()
    ref, rlse, tol, ltol = R.attention_whole(s.q, s.k, s.v, s.table, s.starts, s.lens, 0.1, window)
    # the prefix's weights are rounded to bf16, 2^-8 of each, where that oracle counts 2^-16
    v = s.v.abs()
    mass = R.attention_whole(s.q, s.k, torch.where(torch.isfinite(v), v, 0), s.table, s.starts, s.lens, 0.1, window)[0]
    got, lse = paged.attention_shared(s.q.cuda(), kc, vc, table, starts, lens, gr, pt, pl, 0.1, window, True)
    assert ((got.cpu().double() - ref).abs() <= tol + 2.0 ** -8 * mass).all()
    assert ((lse.cpu().double() - rlse).abs() <= ltol).all()


def test_lengths_and_groups_outside():
    """Sequences shorter than their prefix or out of every range, prefixes past their
    table, ids that are no page: the entries that there are, and nothing past the pool."""
    from attention_nn_amd import paged
    s = Setup([(64, _one(1, 10, 10, 10, 10)), (64, _one(2, 10, 10))], H=2, Hk=2).widened()
    s.k, s.v = torch.nan_to_num(s.k, 1.0), torch.nan_to_num(s.v, 2.0, 2.0, 2.0)
    kc, vc, table, starts, lens, groups, pt, pl = s.dev()
    s.lens = [30, 64, 65, -7, 1, 3]      # inside the prefix, at its end, empty, and fewer than there are tokens
    lens = torch.tensor(s.lens, dtype=I32, device="cuda")
    got, lse = paged.attention_shared(s.q.cuda(), kc, vc, table, starts, lens, groups, pt, pl, 0.1, want_lse=True)
    _check(s, got, lse, 0.1, 0)
    s.lens = [10 ** 9] * 6               # the table's end
    lens = torch.tensor(s.lens, dtype=I32, device="cuda")
    s.table[s.table < 0] = 0
    got, lse = paged.attention_shared(s.q.cuda(), kc, vc, table, starts, lens, groups, pt, pl, 0.1, want_lse=True)
    _check(s, got, lse, 0.1, 0)
    big = torch.tensor([2 ** 31 - 1, 10 ** 6], dtype=I32, device="cuda")
    s.lens = [64, 63, 64, 2, 64, 60]     # prefixes that pass their table and the sequences' ends
    lens = torch.tensor(s.lens, dtype=I32, device="cuda")
    got, lse = paged.attention_shared(s.q.cuda(), kc, vc, table, starts, lens, groups, pt, big, 0.1, want_lse=True)
    _check(s, got, lse, 0.1, 0)
    for bad in ([-5, 4, 9], [0, 4, 2 ** 31 - 1], [3, 1, 0], [2 ** 31 - 1, -1, 5]):
        bad = torch.tensor(bad, dtype=I32, device="cuda")
        paged.attention_shared(s.q.cuda(), kc, vc, table, starts, lens, bad, pt * 0 + 2 ** 30, -big, 0.1)
    torch.cuda.synchronize()
    got, lse = paged.attention_shared(s.q.cuda(), kc, vc, table, starts, lens, groups[:1], pt[:0], pl[:0], 0.1, want_lse=True)
    _check(s, got, lse, 0.1, 0)


@pytest.mark.parametrize("where", ["prefix", "own"])
@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_what_is_not_finite_reaches_only_those_that_see_it(where, bad):
    """A value of one entry that some rows of a tile do not see, by their window or their length."""
    from attention_nn_amd import paged
    s = Setup([(100, [(4, 20), (1, 3), (1, 60), (9, 9)])], H=4, Hk=2, page=32).widened()
    window = 50
    e = 80 if where == "prefix" else 103
    for t in range(4):
        s.v[s.table[t, e // 32], :, e % 32, 5] = bad
    s.v[s.ptable[0, 80 // 32], :, 80 % 32, 5] = s.v[s.table[0, 80 // 32], :, 80 % 32, 5]
    kc, vc, table, starts, lens, groups, pt, pl = s.dev()
    got, lse = paged.attention_shared(s.q.cuda(), kc, vc, table, starts, lens, groups, pt, pl, 0.1, window, True)
    ref, rlse, tol, ltol = R.attention(s.q, s.k, s.v, s.table, s.starts, s.lens, 0.1, window)
    got = got.cpu().double()
    fine = torch.isfinite(ref)
    assert fine.any() and not fine.all()
    assert torch.equal(torch.isfinite(got), fine)
    assert ((got - ref).abs()[fine] <= tol[fine]).all()
    assert torch.equal(torch.isnan(got), torch.isnan(ref))


def test_rows_of_equal_maximum_and_far_scores():
    """Scores that differ by far between prefix and own entries, in both directions."""
    from attention_nn_amd import paged
    for sign in (1.0, -1.0):
        s = Setup([(70, _one(1, 9, 30))], H=2, Hk=2).widened()
        for t in range(2):
            s.k[s.ptable[0].long()] = (s.q[t].float().mean(0) * 0 + 0.1).to(BF)
        s.k = torch.nan_to_num(s.k, 0.0)
        s.v = torch.nan_to_num(s.v, 0.0, 0.0, 0.0)
        s.q[:] = 3.0 * sign
        s.k[s.ptable[0, 0], :, 3] = 30.0
        s.k[s.ptable[0, 0], :, 4] = -30.0
        for t in range(2):      # the tables' common page is the prefix's
            assert s.table[t, 0] == s.ptable[0, 0]
        # the page that the prefix ends in: both copies again
        a, full = int(s.ptable[0, 4]), 70 // 16
        for t in range(2):
            b = int(s.table[t, full])
            s.k[b, :, :70 % 16], s.v[b, :, :70 % 16] = s.k[a, :, :70 % 16], s.v[a, :, :70 % 16]
        kc, vc, table, starts, lens, groups, pt, pl = s.dev()
        got, lse = paged.attention_shared(s.q.cuda(), kc, vc, table, starts, lens, groups, pt, pl, 0.1, want_lse=True)
        _check(s, got, lse, 0.1, 0)


def test_strided_queries_streams_and_graph():
    from attention_nn_amd import paged
    s = Setup([(200, _one(1, *[70] * 9)), (33, _one(1, *[70] * 5))], H=4, Hk=2, page=32).widened()
    kc, vc, table, starts, lens, groups, pt, pl = s.dev()
    wide = torch.full((s.N, 2 * s.H + 3, s.D), math.nan, dtype=BF, device="cuda")
    q = wide[:, 1:1 + 2 * s.H:2]
    q.copy_(s.q)
    args = (kc, vc, table, starts, lens, groups, pt, pl, 0.1)
    want = paged.attention_shared(s.q.cuda(), *args, want_lse=True)
    got = paged.attention_shared(q, *args, want_lse=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    odd = torch.zeros(s.N * s.H * s.D + 3, dtype=BF, device="cuda")[3:].view(s.N, s.H, s.D)
    odd.copy_(s.q)
    wpt = torch.full((2, 2 * s.ptable.shape[1]), -1, dtype=I32, device="cuda")[:, ::2]
    wpt.copy_(s.ptable)
    got = paged.attention_shared(odd, kc, vc, table, starts, lens, groups, wpt, pl, 0.1)
    assert torch.equal(got, want[0])
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = paged.attention_shared(q, *args)
    st.synchronize()
    assert torch.equal(got, want[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = paged.attention_shared(q, *args, want_lse=True)
    for i in range(5):      # replayed with other lengths, prefixes and groups
        s.lens = [min(x, 200 - 40 * i + 30 + j) if j < 9 else 33 + 5 * i + 1 for j, x in enumerate(s.lens)]
        lens.copy_(torch.tensor(s.lens, dtype=I32))
        s.plens = [max(0, 200 - 40 * i), 33]
        pl.copy_(torch.tensor(s.plens, dtype=I32))
        graph.replay()
        torch.cuda.synchronize()
        _check(s, out, lse, 0.1, 0)
        eager = paged.attention_shared(q, *args)
        assert torch.equal(eager, out)
        (torch.ones(1000, device="cuda") * 2).sum()


def test_no_rows_and_no_sequences():
    from attention_nn_amd import paged
    s = Setup([(20, _one(1, 3))], H=2, Hk=2)
    kc, vc, table, starts, lens, groups, pt, pl = s.dev()
    assert paged.attention_shared(s.q.cuda()[:0], kc, vc, table, starts * 0, lens, groups, pt, pl, 0.1).shape == (0, 2, 128)
    out = torch.full((1, 2, 128), 7.0, dtype=BF, device="cuda")
    got = paged.attention_shared(s.q.cuda(), kc, vc, table[:0], starts[:1], lens[:0], groups, pt, pl, 0.1, out=out)
    assert (got == 7.0).all()
