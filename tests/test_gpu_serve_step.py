"""A serving step as it is used: pages for the next tokens, their keys and values
into the cache, attention behind shared prefixes, a token of each row, pages back.
And the sizes on both sides of each rule that picks a kernel."""

import pytest
import torch

import oracle.ref_paged as P
import oracle.ref_serve as R
from tests.test_gpu_page_tables import _pool, _same
from tests.test_gpu_sample_logits import _check

pytestmark = pytest.mark.gpu
BF, F32, I32 = torch.bfloat16, torch.float32, torch.int32
H, HK, D, PAGE, VOCAB, WIDTH = 4, 2, 64, 16, 500, 96


class Server:
    """Six requests: three behind a prefix of 40 entries, two behind one of 20, and one
    without.  A request whose token is in `stop` ends, and starts again behind its prefix."""

    COLS, PAGES, SEQS = 8, 60, 6

    def __init__(self, wide):
        g = torch.Generator().manual_seed(5)
        table = torch.full((self.SEQS, self.COLS), -1, dtype=I32)
        refs = torch.zeros(self.PAGES, dtype=I32)
        # columns that only make the tables wide enough for a prefix to be read once
        self.ptable = torch.full((2, 2048 if wide else 3), -1, dtype=I32)
        self.ptable[0, :3], self.ptable[1, :2] = torch.tensor([41, 3, 17]), torch.tensor([22, 9])
        self.plens, self.groups = [40, 20], [0, 3, 5]
        self.first = [32, 32, 32, 16, 16, 0]        # whole pages of the prefix
        for s in range(self.SEQS):
            if s < 5:
                ids = self.ptable[int(s >= 3), :self.first[s] // PAGE]
                table[s, :len(ids)] = ids
        for p in table[table >= 0].tolist() + [41, 3, 17, 22, 9]:
            refs[p] += 1
        self.h = (table.tolist(), self.first, refs.tolist())
        kc = torch.randn((self.PAGES, HK, PAGE, D), generator=g).to(BF)
        vc = torch.randn((self.PAGES, HK, PAGE, D), generator=g).to(BF)
        ang = torch.rand((256, D // 4), generator=g) * 6.28
        self.host = dict(kc=kc, vc=vc, table=table, refs=refs, lens=torch.tensor(self.first, dtype=I32),
                         new=torch.tensor([9, 9, 9, 6, 6, 11], dtype=I32), last=torch.arange(self.SEQS + 1),
                         u=torch.zeros(self.ROWS))
        self.dev = {k: v.cuda() for k, v in self.host.items()}
        self.cs, self.sn = ang.cos().cuda(), ang.sin().cuda()
        self.emb = torch.randn((VOCAB, WIDTH), generator=g).to(BF).cuda()
        self.wq, self.wk, self.wv = (torch.randn((WIDTH, n * D), generator=g).mul(WIDTH ** -0.5).to(BF).cuda()
                                     for n in (H, HK, HK))
        self.head = torch.randn((H * D, VOCAB), generator=g).mul(0.4).to(BF).cuda()
        self.stop = torch.zeros(VOCAB, dtype=torch.bool, device="cuda")
        self.stop[::7] = True
        self.back = torch.tensor(self.first, dtype=I32, device="cuda")
        self.x = [t.cuda() for t in (torch.tensor(self.groups, dtype=I32), self.ptable, torch.tensor(self.plens, dtype=I32))]
        # a prefix that ends within a page: as far as whole pages of it are everyone's
        self.x[2].copy_(torch.tensor([32, 16], dtype=I32))

    ROWS = 56

    def reset(self):
        for k, v in self.host.items():
            self.dev[k].copy_(v)

    def step(self):
        from attention_nn_amd import kernels, paged
        d = self.dev
        a = paged.assign(d["table"], d["lens"], d["new"], d["refs"], PAGE, self.ROWS, out=d["table"],
                         refs_out=d["refs"], lens_out=d["lens"])
        who = torch.where(a.seq < 0, self.SEQS, a.seq).long()
        x = self.emb[d["last"][who]]
        q, k, v = ((x @ w).view(self.ROWS, -1, D) for w in (self.wq, self.wk, self.wv))
        q = paged.append(q, k, v, self.cs, self.sn, d["kc"], d["vc"], a.table, a.starts, a.lens)
        y, lse = paged.attention_shared(q, d["kc"], d["vc"], a.table, a.starts, a.lens, *self.x, 0.2, want_lse=True,
                                        out=torch.zeros_like(q))
        ends = (a.starts[1:] - 1).clamp(min=0).long()
        logits = y.view(self.ROWS, H * D)[ends] @ self.head
        ids, lp = kernels.sample_logits(logits, d["u"][:self.SEQS], 0.9, 60, 0.95, 0.001, want_logprob=True)
        ran = a.starts[1:] > a.starts[:-1]
        done = ran & self.stop[ids.clamp(min=0).long()]
        d["last"][:self.SEQS] = torch.where(ran, ids.long(), d["last"][:self.SEQS])
        stepped = a.table.clone(), a.refs.clone(), a.lens.clone()
        d["lens"].copy_(torch.where(done, self.back, a.lens))
        d["new"].copy_(torch.where(done, 5, 1))
        paged.release(d["table"], d["lens"], d["refs"], PAGE, out=d["table"], refs_out=d["refs"])
        return dict(a=a, stepped=stepped, q=q, y=y, lse=lse, logits=logits, ids=ids, lp=lp, done=done, ran=ran)


@pytest.mark.parametrize("wide", [True, False])
def test_steps(wide, traced):
    s = Server(wide)
    names = traced(s.step, tries=1)
    assert any("k_paged_shared" in n for n in names) == wide
    s.reset()
    g = torch.Generator().manual_seed(1)
    us = torch.rand((14, s.ROWS), generator=g)
    table, lens, refs = s.h
    new = s.host["new"].tolist()
    eager, ended = [], 0
    for i in range(14):
        s.dev["u"].copy_(us[i])
        r = s.step()
        ref = R.assign(table, lens, new, refs, PAGE, s.ROWS)
        t, rf, ln = (v.cpu() for v in r["stepped"])
        assert t.tolist() == ref["table"] and rf.tolist() == ref["refs"] and ln.tolist() == ref["lens"]
        for name in ("starts", "seq", "pos", "slot"):
            assert getattr(r["a"], name).cpu().tolist() == ref[name], name
        starts = ref["starts"]
        o, lse, tol, ltol = P.attention(r["q"].cpu().float(), s.dev["kc"].cpu().float(), s.dev["vc"].cpu().float(), t,
                                        starts, ref["lens"], 0.2, 0)
        n = starts[-1]
        assert n and ((r["y"].cpu().double() - o).abs() <= tol)[:n].all() and (r["y"].cpu()[n:] == 0).all()
        assert ((r["lse"].cpu().double() - lse).abs() <= ltol)[:n].all()
        _check(r["logits"].cpu(), us[i, :s.SEQS], (r["ids"], r["lp"]), dict(temperature=0.9, top_k=60, top_p=0.95, min_p=0.001))
        done = r["done"].cpu().tolist()
        ended += sum(done)
        lens = [f if d else m for d, f, m in zip(done, s.first, ref["lens"])]
        new = [5 if d else 1 for d in done]
        table, refs = R.release(ref["table"], lens, ref["refs"], PAGE)
        assert s.dev["table"].cpu().tolist() == table and s.dev["refs"].cpu().tolist() == refs
        eager.append((r["ids"].cpu(), r["lp"].cpu(), n))
    assert ended >= 3 and all(refs[p] for p in (41, 3, 17, 22, 9))

    s.reset()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = s.step()
    s.reset()
    for i in range(14):
        s.dev["u"].copy_(us[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(r["ids"].cpu(), eager[i][0]) and torch.equal(r["lp"].cpu(), eager[i][1])
        (torch.ones(1000, device="cuda") * 2).sum()
    assert s.dev["table"].cpu().tolist() == table and s.dev["refs"].cpu().tolist() == refs


# ---- sizes on both sides of the rules ------------------------------------------------

TABLES = [
    # sequences, columns, spare pages, rows, whether one launch assigns, releases
    (64, 64, 5, 64, True, True), (65, 64, 5, 64, False, False), (64, 65, 5, 64, False, False),
    (1, 64 * 64, 5, 300, True, True), (1, 64 * 64 + 1, 5, 300, False, False), (3, 70, 16384 - 210, 40, True, False),
    (3, 70, 16385 - 210, 40, False, False), (3, 70, 12288 - 210, 40, True, True), (3, 70, 12289 - 210, 40, True, False),
    (2, 4, 5, 8192, True, True), (2, 4, 5, 8193, False, True), (16, 200, 5, 8192, True, True),
]


@pytest.mark.parametrize("i", range(len(TABLES)))
def test_tables_by_size(i, traced):
    from attention_nn_amd import paged
    S, cols, spare, rows, one, back = TABLES[i]
    table, lens, refs, g = _pool(S, cols, 16, 40 + i, spare=spare)
    most = max(1, rows // S)
    new = torch.minimum(torch.randint(0, most + 1, (S,), generator=g).to(I32), cols * 16 - lens).to(I32)
    t, l, n, r = table.cuda(), lens.cuda(), new.cuda(), refs.cuda()
    ref = R.assign(table.tolist(), lens.tolist(), new.tolist(), refs.tolist(), 16, rows)
    got = []
    names = traced(lambda: got.append(paged.assign(t, l, n, r, 16, rows)))
    assert any("k_table_one" in x for x in names) == one and any("k_table_fill" in x for x in names) != one
    for x in got:
        _same(x, ref)
    short = torch.where(torch.rand(S, generator=g) < 0.5, lens // 2, 0).to(I32)
    wt, wr = R.release(ref["table"], short.tolist(), ref["refs"], 16)
    names = traced(lambda: got.append(paged.release(x.table, short.cuda(), x.refs, 16)))
    assert any("k_table_release_one" in x for x in names) == back
    assert got[-1][0].cpu().tolist() == wt and got[-1][1].cpu().tolist() == wr
    out = paged.release(x.table, short.cuda(), x.refs, 16, out=x.table, refs_out=x.refs)
    assert out[0].cpu().tolist() == wt and out[1].cpu().tolist() == wr


@pytest.mark.parametrize("page", [16, 64, 128, 1024])
@pytest.mark.parametrize("first", [0, 7777])
def test_long_prompts(first, page):
    """Many columns of one sequence: whole spans, parts of them at both ends, some
    named already; and one that asks for more than there are rows, behind which none is served."""
    from attention_nn_amd import paged
    cols = 70000 // page
    g = torch.Generator().manual_seed(page + first)
    table = torch.full((4, cols), -1, dtype=I32)
    pages = 2 * cols + 40
    order = torch.randperm(pages, generator=g).to(I32)
    table[0, :-(-first // page)] = order[:-(-first // page)]
    held = torch.rand(cols, generator=g) < 0.3
    table[1, held] = order[cols:2 * cols][held]
    refs = torch.zeros(pages, dtype=I32)
    refs[table[table >= 0].long()] = 1
    lens = torch.tensor([first, 1, 0, 0], dtype=I32)
    for new in ([60001, 1, 3, 1], [1, 40000, 0, 2], [5, 66000, 9, 1]):
        rows = 60010
        ref = R.assign(table.tolist(), lens.tolist(), new, refs.tolist(), page, rows)
        got = paged.assign(table.cuda(), lens.cuda(), torch.tensor(new, dtype=I32).cuda(), refs.cuda(), page, rows)
        _same(got, ref)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("k", [895, 896, 897, 4000, 8191, 8192, 8193, 20000])
def test_draws_of_many_kept(k, dtype):
    """The k at which a bound of the threads' maxima ends, and as many entries as a list
    holds, one more and one less."""
    from attention_nn_amd import kernels
    g = torch.Generator().manual_seed(k)
    x = torch.full((2, 30001), -50.0)
    x[:, torch.randperm(30001, generator=g)[:k]] = (torch.rand((2, k), generator=g) - 0.5) * 0.25
    x = x.to(dtype)
    u = torch.tensor([0.37, 0.99])
    for kw in (dict(top_k=k), dict(min_p=0.01), dict(min_p=0.01, top_p=0.7), dict(top_k=k, top_p=0.9), dict(top_p=0.5)):
        _check(x, u, kernels.sample_logits(x.cuda(), u.cuda(), want_logprob=True, **kw), kw)


@pytest.mark.parametrize("n", [255, 256, 257, 511, 513])
def test_draws_by_one_wave_and_by_more(n):
    from attention_nn_amd import kernels
    g = torch.Generator().manual_seed(n)
    x = torch.full((3, 6000), -90.0)
    x[:, torch.randperm(6000, generator=g)[:n]] = torch.rand((3, n), generator=g)
    u = torch.tensor([0.0, 0.5, 0.999])
    for kw in (dict(top_k=n), dict(min_p=0.2), dict(top_k=n, top_p=0.6, min_p=0.3), dict(top_k=n - 1)):
        _check(x, u, kernels.sample_logits(x.cuda(), u.cuda(), want_logprob=True, **kw), kw)


def test_infinite_settings():
    """A temperature past every number makes all alike, an infinite min_p keeps the
    largest, and what is masked stays so."""
    from attention_nn_amd import kernels
    inf = float("inf")
    x = torch.tensor([[1.0, -inf, 3.0, torch.finfo(F32).min, 2.0, -inf]] * 3)
    u = torch.tensor([0.1, 0.6, 0.9])
    for kw in (dict(temperature=inf), dict(min_p=inf), dict(top_p=inf), dict(temperature=inf, top_p=0.4),
               dict(temperature=1e-45), dict(top_k=2 ** 31 - 1)):
        _check(x, u, kernels.sample_logits(x.cuda(), u.cuda(), want_logprob=True, **kw), kw)


def test_two_calls_at_once():
    """Steps of two pools on two streams: neither has a part in the other's workspaces."""
    from attention_nn_amd import kernels, paged
    jobs = []
    for seed in range(2):
        table, lens, refs, g = _pool(200, 12, 16, seed)
        new = torch.randint(0, 9, (200,), generator=g).to(I32)
        x = torch.randn((7, 50257), generator=g)
        u = torch.rand(7, generator=g)
        ref = R.assign(table.tolist(), lens.tolist(), new.tolist(), refs.tolist(), 16, 900)
        want = [R.sample(x[r].numpy(), u[r].item(), top_p=0.9)[0] for r in range(7)]
        jobs.append((torch.cuda.Stream(), [t.cuda() for t in (table, lens, new, refs, x, u)], ref, want, []))
    torch.cuda.synchronize()
    for _ in range(20):
        for st, (t, l, n, r, x, u), _, _, out in jobs:
            with torch.cuda.stream(st):
                out.append((paged.assign(t, l, n, r, 16, 900), kernels.sample_logits(x, u, top_p=0.9)))
    torch.cuda.synchronize()
    for _, _, ref, want, out in jobs:
        for a, ids in out:
            _same(a, ref)
            assert ids.tolist() == want


def test_refused_on_the_gpu():
    """What the Python layer refuses of GPU tensors: types, shapes, layouts."""
    from attention_nn_amd import kernels, paged
    i = torch.zeros((3, 4), dtype=I32, device="cuda")
    n, r = i[:, 0].contiguous(), torch.zeros(9, dtype=I32, device="cuda")
    assert paged.assign(i, n, n, r, 16, 2).starts.tolist() == [0] * 4
    for args, kw in (((i.long(), n, n, r, 16, 2), {}), ((i, n[:2], n, r, 16, 2), {}), ((i, n, n.float(), r, 16, 2), {}),
                     ((i, n, n, r, 24, 2), {}), ((i, n, n, r, 16, -1), {}), ((i[0], n, n, r, 16, 2), {}),
                     ((i, n, n, r, 16, 2), dict(out=i[:, :2])), ((i, n, n, r, 16, 2), dict(refs_out=r[:5])),
                     ((i, n, n, r, 16, 2), dict(refs_out=r[::2])), ((i, n, n, r, 16, 2), dict(lens_out=n[:1])),
                     ((i, n, n.cpu(), r, 16, 2), {}), ((i, n, n, i[0, :2], 16, 2), dict(out=i)),
                     ((i[:1].expand(3, 4), n, n, r, 16, 2), dict(out=i[:1].expand(3, 4)))):
        with pytest.raises((TypeError, ValueError, RuntimeError)):
            paged.assign(*args, **kw)
    for args in ((i, n[:2], r, 16), (i, n, r.long(), 16), (i, n, r, 0), (i, n, r, -16)):
        with pytest.raises((TypeError, ValueError, RuntimeError)):
            paged.release(*args)
    x, u = torch.zeros((3, 50), device="cuda"), torch.zeros(3, device="cuda")
    for args, kw in (((x.double(), u), {}), ((x[0], u), {}), ((x, u[:2]), {}), ((x, u.double()), {}), ((x, u.cpu()), {}),
                     ((x, u), dict(temperature=-1.0)), ((x, u), dict(temperature=u[:1])), ((x, u), dict(top_k=-2)),
                     ((x, u), dict(top_k=u)), ((x, u), dict(top_p=float("nan"))), ((x, u), dict(min_p=-0.1)),
                     ((x[:, :0], u), {}), ((x, None), {})):
        with pytest.raises((TypeError, ValueError, RuntimeError)):
            kernels.sample_logits(*args, **kw)
    q = torch.zeros((3, 2, 64), dtype=BF, device="cuda")
    c = torch.zeros((9, 2, 16, 64), dtype=BF, device="cuda")
    st, g2, t1 = torch.arange(4, dtype=I32, device="cuda"), n[:2] * 0, i[:1]
    ok = dict(q=q, k_cache=c, v_cache=c, table=i, starts=st, lens=n + 1, groups=g2, prefix_table=t1, prefix_lens=n[:1], scale=0.1)
    assert paged.attention_shared(**ok).shape == q.shape
    for kw in (dict(groups=n), dict(prefix_lens=n), dict(prefix_table=t1.long()), dict(prefix_table=t1[0]),
               dict(groups=g2.cpu()), dict(q=q.float()), dict(q=q[:, :, :32]), dict(starts=n), dict(lens=st),
               dict(out=q.float()), dict(out=q[:2]), dict(window=-1), dict(scale=float("inf"))):
        with pytest.raises((TypeError, ValueError, RuntimeError)):
            paged.attention_shared(**{**ok, **kw})


@pytest.mark.parametrize("wide", [True, False])
def test_results_in_place_of_the_queries(wide, traced):
    """Sequences of few tokens and of many behind prefixes, and one of none."""
    from attention_nn_amd import paged
    from tests.test_gpu_paged_shared import Setup
    s = Setup([(130, [(1, 5), (2, 40), (40, 60)]), (70, [(3, 9), (100, 130)]), (None, [(1, 33)])], H=4, Hk=2, D=64, page=32)
    s = s.widened() if wide else s
    args = s.dev()
    q = s.q.cuda()
    want, lse = paged.attention_shared(q.clone(), *args, 0.1, want_lse=True)
    got = []
    names = traced(lambda: got.append(paged.attention_shared(q.clone(), *args, 0.1)))
    assert any("k_paged_shared" in n for n in names) == wide
    for _ in range(3):
        x = q.clone()
        y, l = paged.attention_shared(x, *args, 0.1, want_lse=True, out=x)
        assert y is x and torch.equal(y, want) and torch.equal(l, lse)


@pytest.mark.parametrize("S,cols,spare,rows,runs", [
    (1024, 2, 5, 700, "k_table_fill<true>"), (1025, 2, 5, 700, "k_table_fill<false>"),
    (70, 3, (1 << 20) - 210, 300, "k_table_fill<true>"), (70, 3, (1 << 20) - 209, 300, "k_table_fill<false>"),
    (70, 30, 5, 1 << 21, "k_table_fill<true>"), (70, 30, 5, (1 << 21) + 1, "k_table_fill<false>"),
])
@pytest.mark.parametrize("short", [False, True])
def test_sums_by_one_and_by_all(S, cols, spare, rows, runs, short, traced):
    """Who is served, summed up by every work-group of the last launch or by one before it;
    with rows or pages for half of them."""
    from attention_nn_amd import paged
    page = 16 if rows < 1 << 20 else 1024
    table, lens, refs, g = _pool(S, cols, page, S + spare, spare=spare)
    if short:
        refs[torch.rand(len(refs), generator=g) < 1 - S / 4 / len(refs)] += 3
    new = torch.minimum(torch.randint(0, page + 3, (S,), generator=g).to(I32), cols * page - lens).to(I32)
    ref = R.assign(table.tolist(), lens.tolist(), new.tolist(), refs.tolist(), page, rows)
    t, l, n, r = table.cuda(), lens.cuda(), new.cuda(), refs.cuda()
    got = []
    names = traced(lambda: got.append(paged.assign(t, l, n, r, page, rows)))
    assert any(runs in x for x in names), names
    for x in got:
        _same(x, ref)
    _same(paged.assign(t, l, n, r, page, rows, out=t, refs_out=r, lens_out=l), ref)


def test_more_rows_than_a_launch_holds():
    """Two and a little more launches, settings and results of each row its own."""
    from attention_nn_amd import kernels
    n = (1 << 22) + 3
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.rand((n, 2), generator=g, device="cuda")
    u = torch.rand(n, generator=g, device="cuda")
    t = (torch.rand(n, generator=g, device="cuda") < 0.5).float()
    ids, lp = kernels.sample_logits(x, u, temperature=t, want_logprob=True)
    p0 = torch.softmax(x.double(), 1)[:, 0]
    drawn = (u.double() >= p0).int()
    best = (x[:, 1] > x[:, 0]).int()
    near = (u.double() - p0).abs() < 2.0 ** -40
    want = torch.where(t > 0, drawn, best)
    assert ((ids == want) | near).all()
    share = torch.where(ids == 0, p0, 1 - p0).log()
    assert ((lp.double() - torch.where(t > 0, share, 0.0)).abs() <= 2.0 ** -22).all()


def test_pages_past_32_bits():
    """Prefixes and own entries in pages whose offsets in the cache pass 2^31 elements."""
    from attention_nn_amd import paged
    from tests.test_gpu_paged_shared import Setup
    s = Setup([(70, [(1, 9), (2, 50), (20, 40)]), (33, [(1, 3)])], H=4, Hk=2, D=64, page=16).widened()
    kc, vc, table, starts, lens, groups, pt, pl = s.dev()
    q = s.q.cuda()
    want, lse = paged.attention_shared(q, kc, vc, table, starts, lens, groups, pt, pl, 0.1, want_lse=True)
    pages = kc.shape[0]
    by = (1 << 31) // (kc[0].numel() * (pages // 2))      # the upper half of them lies past
    far = []
    for x in (kc, vc):
        big = torch.empty((pages * by, *x.shape[1:]), dtype=BF, device="cuda")
        big[::by] = x
        far.append(big)
    assert far[0].numel() > 1 << 31
    got, l2 = paged.attention_shared(q, *far, torch.where(table >= 0, table * by, -1), starts, lens, groups,
                                     torch.where(pt >= 0, pt * by, -1), pl, 0.1, want_lse=True)
    assert torch.equal(got, want) and torch.equal(l2, lse)


def test_slots_past_32_bits():
    from attention_nn_amd import paged
    pages, page = (1 << 22) + 5, 1024
    for S in (3, 1200):       # two launches, and three
        refs = torch.ones(pages, dtype=I32, device="cuda")
        refs[-4 * S:] = 0
        table = torch.full((S, 4), -1, dtype=I32, device="cuda")
        new = torch.full((S,), 1500, dtype=I32, device="cuda")
        a = paged.assign(table, new * 0, new, refs, page, S * 1500)
        first = pages - 4 * S
        assert (a.table[:, :2] == first + torch.arange(2 * S, device="cuda").view(S, 2)).all() and (a.table[:, 2:] == -1).all()
        assert torch.equal(a.slot, a.table[a.seq.long(), a.pos.long() // page].long() * page + a.pos % page)
        assert int(a.slot.max()) > 1 << 31 and int(a.refs.sum()) == pages - 4 * S + 2 * S
        table, refs = paged.release(a.table, new * 0 + 1024, a.refs, page)
        assert (table[:, 0] == a.table[:, 0]).all() and (table[:, 1:] == -1).all() and int(refs.sum()) == pages - 3 * S


@pytest.mark.parametrize("dtype", [F32, BF])
def test_rows_past_32_bits(dtype):
    from attention_nn_amd import kernels
    g = torch.Generator().manual_seed(8)
    x, u = torch.randn((4, 777), generator=g).to(dtype), torch.rand(4, generator=g)
    far = torch.empty(3 * (1 << 30) + 777, dtype=dtype, device="cuda").as_strided((4, 777), (1 << 30, 1))
    far.copy_(x)
    _check(x, u, kernels.sample_logits(far, u.cuda(), top_p=0.8, want_logprob=True), dict(top_p=0.8))


@pytest.mark.parametrize("dtype,groups", [(F32, n) for n in (1, 2, 3, 4, 5, 8, 9, 13, 14)] + [(BF, n) for n in (1, 2, 3, 4, 5, 7, 8)])
def test_draws_by_the_row_s_groups(dtype, groups):
    """Rows that fill a number of groups of 16-byte words a wave, and one entry less or more, at
    every alignment: as many as are held in registers, and longer."""
    from attention_nn_amd import kernels
    words = 4 if dtype is F32 else 8
    g = torch.Generator().manual_seed(groups)
    for cols in (groups * 1024 * words, groups * 1024 * words - words + 1, groups * 1024 * words + 1):
        base = torch.empty((2, cols + 8), dtype=dtype, device="cuda")
        x = (3.0 * torch.randn((2, cols), generator=g)).to(dtype)
        u = torch.rand(2, generator=g)
        for off in (0, 1, words - 1):
            v = base[:, off:off + cols]
            v.copy_(x)
            for kw in (dict(top_p=0.9), dict(temperature=0.5, min_p=0.01), dict(top_k=40), dict(temperature=0.0)):
                _check(x, u, kernels.sample_logits(v, u.cuda(), want_logprob=True, **kw), kw)
