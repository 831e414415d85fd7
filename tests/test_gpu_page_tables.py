"""Pages given to sequences and taken back (paged.assign, paged.release) against
plain lists: exact numbers."""

import pytest
import torch

import oracle.ref_serve as R

pytestmark = pytest.mark.gpu
I32 = torch.int32


def _pool(S, cols, page, seed, full=0.4, junk=True, spare=5):
    """A table that holds pages for random lengths, a pool with others in use."""
    g = torch.Generator().manual_seed(seed)
    pages = S * cols + spare
    order = torch.randperm(pages, generator=g).to(I32)
    cap = cols * page
    lens = torch.randint(0, cap + 1, (S,), generator=g).to(I32)
    have = (lens + page - 1) // page
    c = torch.arange(cols)
    held = c < have[:, None]
    table = torch.where(held, order[:S * cols].view(S, cols), -1).to(I32)
    if junk:   # columns behind may name a page already, or hold what is no page
        some = (torch.rand((S, cols), generator=g) < 0.1) & ~held
        table = torch.where(some, order[:S * cols].view(S, cols), table)
        some = (torch.rand((S, cols), generator=g) < 0.1) & ~held & ~some
        table = torch.where(some, pages + 7, table)
    refs = torch.zeros(pages, dtype=I32)
    for p in table[(table >= 0) & (table < pages)].tolist():
        refs[p] += 1
    refs += ((torch.rand(pages, generator=g) < full) & (refs == 0)).to(I32)
    refs[::7] = torch.where(refs[::7] == 0, -2, refs[::7])
    return table, lens, refs, g


def _same(got, ref):
    for name in ("table", "refs", "starts", "lens", "seq", "pos", "slot"):
        want = torch.tensor(ref[name], dtype=getattr(got, name).dtype)
        assert torch.equal(getattr(got, name).cpu().flatten(), want.flatten()), name


CASES = [
    # sequences, columns, page, most new tokens, share of the asked rows that there are
    (1, 1, 16, 1, 1.0), (1, 3, 16, 40, 1.0), (3, 5, 32, 1, 1.0), (64, 8, 16, 1, 1.0),
    (65, 4, 16, 30, 0.7), (7, 40, 64, 2000, 1.0), (5, 9, 1024, 5000, 1.0), (4, 300, 16, 4800, 1.0),
    (300, 3, 16, 20, 1.0), (1100, 2, 16, 3, 0.9), (2, 700, 16, 9000, 1.0), (1, 70, 128, 8000, 1.0),
    (12, 33, 256, 1500, 0.5), (2500, 2, 32, 1, 1.0),
]


@pytest.mark.parametrize("full", [0.0, 0.5, 0.97])
@pytest.mark.parametrize("i", range(len(CASES)))
def test_assign(i, full):
    from attention_nn_amd import paged
    S, cols, page, most, share = CASES[i]
    table, lens, refs, g = _pool(S, cols, page, i, full)
    new = torch.randint(0, most + 1, (S,), generator=g).to(I32)
    new = torch.where(torch.rand(S, generator=g) < 0.7, torch.minimum(new, cols * page - lens), new).to(I32)
    rows = int(int(new.sum()) * share) + 3
    ref = R.assign(table.tolist(), lens.tolist(), new.tolist(), refs.tolist(), page, rows)
    t, l, n, r = table.cuda(), lens.cuda(), new.cuda(), refs.cuda()
    got = paged.assign(t, l, n, r, page, rows)
    _same(got, ref)
    assert torch.equal(t.cpu(), table) and torch.equal(r.cpu(), refs) and torch.equal(l.cpu(), lens)
    # in place, and again: what is held already is kept
    again = paged.assign(t, l, n, r, page, rows, out=t, refs_out=r, lens_out=l)
    assert again.table is t and again.refs is r and again.lens is l
    _same(again, ref)
    third = paged.assign(got.table, lens.cuda(), (got.starts[1:] - got.starts[:-1]), got.refs, page, rows)
    _same(third, {**ref})


def test_assign_odd_numbers():
    from attention_nn_amd import paged
    big = 2 ** 31 - 1
    table = torch.tensor([[0, 1], [2, -1], [-5, 99], [big, -big - 1], [3, -1]], dtype=I32)
    lens = torch.tensor([-4, 9, 70, 0, 16], dtype=I32)
    new = torch.tensor([3, big, 1, 20, -9], dtype=I32)
    refs = torch.tensor([1, 1, 1, 1, 0, 0, -big, 4], dtype=I32)
    ref = R.assign(table.tolist(), lens.tolist(), new.tolist(), refs.tolist(), 16, 64)
    _same(paged.assign(table.cuda(), lens.cuda(), new.cuda(), refs.cuda(), 16, 64), ref)


def test_assign_of_nothing():
    from attention_nn_amd import paged

    def i(*shape):
        return torch.zeros(shape, dtype=I32, device="cuda")

    got = paged.assign(i(0, 4), i(0), i(0), i(70), 16, 3)
    assert got.starts.tolist() == [0] and got.seq.tolist() == [-1] * 3 and got.slot.tolist() == [-1] * 3
    assert got.refs.tolist() == [0] * 70
    got = paged.assign(i(3, 0), i(3), i(3) + 1, i(9), 16, 3)
    assert got.starts.tolist() == [0] * 4 and got.table.shape == (3, 0)
    got = paged.assign(i(2, 2) - 1, i(2), i(2) + 1, i(9), 16, 0)
    assert got.starts.tolist() == [0] * 3 and got.seq.shape == (0,)


def test_assign_strided_and_other_stream():
    from attention_nn_amd import paged
    table, lens, refs, g = _pool(9, 6, 16, 3)
    new = torch.full((9,), 5, dtype=I32)
    ref = R.assign(table.tolist(), lens.tolist(), new.tolist(), refs.tolist(), 16, 60)
    wide = torch.full((18, 9), 77, dtype=I32, device="cuda")
    t = wide[::2, 2:8]
    t.copy_(table)
    other = torch.full((9, 11), 55, dtype=I32, device="cuda")
    l2 = torch.stack((lens, new), 1).cuda()
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        got = paged.assign(t, l2[:, 0], l2[:, 1], refs.cuda(), 16, 60, out=other[:, 3:9])
    st.synchronize()
    _same(got, ref)
    assert (other[:, :3] == 55).all() and (other[:, 9:] == 55).all()
    got = paged.assign(t, l2[:, 0], l2[:, 1], refs.cuda(), 16, 60, out=t)
    _same(got, ref)
    assert (wide[1::2] == 77).all() and (wide[:, :2] == 77).all() and (wide[:, 8:] == 77).all()
    across = torch.empty((6, 9), dtype=I32, device="cuda").t()   # columns apart: a copy is read
    across.copy_(table)
    _same(paged.assign(across, l2[:, 0], l2[:, 1], refs.cuda(), 16, 60), ref)


@pytest.mark.parametrize("i", range(len(CASES)))
def test_release(i):
    from attention_nn_amd import paged
    S, cols, page, _, _ = CASES[i]
    table, lens, refs, g = _pool(S, cols, page, i)
    table[0] = table[S - 1]     # shared pages lose both
    left = (lens.float() * torch.rand(S, generator=g)).to(I32)
    left = torch.where(torch.rand(S, generator=g) < 0.4, 0, left).to(I32)
    left[0] = -3
    want_t, want_r = R.release(table.tolist(), left.tolist(), refs.tolist(), page)
    t, r = table.cuda(), refs.cuda()
    got_t, got_r = paged.release(t, left.cuda(), r, page)
    assert got_t.cpu().tolist() == want_t and got_r.cpu().tolist() == want_r
    assert torch.equal(t.cpu(), table) and torch.equal(r.cpu(), refs)
    assert paged.release(t, left.cuda(), r, page, out=t, refs_out=r)[0] is t
    assert torch.equal(t, got_t) and torch.equal(r, got_r)
    paged.release(t, left.cuda(), r, page, out=t, refs_out=r)   # nothing is left to give back
    assert torch.equal(t, got_t) and torch.equal(r, got_r)
    one = paged.release(table.cuda(), left.cuda(), refs.cuda(), page, refs_out=(x := refs.cuda()))
    assert one[1] is x and torch.equal(x, got_r) and torch.equal(one[0], got_t)


def test_steps_in_a_graph():
    """Assign in place, then one request ends and gives its pages back: replayed, the
    tables go on from where they were."""
    from attention_nn_amd import paged
    S, cols, page, rows = 6, 12, 16, 64
    table = torch.full((S, cols), -1, dtype=I32)
    lens, new = torch.zeros(S, dtype=I32), torch.tensor([5, 17, 1, 0, 9, 20], dtype=I32)
    refs = torch.zeros(40, dtype=I32)
    t, l, n, r = table.cuda(), lens.cuda(), new.cuda(), refs.cuda()
    drop = torch.zeros(S, dtype=I32, device="cuda")

    def step():
        a = paged.assign(t, l, n, r, page, rows, out=t, refs_out=r, lens_out=l)
        l.copy_(torch.where(drop > 0, 0, l))
        paged.release(t, l, r, page, out=t, refs_out=r)
        return a

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()      # warm
        side.synchronize()
    torch.cuda.current_stream().wait_stream(side)
    t.copy_(table), l.copy_(lens), r.copy_(refs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a = step()
    ht, hl, hr = table.tolist(), lens.tolist(), refs.tolist()
    t.copy_(table), l.copy_(lens), r.copy_(refs)
    for i in range(12):
        gone = [int(i % 5 == s) for s in range(S)]
        drop.copy_(torch.tensor(gone, dtype=I32))
        graph.replay()
        torch.cuda.synchronize()
        ref = R.assign(ht, hl, new.tolist(), hr, page, rows)
        hl = [0 if d else x for d, x in zip(gone, ref["lens"])]
        ht, hr = R.release(ref["table"], hl, ref["refs"], page)
        assert t.cpu().tolist() == ht and r.cpu().tolist() == hr and l.cpu().tolist() == hl
        assert a.starts.cpu().tolist() == ref["starts"] and a.slot.cpu().tolist() == ref["slot"]
        (torch.ones(1000, device="cuda") * 2).sum()     # eager work between replays
    assert max(hr) <= 1 and sum(hr) == sum(x >= 0 for row in ht for x in row)
