"""A serving step around the paged cache, as cases that can be timed and checked:
the block tables of a step from the requests' lengths and the pages' return, the
attention of a batch whose sequences begin with the same prefix, and the draw of
the next tokens from the logits.

    listed()        the named cases
    draw(rng)       one more case of the same ranges
    prepare(c, s)   what a program holds before the call, made from seed s
    run(state)      one pass; returns its outputs
    work(c)         bytes and operations that a pass cannot do without
    exact(c, s)     the same outputs from the definition, on the host or in 64 bits

A cache is two tensors (pages, kv_heads, page, head_dim) in bf16; row s of a
table holds the pages of sequence s in order, -1 where it has none.  refs counts
the tables that name each page; a page that none names is free.  Head layouts
are those of the 155M shape (6 x 128), the command line's default (8 x 64), the
wide shape (12 x 128) and two with shared key/value heads; the vocabulary is the
framework's 50257 tokens in rows of 50304, or another one.
"""

import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
EPS = 1e-6
SCALE = 0.1             # the framework's attention scale
WINDOW = 384            # and its sliding window
VOCAB, WIDTH = 50257, 50304
LEAST = 2.0 ** -40      # entries of a smaller share of the largest's weight are not drawn

# (query heads, key/value heads, head_dim)
HEADS = ((6, 6, 128), (8, 8, 64), (12, 12, 128), (8, 2, 128), (12, 3, 64))


# ---- the cases ----------------------------------------------------------------

def _case(kind, **kw):
    return {"kind": kind, **kw}


def listed():
    return [
        # a decode step of a serving batch: a new page now and then
        dict(_case("assign", seqs=64, new=1, ctx=1024, page=16, rows=64, full=0.5),
             name="assign_decode"),
        # prompts of several requests beside decoding ones, in a pool that does
        # not hold them all
        dict(_case("assign", seqs=48, new=2000, ctx=4096, page=32, rows=16384, full=0.8),
             name="assign_prompts"),
        # a wide step over a large pool
        dict(_case("assign", seqs=1000, new=8, ctx=8192, page=16, rows=8192, full=0.4),
             name="assign_wide"),
        # a few requests of a batch end or are cut back
        dict(_case("release", seqs=64, ctx=1024, page=16, ends=0.3), name="release_some"),
        # many of long ones do
        dict(_case("release", seqs=1000, ctx=8192, page=16, ends=0.5), name="release_wide"),
        # one decode step of a small batch behind one instruction
        dict(_case("shared", groups=1, seqs=8, new=1, prefix=1000, own=200, heads=6, kv_heads=6,
                   head_dim=128, page=16, window=0), name="shared_small"),
        # a large one behind a long one
        dict(_case("shared", groups=1, seqs=64, new=1, prefix=8192, own=256, heads=12, kv_heads=12,
                   head_dim=128, page=64, window=0), name="shared_long"),
        # several prefixes, shared key/value heads, a few drafted tokens each
        dict(_case("shared", groups=4, seqs=12, new=4, prefix=3001, own=333, heads=8, kv_heads=2,
                   head_dim=128, page=32, window=0), name="shared_groups"),
        # chunks of prompts beside decoding requests
        dict(_case("shared", groups=2, seqs=12, new=300, prefix=4096, own=700, heads=8, kv_heads=8,
                   head_dim=64, page=64, window=0), name="shared_mixed"),
        # interactive generation: one row, the command line's settings
        dict(_case("draw", dtype="f32", rows=1, vocab=VOCAB, width=WIDTH, temperature=0.8, top_k=50,
                   top_p=1.0, min_p=0.0, each=False), name="draw_one"),
        # a serving batch whose requests have settings of their own
        dict(_case("draw", dtype="f32", rows=64, vocab=VOCAB, width=WIDTH, temperature=1.0, top_k=0,
                   top_p=0.95, min_p=0.0, each=True), name="draw_batch"),
        # many samples of one model in 16 bits: many equal values
        dict(_case("draw", dtype="bf16", rows=512, vocab=VOCAB, width=VOCAB, temperature=0.7, top_k=0,
                   top_p=0.9, min_p=0.02, each=False), name="draw_many"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(("assign", "release", "shared", "shared", "shared", "draw", "draw", "draw"))
    page = rng.choice((16, 32, 64, 128, 256))
    if kind in ("assign", "release"):
        ctx = _log_int(rng, 1, 8192)
        seqs = _log_int(rng, 1, min(1000, max(1, (1 << 19) // ctx)))
        if kind == "release":
            return _case(kind, seqs=seqs, ctx=ctx, page=page, ends=round(rng.uniform(0.0, 1.0), 3))
        new = 1 if rng.random() < 0.4 else _log_int(rng, 1, ctx)
        new = max(1, min(new, 65536 // seqs))
        return _case(kind, seqs=seqs, new=new, ctx=ctx, page=page,
                     rows=max(1, int(seqs * new * rng.uniform(0.3, 1.1))),
                     full=round(rng.uniform(0.0, 1.0), 3))
    if kind == "shared":
        h, hk, d = rng.choice(HEADS)
        prefix, own_ = _log_int(rng, 1, 16384), _log_int(rng, 1, 1024)
        new = 1 if rng.random() < 0.6 else _log_int(rng, 1, min(own_, 300))
        groups = rng.choice((1, 1, 2, 5))
        # no more products than the largest listed, and no more entries
        most = (64 * 8448 * 12) // ((prefix + own_) * h * groups * new)
        seqs = _log_int(rng, 1, max(1, min(96, most)))
        return _case(kind, groups=groups, seqs=seqs, new=new, prefix=prefix, own=own_, heads=h,
                     kv_heads=hk, head_dim=d, page=page, window=rng.choice((0, 0, 0, WINDOW)))
    vocab = VOCAB if rng.random() < 0.5 else _log_int(rng, 2, 150000)
    rows = _log_int(rng, 1, max(1, min(512, 512 * VOCAB // vocab)))
    return _case(kind, dtype=rng.choice(("f32", "bf16")), rows=rows, vocab=vocab,
                 width=vocab + rng.choice((0, 0, 47, 8)),
                 temperature=rng.choice((0.0, 0.3, 0.8, 1.0, 1.5)),
                 top_k=rng.choice((0, 0, 1, 50, _log_int(rng, 1, vocab))),
                 top_p=rng.choice((1.0, 0.95, 0.8, round(rng.uniform(0.01, 1.0), 3))),
                 min_p=rng.choice((0.0, 0.0, 0.05, round(rng.uniform(0.0, 0.5), 3))),
                 each=rng.random() < 0.4)


def _host(case, *what):
    """Numbers of the case's own, so that every seed has the same amount of work."""
    return random.Random(" ".join(str(case.get(x)) for x in ("kind", "seqs", "ctx", "new", "prefix", "own"))
                         + str(what))


def _requests(case):
    """([entries], [new tokens]) of the sequences of a step."""
    rng = _host(case)
    lens, new = [], []
    for _ in range(case["seqs"]):
        n = case["new"]
        if n > 1:   # a third of the requests decode, the others bring a part of their prompt
            n = 1 if rng.random() < 0.33 else rng.randint(1, n)
        new.append(n)
        lens.append(rng.randint(0, case["ctx"] - n))
    return lens, new


def _left(case):
    """([entries], [entries that stay]) of sequences of which some end or are cut back."""
    rng = _host(case)
    lens = [rng.randint(case["ctx"] // 2, case["ctx"]) for _ in range(case["seqs"])]
    left = [c if rng.random() >= case["ends"] else 0 if rng.random() < 0.6 else rng.randint(0, c)
            for c in lens]
    return lens, left


def _lens(case):
    """([new tokens], [own entries with these]) of all groups' sequences."""
    rng = _host(case)
    new, mine = [], []
    for _ in range(case["groups"] * case["seqs"]):
        n = case["new"]
        if n > 8:
            n = 1 if rng.random() < 0.33 else rng.randint(1, n)
        new.append(n)
        mine.append(rng.randint(max(n, case["own"] // 2), max(n, case["own"])))
    return new, mine


# ---- inputs -------------------------------------------------------------------

def _gen(seed, stream):
    g = torch.Generator(device=DEV)
    g.manual_seed((int(seed) * 1000003 + stream) % (1 << 62))
    return g


def _normal(seed, stream, dtype, *shape):
    x = torch.empty(shape, device=DEV).normal_(0.0, 1.0, generator=_gen(seed, stream))
    return x.to(dtype)


def _uniform(seed, stream, *shape):
    return torch.rand(shape, device=DEV, generator=_gen(seed, stream))


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _unit(x):
    """Rows of mean square one, as the norms leave queries and keys."""
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)


def _pool_state(case, seed, lens):
    """A table whose sequences hold pages for their entries, in no order, in a
    pool with other pages in use, and each page's count.  A few of the first
    pages are shared."""
    S, page = case["seqs"], case["page"]
    cols = -(-case["ctx"] // page)
    pages = S * cols + 8
    order = torch.randperm(pages, device=DEV, generator=_gen(seed, 1)).to(torch.int32)
    have = (lens + page - 1) // page
    c = torch.arange(cols, device=DEV)
    held = c < have[:, None]
    table = torch.where(held, order[:S * cols].view(S, cols), -1).contiguous()
    pair = held[::2, 0][:S // 2] & held[1::2, 0]    # the first page of the next sequence too
    table[0:2 * (S // 2):2, 0] = torch.where(pair, table[1::2, 0], table[0:2 * (S // 2):2, 0])
    refs = torch.zeros(pages, dtype=torch.int32, device=DEV)
    ids = torch.where(table >= 0, table, 0).long().flatten()
    refs.index_add_(0, ids, (table >= 0).to(torch.int32).flatten())
    # pages that others hold
    other = (_uniform(seed, 2, pages) < case.get("full", 0.0)) & (refs == 0)
    return table, refs + other.to(torch.int32)


def _prepare_draw(case, seed):
    R, V, W = case["rows"], case["vocab"], case["width"]
    # a model's scores: a broad middle and a few tokens far above it, softcapped
    z = 2.0 * _normal(seed, 1, torch.float32, R, W)
    z += torch.where(_uniform(seed, 2, R, W) < 0.002, 6.0 * _uniform(seed, 3, R, W), 0.0)
    x = 23.0 * torch.sigmoid((z + 5.0) / 7.5)
    if V > 100:   # a few tokens that a request forbids
        x[:, 17:23] = float("-inf")
    x = x.to(torch.float32 if case["dtype"] == "f32" else torch.bfloat16)
    st = {"logits": x[:, :V], "u": _uniform(seed, 4, R)}
    for i, name in enumerate(("temperature", "top_k", "top_p", "min_p")):
        st[name] = case[name]
    if case["each"]:
        f = _uniform(seed, 5, 4, R)
        st["temperature"] = torch.where(f[0] < 0.2, 0.0, case["temperature"] * (0.5 + f[0])).contiguous()
        st["top_k"] = torch.where(f[1] < 0.5, case["top_k"], (1.0 + 60.0 * f[1]).to(torch.int32)).to(torch.int32)
        st["top_p"] = torch.where(f[2] < 0.3, 1.0, case["top_p"] * f[2]).contiguous()
        st["min_p"] = torch.where(f[3] < 0.6, case["min_p"], 0.1 * f[3]).contiguous()
    return st


def prepare(case, seed):
    kind = case["kind"]
    st = {"case": case}
    if kind == "draw":
        st.update(_prepare_draw(case, seed))
        return st
    if kind in ("assign", "release"):
        lens, other = _requests(case) if kind == "assign" else _left(case)
        st["lens"] = _i32(lens)
        st["table"], st["refs"] = _pool_state(case, seed, st["lens"])
        if kind == "assign":
            st["new"] = _i32(other)
        else:
            st["lens"] = _i32(other)
        return st
    new, mine = _lens(case)
    page, P, G = case["page"], case["prefix"], case["groups"]
    S = len(new)
    h, hk, d = case["heads"], case["kv_heads"], case["head_dim"]
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    common = P // page                        # pages that a group's sequences share
    lens = [P + m for m in mine]              # behind a prefix that ends inside a page its last
    cols = -(-max(lens) // page)              # entries lie in each sequence's own next page
    pages = G * (common + 1) + S * (cols - common) + 8
    order = torch.randperm(pages, device=DEV, generator=_gen(seed, 9)).to(torch.int32)
    first = order[:G * (common + 1)].view(G, common + 1)
    rest = order[G * (common + 1):G * (common + 1) + S * (cols - common)].view(S, cols - common)
    st["table"] = torch.cat((first[:, :common].repeat_interleave(S // G, 0), rest), 1).contiguous()
    st["prefix_table"] = first.contiguous()
    st["prefix_lens"] = _i32([P] * G)
    st["groups"] = _i32([g * (S // G) for g in range(G + 1)])
    st["starts"], st["lens"], st["max_len"], st["max_new"] = _i32(starts), _i32(lens), max(lens), max(new)
    shape = (pages, hk, page, d)
    k = _unit(torch.empty(shape, device=DEV).normal_(0.0, 1.0, generator=_gen(seed, 7))).to(torch.bfloat16)
    v = _normal(seed, 8, torch.bfloat16, *shape)
    if P % page:
        for x in (k, v):
            x[rest[:, 0].long(), :, :P % page] = x[first[:, common].long()].repeat_interleave(S // G, 0)[:, :, :P % page]
    st["k_cache"], st["v_cache"] = k, v
    st["q"] = _unit(_normal(seed, 1, torch.float32, starts[-1], h, d)).to(torch.bfloat16)
    return st


# ---- one pass: plain forms ------------------------------------------------------

def _plain_assign(st, page, rows):
    table, refs = st["table"], st["refs"]
    S, cols = table.shape
    pages = refs.shape[0]
    at, n = st["lens"].long().clamp(0, cols * page), st["new"].long().clamp(min=0)
    fit = at + n <= cols * page
    c = torch.arange(cols, device=DEV)
    touched = (c >= (at // page)[:, None]) & (c < ((at + n + page - 1) // page)[:, None])
    touched = touched & (fit & (n > 0))[:, None]
    missing = touched & ((table < 0) | (table >= pages))
    need = missing.sum(1)
    free = refs <= 0
    ok = fit & ((n * fit).cumsum(0) <= rows) & ((need == 0) | (need.cumsum(0) <= free.sum()))
    n = n * ok
    starts = torch.zeros(S + 1, dtype=torch.int32, device=DEV)
    starts[1:] = n.cumsum(0)
    # the i-th missing column takes the i-th free page
    take = missing & ok[:, None]
    rank = (take.flatten().cumsum(0) - 1).view(S, cols)
    place = free.cumsum(0) - 1
    ids = torch.zeros(pages + 1, dtype=torch.int32, device=DEV)
    ids[torch.where(free, place, pages)] = torch.arange(pages, dtype=torch.int32, device=DEV)
    table = torch.where(take, ids[rank.clamp(0, pages)], table)
    refs = torch.where(free & (place < take.sum()), 1, refs)
    r = torch.arange(rows, device=DEV)
    seq = torch.searchsorted(starts[1:].long(), r, right=True)
    real = seq < S
    s = seq.clamp(max=S - 1)
    pos = at[s] + r - starts[s]
    col = torch.where(real, pos, 0) // page
    slot = table[s, col].long() * page + pos % page
    return {"table": table, "refs": refs, "starts": starts, "lens": (at + n).to(torch.int32),
            "seq": torch.where(real, s, -1).to(torch.int32),
            "pos": torch.where(real, pos, -1).to(torch.int32), "slot": torch.where(real, slot, -1)}


def _plain_release(st, page):
    table, refs = st["table"], st["refs"]
    S, cols = table.shape
    have = (st["lens"].long().clamp(0, cols * page) + page - 1) // page
    gone = torch.arange(cols, device=DEV) >= have[:, None]
    named = gone & (table >= 0) & (table < refs.shape[0])
    refs = refs.index_add(0, torch.where(named, table, 0).long().flatten(),
                          -named.to(torch.int32).flatten())
    return {"table": torch.where(gone, -1, table), "refs": refs}


def _entries(cache, table, most):
    """The first `most` entries of each sequence in 32 bits: (S, Hkv, most, D)."""
    x = cache[table.long()].permute(0, 2, 1, 3, 4)
    return x.reshape(x.shape[0], x.shape[1], -1, x.shape[4])[:, :, :most].float()


def _tokens(st):
    """(sequence, place in its new tokens, cache entry) of each row."""
    starts, lens = st["starts"].long(), st["lens"].long()
    rows = torch.arange(st["q"].shape[0], device=DEV)
    seq = torch.searchsorted(starts, rows, right=True) - 1
    at = rows - starts[seq]
    return seq, at, lens[seq] - (starts[seq + 1] - starts[seq]) + at


def _plain_shared(st, window):
    """The prefix once for all rows of a group, each sequence's own entries behind
    it, and the two joined."""
    q, H = st["q"].float(), st["q"].shape[1]
    Hk, D = st["k_cache"].shape[1], st["q"].shape[2]
    P = st["case"]["prefix"]
    seq, at, entry = _tokens(st)
    N, n_groups = q.shape[0], st["groups"].shape[0] - 1
    group = torch.searchsorted(st["groups"].long(), seq, right=True) - 1
    x = q.view(N, Hk, H // Hk, D)
    # scores against every group's prefix, the others' masked
    most = st["case"]["seqs"] * st["max_new"]
    first = st["starts"].long()[st["groups"].long()]
    t = torch.arange(most, device=DEV)
    rows = (first[:-1, None] + t).clamp(max=N - 1)
    xg = x[rows].permute(0, 2, 3, 1, 4).reshape(n_groups, Hk, -1, D)
    kp, vp = (_entries(st[c], st["prefix_table"], P) for c in ("k_cache", "v_cache"))
    j = torch.arange(P, device=DEV)
    eg = entry[rows][:, None, None, :, None]
    sees = j <= eg
    if window:
        sees = sees & (eg - j < window)
    s = torch.matmul(xg, kp.transpose(2, 3).contiguous()).view(n_groups, Hk, H // Hk, most, P) * SCALE
    s = torch.where(sees, s, float("-inf"))
    m1 = s.amax(-1, keepdim=True).clamp_min(-3e38)
    e = torch.exp(s - m1)
    l1 = e.sum(-1, keepdim=True)
    o1 = torch.matmul(e.view(n_groups, Hk, -1, P), vp).view(n_groups, Hk, H // Hk, most, D)
    place = torch.arange(N, device=DEV) - first[group]
    m1, l1, o1 = (y[group, :, :, place] for y in (m1, l1, o1))
    # and against each sequence's own entries
    S, T, C = st["lens"].shape[0], st["max_new"], st["max_len"] - P
    tt = torch.arange(T, device=DEV)
    rows = (st["starts"].long()[:-1, None] + tt).clamp(max=N - 1)
    new = (st["starts"][1:] - st["starts"][:-1]).long()[:, None]
    xs = x[rows].permute(0, 2, 3, 1, 4).reshape(S, Hk, -1, D)
    ko, vo = (_entries(st[c], st["table"], st["max_len"])[:, :, P:].contiguous()
              for c in ("k_cache", "v_cache"))
    j = P + torch.arange(C, device=DEV)
    es = (st["lens"].long()[:, None] - new + tt)[:, None, None, :, None]
    sees = j <= es
    if window:
        sees = sees & (es - j < window)
    s = torch.matmul(xs, ko.transpose(2, 3).contiguous()).view(S, Hk, H // Hk, T, C) * SCALE
    s = torch.where(sees, s, float("-inf"))
    m2 = s.amax(-1, keepdim=True).clamp_min(-3e38)
    e = torch.exp(s - m2)
    l2 = e.sum(-1, keepdim=True)
    o2 = torch.matmul(e.view(S, Hk, -1, C), vo).view(S, Hk, H // Hk, T, D)
    m2, l2, o2 = (y[seq, :, :, at] for y in (m2, l2, o2))
    m = torch.maximum(m1, m2)
    f1, f2 = torch.exp(m1 - m), torch.exp(m2 - m)
    total = l1 * f1 + l2 * f2
    out = (o1 * f1 + o2 * f2) / total
    return {"out": out.flatten(1, 2).to(torch.bfloat16),
            "lse": (m + torch.log(total))[..., 0].flatten(1, 2)}


def _column(value, rows, dtype):
    if isinstance(value, torch.Tensor):
        return value.to(dtype)[:, None]
    return torch.full((rows, 1), value, dtype=dtype, device=DEV)


def _plain_draw(st):
    x = st["logits"].double()      # 64 bits: a draw may fall next to a border
    R, V = x.shape
    x = torch.where(torch.isnan(x), float("-inf"), x)
    # the settings as the 32-bit numbers that a call takes
    T, P, M = (_column(st[n], R, torch.float32).double() for n in ("temperature", "top_p", "min_p"))
    k = _column(st["top_k"], R, torch.int64)
    u = st["u"].double()[:, None]
    top = x.amax(1, keepdim=True)
    greedy = ~(T > 0)
    w = torch.exp((x - top) / torch.where(greedy, 1.0, T))
    w = torch.where(x == top, 1.0, torch.where(x == float("-inf"), 0.0, w))
    w = torch.where(greedy & (x < top), 0.0, w)
    w = torch.where(w >= M.clamp(LEAST, 1.0), w, 0.0)
    order = torch.argsort(x, dim=1, descending=True, stable=True)
    sx, sw = x.gather(1, order), w.gather(1, order)
    kth = sx.gather(1, torch.where((k > 0) & (k < V), k - 1, V - 1))
    sw = torch.where(sx >= kth, sw, 0.0)
    cum = sw.cumsum(1)
    enough = (cum < P.clamp(0.0, 1.0) * cum[:, -1:]).sum(1, keepdim=True).clamp(max=V - 1)
    least = torch.where(P < 1.0, torch.maximum(kth, sx.gather(1, enough)), kth)
    w = torch.where(x >= least, w, 0.0)
    cum = w.cumsum(1)
    total = cum[:, -1:]
    idx = torch.arange(V, device=DEV)
    last = torch.where(w > 0.0, idx, -1).amax(1, keepdim=True)
    pick = torch.minimum((cum <= u * total).sum(1, keepdim=True), last)
    first = torch.where(w > 0.0, idx, V).amin(1, keepdim=True)
    pick = torch.where(greedy, first, pick)
    logprob = torch.where(greedy, 0.0, torch.log(w.gather(1, pick) / total))
    return {"ids": pick[:, 0].to(torch.int32), "logprob": logprob[:, 0].float()}


def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        from attention_nn_amd import kernels, paged
    if kind == "assign":
        if not own:
            return _plain_assign(state, case["page"], case["rows"])
        a = paged.assign(state["table"], state["lens"], state["new"], state["refs"], case["page"],
                         case["rows"])
        return {"table": a.table, "refs": a.refs, "starts": a.starts, "lens": a.lens, "seq": a.seq,
                "pos": a.pos, "slot": a.slot}
    if kind == "release":
        if not own:
            return _plain_release(state, case["page"])
        table, refs = paged.release(state["table"], state["lens"], state["refs"], case["page"])
        return {"table": table, "refs": refs}
    if kind == "shared":
        if not own:
            return _plain_shared(state, case["window"])
        out, lse = paged.attention_shared(
            state["q"], state["k_cache"], state["v_cache"], state["table"], state["starts"],
            state["lens"], state["groups"], state["prefix_table"], state["prefix_lens"], SCALE,
            window=case["window"], want_lse=True)
        return {"out": out, "lse": lse}
    if not own:
        return _plain_draw(state)
    ids, logprob = kernels.sample_logits(state["logits"], state["u"], state["temperature"],
                                         state["top_k"], state["top_p"], state["min_p"],
                                         want_logprob=True)
    return {"ids": ids, "logprob": logprob}


# ---- what a pass cannot do without ----------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "draw":
        size = 4 if case["dtype"] == "f32" else 2
        n = case["rows"] * case["vocab"]
        # a comparison, a difference and an exponential for each entry
        return {"bytes": float(n * size + case["rows"] * (4 + 8 + (16 if case["each"] else 0))),
                "flops": 3.0 * n}
    if kind in ("assign", "release"):
        S, cols = case["seqs"], -(-case["ctx"] // case["page"])
        both = 2 * 4 * (S * cols + S * cols + 8)      # the table and the pages' counts, in and out
        if kind == "release":
            return {"bytes": float(both + 4 * S), "flops": float(S * cols)}
        return {"bytes": float(both + 8 * S + 8 * S + 16 * case["rows"]), "flops": float(S * cols)}
    new, mine = _lens(case)
    h, hk, d, P, w = case["heads"], case["kv_heads"], case["head_dim"], case["prefix"], case["window"]
    pairs, entries, seen = 0, 0, 0
    for n, m in zip(new, mine):
        c = P + m
        if w:
            pairs += sum(min(w, i + 1) for i in range(c - n, c))
            entries += min(m, n + w - 1)
            seen = max(seen, P - max(0, c - n - w + 1))
        else:
            pairs += n * c - n * (n - 1) // 2
            entries += m
            seen = P
    N, S = sum(new), len(new)
    entries += case["groups"] * max(seen, 0)
    pages = 4 * (case["groups"] * -(-P // case["page"]) + sum(-(-m // case["page"]) for m in mine))
    return {"bytes": float(2 * entries * hk * d * 2 + N * h * (2 * d * 2 + 4) + pages + 12 * S),
            "flops": 4.0 * pairs * h * d}


# ---- the same from the definition -------------------------------------------------

def _assign_host(st, page, rows):
    """Request by request, with lists."""
    table, refs = st["table"].cpu().tolist(), st["refs"].cpu().tolist()
    cap = len(table[0]) * page
    free = [i for i, r in enumerate(refs) if r <= 0]
    want_rows = want_pages = taken = 0
    starts, lens, seq, pos, slot = [0], [], [], [], []
    for s, (c, n) in enumerate(zip(st["lens"].tolist(), st["new"].tolist())):
        got = 0
        if c + n <= cap:
            cols = [x for x in range(c // page, -(-(c + n) // page)) if not 0 <= table[s][x] < len(refs)]
            want_rows += n
            want_pages += len(cols)
            if want_rows <= rows and (not cols or want_pages <= len(free)):
                got = n
                for x in cols:
                    table[s][x] = free[taken]
                    refs[free[taken]] = 1
                    taken += 1
        for e in range(c, c + got):
            seq.append(s)
            pos.append(e)
            slot.append(table[s][e // page] * page + e % page)
        starts.append(starts[-1] + got)
        lens.append(c + got)
    behind = [-1] * (rows - len(seq))
    i32 = {"table": table, "refs": refs, "starts": starts, "lens": lens, "seq": seq + behind,
           "pos": pos + behind}
    out = {n: torch.tensor(v, dtype=torch.int32) for n, v in i32.items()}
    out["slot"] = torch.tensor(slot + behind, dtype=torch.int64)
    return out


def _release_host(st, page):
    table, refs = st["table"].cpu().tolist(), st["refs"].cpu().tolist()
    for row, c in zip(table, st["lens"].tolist()):
        for x in range(-(-c // page), len(row)):
            if 0 <= row[x] < len(refs):
                refs[row[x]] -= 1
            row[x] = -1
    return {"table": torch.tensor(table, dtype=torch.int32), "refs": torch.tensor(refs, dtype=torch.int32)}


def _attention64(st, case):
    """Sequence by sequence over its whole table and head by head, in 64 bits."""
    new, mine = _lens(case)
    H, Hk, page = st["q"].shape[1], st["k_cache"].shape[1], case["page"]
    out, lse, at = [], [], 0
    for s, (n, m) in enumerate(zip(new, mine)):
        c = case["prefix"] + m
        k, v = (torch.cat(st[x][st["table"][s, :-(-c // page)].long()].unbind(0), dim=1)[:, :c].double()
                for x in ("k_cache", "v_cache"))
        i = torch.arange(c - n, c, device=DEV)[:, None]
        j = torch.arange(c, device=DEV)[None, :]
        hidden = (j > i) | (i - j >= case["window"]) if case["window"] else j > i
        o, l = [], []
        for g in range(H):
            kh = g * Hk // H
            x = st["q"][at:at + n, g].double() @ k[kh].t().contiguous() * SCALE
            x = x.masked_fill(hidden, float("-inf"))
            o.append(torch.softmax(x, -1) @ v[kh])
            l.append(torch.logsumexp(x, -1))
        out.append(torch.stack(o, 1))
        lse.append(torch.stack(l, 1))
        at += n
    return {"out": torch.cat(out), "lse": torch.cat(lse)}


def _draw_host(st):
    """Row by row on the host: sorted values, sums in extended precision."""
    x = st["logits"].float().cpu().numpy()
    R, V = x.shape

    def column(name):
        v = st[name]
        return v.cpu().numpy() if isinstance(v, torch.Tensor) else [np.float32(v)] * R

    ids, logprob = [], []
    rows = zip(x, st["u"].cpu().numpy(), column("temperature"), column("top_k"), column("top_p"),
               column("min_p"))
    for row, u, t, k, p, least in rows:
        top = row.max()
        if not t > 0:
            ids.append(int(np.flatnonzero(row == top)[0]))
            logprob.append(0.0)
            continue
        # candidates in the order of their indices
        i = np.flatnonzero(row > -np.inf)
        with np.errstate(under="ignore"):
            w = np.exp((row[i].astype(np.float64) - float(top)) / float(t)).astype(np.longdouble)
        some = w >= max(min(float(least), 1.0), LEAST)
        i, w = i[some], w[some]
        if 0 < k < V:
            kth = np.partition(row, V - int(k))[V - int(k)]
            some = row[i] >= kth
            i, w = i[some], w[some]
        if p < 1.0:
            by = np.argsort(-row[i].astype(np.float64), kind="stable")
            run_ = np.cumsum(w[by])
            least_x = row[i[by[min(int((run_ < max(float(p), 0.0) * run_[-1]).sum()), len(by) - 1)]]]
            some = row[i] >= least_x
            i, w = i[some], w[some]
        run_ = np.cumsum(w)
        at = min(int((run_ <= np.longdouble(u) * run_[-1]).sum()), len(i) - 1)
        ids.append(int(i[at]))
        logprob.append(float(np.log(w[at] / run_[-1])))
    return {"ids": torch.tensor(ids, dtype=torch.int32),
            "logprob": torch.tensor(logprob, dtype=torch.float64)}


def exact(case, seed):
    st, kind = prepare(case, seed), case["kind"]
    if kind == "assign":
        return _assign_host(st, case["page"], case["rows"])
    if kind == "release":
        return _release_host(st, case["page"])
    if kind == "shared":
        return _attention64(st, case)
    return _draw_host(st)
