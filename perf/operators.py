"""Serving a paged key/value cache, and the rows that enter it, as cases that
can be timed and checked: the norms and rotation of queries and keys (with
their gradient), the append to the cache, the attention of new tokens over it,
the attention weight that its entries receive and the eviction that goes by it.

    listed()        the named cases
    draw(rng)       one more case of the same ranges
    prepare(c, s)   what a program holds before the call, made from seed s
    run(state)      one pass; returns its outputs
    work(c)         bytes and operations that a pass cannot do without
    exact(c, s)     the same outputs in 64 bits by plain torch

A cache is two tensors (pages, kv_heads, page, head_dim) in bf16; row s of a
table holds the pages of sequence s in order.  New tokens of all sequences lie
behind one another: those of sequence s are rows starts[s] .. starts[s + 1] - 1,
and lens[s] counts its cache entries with these.  Head layouts are those of the
155M shape (6 x 128), the command line's default (8 x 64), the wide shape (12 x
128) and two with shared key/value heads.
"""

import math
import random

import torch

own = False

DEV = "cuda"
EPS = 1e-6
SCALE = 0.1             # the framework's attention scale
WINDOW = 384            # and its sliding window

# (query heads, key/value heads, head_dim)
HEADS = ((6, 6, 128), (8, 8, 64), (12, 12, 128), (8, 2, 128), (12, 3, 64))


# ---- the cases ----------------------------------------------------------------

def _case(kind, **kw):
    return {"kind": kind, **kw}


def listed():
    return [
        # queries and keys of a training batch, read from the fused projection
        dict(_case("norm_rope", dtype="bf16", batch=64, length=512, heads=6, kv_heads=6,
                   head_dim=128, fused=True), name="norm_rope_batch"),
        # their gradient at an odd length, in 32 bits
        dict(_case("norm_rope_bwd", dtype="f32", batch=16, length=1023, heads=8, kv_heads=8,
                   head_dim=64, fused=False), name="norm_rope_bwd_odd"),
        # one decode step of a serving batch enters the cache
        dict(_case("append", seqs=64, new=1, ctx=1024, ragged=True, heads=6, kv_heads=6,
                   head_dim=128, page=16), name="append_decode"),
        # prompt chunks of several requests enter it
        dict(_case("append", seqs=12, new=1024, ctx=4096, ragged=True, heads=12, kv_heads=12,
                   head_dim=128, page=64), name="append_chunks"),
        # interactive generation: one token of one sequence
        dict(_case("attention", seqs=1, new=1, ctx=777, ragged=False, heads=6, kv_heads=6,
                   head_dim=128, page=16, window=0), name="attend_one"),
        # a decode step over long contexts
        dict(_case("attention", seqs=16, new=1, ctx=8192, ragged=True, heads=6, kv_heads=6,
                   head_dim=128, page=32, window=0), name="attend_decode_long"),
        # ragged prompt chunks beside decoding requests on a windowed layer
        dict(_case("attention", seqs=24, new=517, ctx=2048, ragged=True, heads=6, kv_heads=6,
                   head_dim=128, page=16, window=WINDOW), name="attend_mixed_window"),
        # a long chunk against a long context on a full-causal layer
        dict(_case("attention", seqs=1, new=2048, ctx=16384, ragged=False, heads=12, kv_heads=12,
                   head_dim=128, page=64, window=0), name="attend_chunk_long"),
        # the weight that a decode step gives each entry
        dict(_case("weight", seqs=16, new=1, ctx=4096, ragged=True, heads=6, kv_heads=6,
                   head_dim=128, page=32), name="weight_decode"),
        # and that a prompt chunk gives them
        dict(_case("weight", seqs=4, new=512, ctx=4096, ragged=True, heads=8, kv_heads=8,
                   head_dim=64, page=64), name="weight_chunk"),
        # one conversation cut back
        dict(_case("evict", seqs=1, ctx=1500, ragged=False, keep=1024, recent=256, heads=6,
                   kv_heads=6, head_dim=128, page=16), name="evict_one"),
        # a batch of long ones
        dict(_case("evict", seqs=16, ctx=8192, ragged=True, keep=4096, recent=384, heads=6,
                   kv_heads=6, head_dim=128, page=32), name="evict_batch"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(("norm_rope", "norm_rope_bwd", "append", "attention", "attention",
                       "attention", "weight", "evict"))
    h, hk, d = rng.choice(HEADS)
    if kind in ("norm_rope", "norm_rope_bwd"):
        if rng.random() < 0.25:
            h, hk, d = rng.choice(((3, 3, 36), (4, 2, 96), (5, 1, 20)))
        length = _log_int(rng, 1, 2048)
        return _case(kind, dtype=rng.choice(("f32", "bf16")),
                     batch=_log_int(rng, 1, max(1, 16384 // length)), length=length, heads=h,
                     kv_heads=hk, head_dim=d, fused=rng.random() < 0.5)
    page = rng.choice((16, 32, 64, 128, 256))
    if kind == "evict":
        ctx = _log_int(rng, 2, 16384)
        keep = _log_int(rng, 1, ctx)
        return _case(kind, seqs=_log_int(rng, 1, max(1, min(64, 131072 // ctx))), ctx=ctx,
                     ragged=rng.random() < 0.7, keep=keep, recent=rng.randrange(0, keep + 1),
                     heads=h, kv_heads=hk, head_dim=d, page=page)
    new = 1 if rng.random() < 0.4 else _log_int(rng, 1, 1024)
    ctx = _log_int(rng, new, 16384)
    most = 131072 if kind == "append" else 65536
    seqs = _log_int(rng, 1, max(1, min(128, most // ctx, 8192 // new)))
    # at most a third of the longest chunk's products
    seqs = max(1, min(seqs, (1 << 27) // max(1, new * ctx * h // 8)))
    case = _case(kind, seqs=seqs, new=new, ctx=ctx, ragged=rng.random() < 0.7, heads=h, kv_heads=hk,
                 head_dim=d, page=page)
    if kind == "attention":
        case["window"] = rng.choice((0, 0, WINDOW, 100))
    return case


def _lens(case):
    """([new tokens], [cache entries with them]) of the sequences: the case's
    own, so that every seed has the same amount of work."""
    rng = random.Random("%s %d %d %d" % (case["kind"], case["seqs"], case.get("new", 0), case["ctx"]))
    new, lens = [], []
    for s in range(case["seqs"]):
        n = case.get("new", 0)
        if case["ragged"] and n > 1:
            # a third of the requests decode, the others bring a part of their prompt
            n = 1 if rng.random() < 0.33 else rng.randint(1, n)
        c = case["ctx"] if not case["ragged"] else rng.randint(max(n, case["ctx"] // 2), case["ctx"])
        new.append(n)
        lens.append(max(n, c))
    return new, lens


# ---- inputs -------------------------------------------------------------------

def _gen(seed, stream):
    g = torch.Generator(device=DEV)
    g.manual_seed((int(seed) * 1000003 + stream) % (1 << 62))
    return g


def _normal(seed, stream, dtype, *shape):
    x = torch.empty(shape, device=DEV).normal_(0.0, 1.0, generator=_gen(seed, stream))
    return x.to(dtype)


def _unit(x):
    """Rows of mean square one, as the norms leave queries and keys."""
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)


def _rope_tables(length, head_dim):
    d4 = head_dim // 4
    freq = (1.0 / 1024.0) ** torch.linspace(0.0, 1.0, d4, device=DEV, dtype=torch.float64)
    theta = torch.arange(length, device=DEV, dtype=torch.float64)[:, None] * freq[None, :]
    return torch.cos(theta).float(), torch.sin(theta).float()


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _qkv(case, seed, dtype, *lead):
    """q, k, v of each token: views of one fused projection, or tensors of their own."""
    h, hk, d = case["heads"], case["kv_heads"], case["head_dim"]
    if case.get("fused", True):
        x = _normal(seed, 1, dtype, *lead, h + 2 * hk, d)
        return x[..., :h, :], x[..., h:h + hk, :], x[..., h + hk:, :]
    return tuple(_normal(seed, 1 + i, dtype, *lead, n, d) for i, n in enumerate((h, hk, hk)))


def _cache(case, seed, lens, spare=0):
    """A pool of pages in use, in no order, with as many others again; `spare`
    more pages for each sequence in a table of their own."""
    page, S = case["page"], case["seqs"]
    cols = -(-max(lens) // page)
    pages = S * (cols + spare) + 8
    order = torch.randperm(pages, device=DEV, generator=_gen(seed, 9)).to(torch.int32)
    shape = (pages, case["kv_heads"], page, case["head_dim"])
    k = torch.empty(shape, device=DEV).normal_(0.0, 1.0, generator=_gen(seed, 7))
    k = _unit(k).to(torch.bfloat16)
    v = _normal(seed, 8, torch.bfloat16, *shape)
    table = order[:S * cols].view(S, cols).contiguous()
    more = order[S * cols:S * (cols + spare)].view(S, spare).contiguous()
    return k, v, table, more


def prepare(case, seed):
    kind, h, d = case["kind"], case["heads"], case["head_dim"]
    st = {"case": case}
    if kind in ("norm_rope", "norm_rope_bwd"):
        dt = torch.float32 if case["dtype"] == "f32" else torch.bfloat16
        B, T = case["batch"], case["length"]
        st["q"], st["k"], _ = _qkv(case, seed, dt, B, T)
        st["cs"], st["sn"] = _rope_tables(T, d)
        if kind == "norm_rope_bwd":
            st["gq"] = _normal(seed, 5, dt, B, T, h, d)
            st["gk"] = _normal(seed, 6, dt, B, T, case["kv_heads"], d)
        return st
    new, lens = _lens(case)
    st["lens"] = _i32(lens)
    st["max_len"], st["max_new"] = max(lens), max(new)
    if kind == "evict":
        cols = -(-case["keep"] // case["page"])
        st["k_cache"], st["v_cache"], st["table"], st["out_table"] = _cache(case, seed, lens, cols)
        cap = st["table"].shape[1] * case["page"]
        # weights as attention leaves them: positive, a few entries far above
        # the rest, and many equal ones among the small
        w = torch.exp(2.0 * _normal(seed, 5, torch.float32, case["seqs"], cap))
        st["weight"] = torch.where(w < 0.5, torch.floor(w * 64.0) / 64.0, w)
        return st
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    st["starts"] = _i32(starts)
    N = starts[-1]
    st["k_cache"], st["v_cache"], st["table"], _ = _cache(case, seed, lens)
    if kind == "append":
        st["q"], st["k"], st["v"] = _qkv(case, seed, torch.bfloat16, N)
        st["cs"], st["sn"] = _rope_tables(case["ctx"], d)
        return st
    st["q"] = _unit(_normal(seed, 1, torch.float32, N, h, d)).to(torch.bfloat16)
    if kind == "weight":
        # the log of each query's softmax sum, as the attention call returns it
        st["lse"] = _attention64(st, 0)[1].float()
        cap = st["table"].shape[1] * case["page"]
        st["weight"] = torch.exp(_normal(seed, 5, torch.float32, case["seqs"], cap))
    return st


# ---- one pass: plain forms ------------------------------------------------------

def _plain_norm_rope(x, cs, sn):
    """x (..., H, D) in 32 bits; cs, sn broadcast against (..., 1, D / 4)."""
    n = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    half = x.shape[-1] // 2
    a, b = n[..., 0:half:2], n[..., 1:half:2]
    turned = torch.stack((cs * a + sn * b, cs * b - sn * a), -1).flatten(-2)
    return torch.cat((turned, n[..., half:]), -1)


def _plain_norm_rope_bwd(g, x, cs, sn):
    half = x.shape[-1] // 2
    a, b = g[..., 0:half:2], g[..., 1:half:2]
    back = torch.stack((cs * a - sn * b, cs * b + sn * a), -1).flatten(-2)
    g = torch.cat((back, g[..., half:]), -1)
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    return r * (g - x * (r * r * (x * g).mean(-1, keepdim=True)))


def _tokens(st):
    """(sequence, place in its new tokens, cache entry) of each row."""
    starts, lens = st["starts"].long(), st["lens"].long()
    rows = torch.arange(st["q"].shape[0], device=DEV)
    seq = torch.searchsorted(starts, rows, right=True) - 1
    at = rows - starts[seq]
    return seq, at, lens[seq] - (starts[seq + 1] - starts[seq]) + at


def _plain_append(st):
    page = st["k_cache"].shape[2]
    seq, _, entry = _tokens(st)
    cs, sn = st["cs"][entry][:, None, :], st["sn"][entry][:, None, :]
    q = _plain_norm_rope(st["q"].float(), cs, sn).to(torch.bfloat16)
    k = _plain_norm_rope(st["k"].float(), cs, sn).to(torch.bfloat16)
    where = st["table"][seq, entry // page].long()
    st["k_cache"][where, :, entry % page] = k
    st["v_cache"][where, :, entry % page] = st["v"]
    return {"q": q, "k_cache": st["k_cache"], "v_cache": st["v_cache"]}


def _entries(cache, table, most):
    """The first `most` entries of each sequence in 32 bits: (S, Hkv, most, D)."""
    x = cache[table.long()].permute(0, 2, 1, 3, 4)
    return x.reshape(x.shape[0], x.shape[1], -1, x.shape[4])[:, :, :most].float()


def _scores(st, window):
    """Scaled scores (S, Hkv, G * new, entries) of the new tokens, minus infinity
    where a token does not see an entry."""
    S, Hk, D, T = st["lens"].shape[0], st["k_cache"].shape[1], st["q"].shape[2], st["max_new"]
    G = st["q"].shape[1] // Hk
    starts, lens = st["starts"].long(), st["lens"].long()
    t = torch.arange(T, device=DEV)
    rows = (starts[:-1, None] + t).clamp(max=st["q"].shape[0] - 1)
    new = (starts[1:] - starts[:-1])[:, None]
    q = st["q"][rows].float().view(S, T, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(S, Hk, G * T, D)
    keys = _entries(st["k_cache"], st["table"], st["max_len"])
    s = torch.matmul(q, keys.transpose(2, 3).contiguous()) * SCALE
    entry = (lens[:, None] - new + t)[:, None, None, :, None]
    j = torch.arange(st["max_len"], device=DEV)
    sees = (j <= entry) & (t < new)[:, None, None, :, None]
    if window:
        sees = sees & (entry - j < window)
    s = s.view(S, Hk, G, T, -1)
    return torch.where(sees, s, float("-inf"))


def _plain_attention(st, window):
    s = _scores(st, window)
    S, Hk, G, T, C = s.shape
    m = s.amax(-1, keepdim=True).clamp_min(-3e38)
    e = torch.exp(s - m)
    total = e.sum(-1, keepdim=True)
    v = _entries(st["v_cache"], st["table"], st["max_len"])
    o = torch.matmul((e / total).view(S, Hk, G * T, C), v).view(S, Hk, G, T, -1)
    seq, at, _ = _tokens(st)
    out = o[seq, :, :, at].flatten(1, 2).to(torch.bfloat16)
    lse = (m + torch.log(total))[..., 0][seq, :, :, at].flatten(1, 2)
    return {"out": out, "lse": lse}


def _plain_weight(st):
    s = _scores(st, 0)
    S, Hk, G, T, C = s.shape
    starts = st["starts"].long()
    rows = (starts[:-1, None] + torch.arange(T, device=DEV)).clamp(max=st["q"].shape[0] - 1)
    lse = st["lse"][rows].view(S, T, Hk, G).permute(0, 2, 3, 1)
    got = torch.exp(s - lse[..., None]).sum((1, 2, 3))
    out = st["weight"].clone()
    out[:, :C] += torch.where(torch.arange(C, device=DEV) < st["lens"][:, None], got, 0.0)
    return out


def _plain_evict(st, keep, recent):
    k, v, w, lens = st["k_cache"], st["v_cache"], st["weight"], st["lens"].long()[:, None]
    page, cap = k.shape[2], w.shape[1]
    j = torch.arange(cap, device=DEV)
    # the last `recent` entries first, then by weight, the lower entry at a tie
    key = torch.where(j < lens, w, -1.0)
    key = torch.where((j < lens) & (j >= lens - recent), float("inf"), key)
    order = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :keep]
    if order.shape[1] < keep:
        order = torch.nn.functional.pad(order, (0, keep - order.shape[1]), value=cap)
    left = lens.clamp(max=keep)
    i = torch.arange(keep, device=DEV)
    order = torch.where(i < left, order, cap).sort(1).values
    src = torch.where(i < left, order, 0)
    dst = torch.where(i < left, i, 0)            # those behind the end repeat entry 0
    src = torch.where(i < left, src, order[:, :1])
    s = torch.arange(w.shape[0], device=DEV)[:, None]
    a, b = st["table"][s, src // page].long(), st["out_table"][s, dst // page].long()
    k[b, :, dst % page] = k[a, :, src % page]
    v[b, :, dst % page] = v[a, :, src % page]
    out = torch.zeros_like(w)
    out[:, :keep] = torch.where(i < left, w.gather(1, src), 0.0)[:, :cap]
    return {"index": torch.where(i < left, order, -1).to(torch.int32),
            "lens": left[:, 0].to(torch.int32), "weight": out, "k_cache": k, "v_cache": v}


def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        from attention_nn_amd import kernels, paged
    if kind == "norm_rope":
        if own:
            q, k = kernels.qk_norm_rope(state["q"], state["k"], state["cs"], state["sn"])
            return {"q": q, "k": k}
        cs, sn = state["cs"][:, None, :], state["sn"][:, None, :]
        return {n: _plain_norm_rope(state[n].float(), cs, sn).to(state[n].dtype) for n in "qk"}
    if kind == "norm_rope_bwd":
        if own:
            q, k = kernels.qk_norm_rope_bwd(state["gq"], state["gk"], state["q"], state["k"],
                                            state["cs"], state["sn"])
            return {"q": q, "k": k}
        cs, sn = state["cs"][:, None, :], state["sn"][:, None, :]
        return {n: _plain_norm_rope_bwd(state["g" + n].float(), state[n].float(), cs, sn)
                .to(state[n].dtype) for n in "qk"}
    if kind == "append":
        if not own:
            return _plain_append(state)
        q = paged.append(state["q"], state["k"], state["v"], state["cs"], state["sn"],
                         state["k_cache"], state["v_cache"], state["table"], state["starts"],
                         state["lens"])
        return {"q": q, "k_cache": state["k_cache"], "v_cache": state["v_cache"]}
    if kind == "attention":
        if not own:
            return _plain_attention(state, case["window"])
        out, lse = paged.attention(state["q"], state["k_cache"], state["v_cache"], state["table"],
                                   state["starts"], state["lens"], SCALE, window=case["window"],
                                   want_lse=True)
        return {"out": out, "lse": lse}
    if kind == "weight":
        if not own:
            return _plain_weight(state)
        return paged.attention_weight(state["q"], state["lse"], state["k_cache"], state["table"],
                                      state["starts"], state["lens"], state["weight"], SCALE)
    if not own:
        return _plain_evict(state, case["keep"], case["recent"])
    index, lens, weight = paged.evict(state["k_cache"], state["v_cache"], state["table"],
                                      state["lens"], state["weight"], case["keep"],
                                      recent=case["recent"], out_table=state["out_table"])
    return {"index": index, "lens": lens, "weight": weight, "k_cache": state["k_cache"],
            "v_cache": state["v_cache"]}


# ---- what a pass cannot do without ----------------------------------------------

def _seen(n, c, window):
    """(pairs of a new token and an entry it sees, entries that any of them sees)."""
    if not window:
        return n * c - n * (n - 1) // 2, c
    pairs = sum(min(window, i + 1) for i in range(c - n, c))
    return pairs, min(c, n + window - 1)


def work(case):
    kind, h, hk, d = case["kind"], case["heads"], case["kv_heads"], case["head_dim"]
    if kind in ("norm_rope", "norm_rope_bwd"):
        n = case["batch"] * case["length"] * (h + hk) * d
        size = 4 if case["dtype"] == "f32" else 2
        touched = 3 if kind == "norm_rope_bwd" else 2
        return {"bytes": float(touched * n * size + 2 * case["length"] * d),
                "flops": (10.0 if kind == "norm_rope_bwd" else 5.0) * n}
    new, lens = _lens(case)
    N, S = sum(new), case["seqs"]
    if kind == "append":
        # q, k, v read and written, a row of each table for each token
        return {"bytes": float(N * (2 * 2 * (h + 2 * hk) * d + 2 * d) + 12 * S),
                "flops": 5.0 * N * (h + hk) * d}
    if kind == "evict":
        cap = -(-max(lens) // case["page"]) * case["page"]
        kept = [min(c, case["keep"]) for c in lens]
        return {"bytes": float(sum(kept) * hk * d * 2 * 2 * 2 + 4 * sum(lens)
                               + 4 * S * (cap + case["keep"] + 2)), "flops": float(sum(lens))}
    seen = [_seen(n, c, case.get("window", 0)) for n, c in zip(new, lens)]
    pairs, entries = sum(p for p, _ in seen), sum(e for _, e in seen)
    pages = 4 * sum(-(-c // case["page"]) for c in lens)
    if kind == "attention":
        return {"bytes": float(2 * entries * hk * d * 2 + N * h * (2 * d * 2 + 4) + pages),
                "flops": 4.0 * pairs * h * d}
    cap = -(-max(lens) // case["page"]) * case["page"]
    return {"bytes": float(entries * hk * d * 2 + N * h * (d * 2 + 4) + 8 * S * cap + pages),
            "flops": 2.0 * pairs * h * d}


# ---- the same in 64 bits ----------------------------------------------------------

def _turn64(x, angle, sign):
    """Adjacent pairs of the first half of each row, as complex numbers, turned
    by -sign * angle (..., D / 4)."""
    x = x.clone()
    half = x.shape[-1] // 2
    z = torch.view_as_complex(x[..., :half].reshape(*x.shape[:-1], half // 2, 2).contiguous())
    z = z * torch.complex(angle[0], -sign * angle[1])
    x[..., :half] = torch.view_as_real(z).flatten(-2)
    return x


def _norm_rope64(x, cs, sn):
    x = x.double()
    x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS)
    return _turn64(x, (cs.double(), sn.double()), 1.0)


def _norm_rope_bwd64(g, x, cs, sn):
    """Jacobian of x / sqrt(|x|^2 / D + eps) times the turned-back gradient."""
    x, g = x.double(), _turn64(g.double(), (cs.double(), sn.double()), -1.0)
    size = torch.sqrt(x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS)
    return g / size - x * (x * g).sum(-1, keepdim=True) / (x.shape[-1] * size ** 3)


def _rows64(cache, table, s, count):
    """Entries 0 .. count - 1 of sequence s: (Hkv, count, D)."""
    page = cache.shape[2]
    x = cache[table[s, :-(-count // page)].long()]
    return torch.cat(x.unbind(0), dim=1)[:, :count].double()


def _attention64(st, window):
    """Sequence by sequence and head by head, in 64 bits: (out, lse)."""
    new, lens = _lens(st["case"])
    H, Hk = st["q"].shape[1], st["k_cache"].shape[1]
    out, lse, at = [], [], 0
    for s, (n, c) in enumerate(zip(new, lens)):
        k, v = (_rows64(st[x], st["table"], s, c) for x in ("k_cache", "v_cache"))
        i = torch.arange(c - n, c, device=DEV)[:, None]
        j = torch.arange(c, device=DEV)[None, :]
        hidden = (j > i) | (i - j >= window) if window else j > i
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
    return torch.cat(out), torch.cat(lse)


def _weight64(st):
    new, lens = _lens(st["case"])
    H, Hk = st["q"].shape[1], st["k_cache"].shape[1]
    out, at = st["weight"].double(), 0
    for s, (n, c) in enumerate(zip(new, lens)):
        k = _rows64(st["k_cache"], st["table"], s, c)
        i = torch.arange(c - n, c, device=DEV)[:, None]
        hidden = torch.arange(c, device=DEV)[None, :] > i
        for g in range(H):
            x = st["q"][at:at + n, g].double() @ k[g * Hk // H].t().contiguous() * SCALE
            p = torch.exp(x - st["lse"][at:at + n, g].double()[:, None])
            out[s, :c] += p.masked_fill(hidden, 0.0).sum(0)
        at += n
    return out


def _evict64(st, keep, recent):
    """Index and lengths from sorted lists on the host; the moved rows by them."""
    k, v, page = st["k_cache"].double(), st["v_cache"].double(), st["k_cache"].shape[2]
    weight = torch.zeros_like(st["weight"], dtype=torch.float64)
    host, lens = st["weight"].cpu().numpy(), st["lens"].tolist()
    index = torch.full((len(lens), keep), -1, dtype=torch.int32)
    for s, c in enumerate(lens):
        old = max(0, c - recent)
        ranked = sorted(range(old), key=lambda e: (-host[s][e], e))
        kept = sorted(ranked[:max(0, keep - (c - old))]) + list(range(old, c))
        e = torch.tensor(kept, device=DEV)
        at = torch.arange(len(kept), device=DEV)
        index[s, :len(kept)] = e.int().cpu()
        a, b = st["table"][s, e // page].long(), st["out_table"][s, at // page].long()
        k[b, :, at % page] = k[a, :, e % page]
        v[b, :, at % page] = v[a, :, e % page]
        weight[s, :len(kept)] = st["weight"][s, e].double()
    return {"index": index, "lens": torch.tensor([min(c, keep) for c in lens], dtype=torch.int32),
            "weight": weight, "k_cache": k, "v_cache": v}


def exact(case, seed):
    st, kind = prepare(case, seed), case["kind"]
    if kind in ("norm_rope", "norm_rope_bwd"):
        cs, sn = st["cs"][:, None, :], st["sn"][:, None, :]
        if kind == "norm_rope":
            return {n: _norm_rope64(st[n], cs, sn) for n in "qk"}
        return {n: _norm_rope_bwd64(st["g" + n], st[n], cs, sn) for n in "qk"}
    if kind == "attention":
        out, lse = _attention64(st, case["window"])
        return {"out": out, "lse": lse}
    if kind == "weight":
        return _weight64(st)
    if kind == "evict":
        return _evict64(st, case["keep"], case["recent"])
    new, lens = _lens(case)
    page, at = case["page"], 0
    k, v, q = st["k_cache"].double(), st["v_cache"].double(), []
    for s, (n, c) in enumerate(zip(new, lens)):
        e = torch.arange(c - n, c, device=DEV)
        cs, sn = st["cs"][e][:, None, :], st["sn"][e][:, None, :]
        q.append(_norm_rope64(st["q"][at:at + n], cs, sn))
        where = st["table"][s, e // page].long()
        k[where, :, e % page] = _norm_rope64(st["k"][at:at + n], cs, sn)
        v[where, :, e % page] = st["v"][at:at + n].double()
        at += n
    return {"q": torch.cat(q), "k_cache": k, "v_cache": v}
