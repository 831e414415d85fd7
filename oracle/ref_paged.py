"""ORACLE -- test infrastructure only.

The paged cache's operators in 64 bits, token by token, on the CPU: the plain
implementations that the GPU tests compare with."""
import math

import torch

EPS = 1e-6


def entries(cache, table_row, count):
    """The first `count` entries of a sequence, (count, heads, dim) float64."""
    page = cache.shape[2]
    ids = [int(table_row[e // page]) for e in range(count)]
    ids = [i if 0 <= i < cache.shape[0] else 0 for i in ids]
    rows = [cache[i, :, e % page] for e, i in enumerate(ids)]
    return torch.stack(rows).double() if rows else torch.zeros(0, cache.shape[1], cache.shape[3]).double()


def norm_rope(x, cs, sn):
    """x (..., D) float64; cs, sn broadcast against (..., D / 4)."""
    n = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
    y = n.clone()
    half = x.shape[-1] // 2
    a, b = n[..., 0:half:2], n[..., 1:half:2]
    y[..., 0:half:2] = cs * a + sn * b
    y[..., 1:half:2] = cs * b - sn * a
    return y


def tokens(starts, lens, cap):
    """(row, sequence, entry) of every new token."""
    out = []
    for s in range(len(lens)):
        n = starts[s + 1] - starts[s]
        length = min(max(lens[s], 0), cap)
        out += [(starts[s] + i, s, length - n + i) for i in range(n)]
    return out


def attention(q, kc, vc, table, starts, lens, scale, window):
    """-> out, lse and the bounds that a bf16 result may be off by: one rounding
    of the weights and one of the result (2^-8 each), the scores' fp32 error in
    the exponent, and the fp32 sums.  Rows without a token keep NaN."""
    N, H, D = q.shape
    Hk, page = kc.shape[1], kc.shape[2]
    q = q.double()
    out = torch.full((N, H, D), math.nan, dtype=torch.float64)
    lse = torch.full((N, H), math.nan, dtype=torch.float64)
    tol, ltol = torch.zeros(N, H, D).double(), torch.zeros(N, H).double()
    for n, s, e in tokens(starts, lens, table.shape[1] * page):
        lo = max(0, e - window + 1) if window else 0
        k = entries(kc, table[s], max(e + 1, 0))[lo:]
        v = entries(vc, table[s], max(e + 1, 0))[lo:]
        for h in range(H):
            g = h * Hk // H
            if not len(k):
                out[n, h], lse[n, h] = 0.0, -math.inf
                continue
            x = scale * (k[:, g] @ q[n, h])
            size = abs(scale) * (k[:, g].abs() @ q[n, h].abs())
            lse[n, h] = torch.logsumexp(x, 0)
            p = torch.softmax(x, 0)
            out[n, h] = p @ v[:, g]
            # a score's sum of D products, and its scaling; exp2 of it
            d = (size.max() * (D + 4) + x.abs().max() * 2 + 4) * 2.0 ** -24
            sums = (len(k) + 16) * 2.0 ** -24
            mass = p @ v[:, g].abs()
            tol[n, h] = 2.0 ** -8 * out[n, h].abs() + (2.0 ** -8 + 2 * d + 2 * sums) * mass + 1e-30
            ltol[n, h] = d + sums + 2.0 ** -22 * (1 + lse[n, h].abs())
    return out, lse, tol, ltol


def attention_whole(q, kc, vc, table, starts, lens, scale, window):
    """``attention`` a sequence and cache head at a time, for long ones.  Its bounds
    take the weights in two bf16 halves (2^-16 of each, the second rounded to 2^-8
    of at most 2^-8 of the first) where a sequence has up to 16 rows."""
    N, H, D = q.shape
    Hk, page, cap = kc.shape[1], kc.shape[2], table.shape[1] * kc.shape[2]
    G = H // Hk
    out = torch.full((N, H, D), math.nan, dtype=torch.float64)
    lse = torch.full((N, H), math.nan, dtype=torch.float64)
    tol, ltol = torch.zeros(N, H, D).double(), torch.zeros(N, H).double()
    for s in range(len(lens)):
        a, n = starts[s], starts[s + 1] - starts[s]
        length = min(max(lens[s], 0), cap)
        if not n:
            continue
        ids = table[s, :-(-length // page)].long()
        ids = torch.where((ids >= 0) & (ids < kc.shape[0]), ids, 0)
        k, v = (x[ids].transpose(1, 2).reshape(-1, Hk, D)[:length] for x in (kc, vc))
        e = torch.arange(length - n, length)[:, None]
        j = torch.arange(length)[None, :]
        sees = (j <= e) & (e - j < window) if window else j <= e
        some = sees.any(1)
        rounding = 2.0 ** -16 if n * G <= 16 else 2.0 ** -8
        for h in range(H):
            kh, vh, qh = k[:, h // G].double(), v[:, h // G].double(), q[a:a + n, h].double()
            x = torch.where(sees, scale * (qh @ kh.t()), -math.inf)
            size = torch.where(sees, abs(scale) * (qh.abs() @ kh.abs().t()), 0.0)
            lse[a:a + n, h] = torch.logsumexp(x, 1) if length else -math.inf
            p = torch.where(some[:, None], torch.softmax(x, 1), 0.0)
            o, mass = p @ vh, p @ vh.abs()
            # NaN and infinities of entries that some rows see
            for i in torch.nonzero(~torch.isfinite(o).all(1)).flatten().tolist():
                o[i], mass[i] = p[i, sees[i]] @ vh[sees[i]], p[i, sees[i]] @ vh[sees[i]].abs()
            out[a:a + n, h] = o
            if not length:
                continue
            top = torch.where(sees, x.abs(), 0.0).amax(1)
            d = (size.amax(1) * (D + 4) + top * 2 + 4) * 2.0 ** -24
            sums = (sees.sum(1) + 16) * 2.0 ** -24
            tol[a:a + n, h] = 2.0 ** -8 * o.abs() + (rounding + 2 * d + 2 * sums)[:, None] * mass + 1e-30
            ltol[a:a + n, h] = d + sums + 2.0 ** -22 * (1 + lse[a:a + n, h].abs())
    return out, lse, tol, ltol


def weight(q, lse, kc, table, starts, lens, w, scale, window):
    """-> the new weights and the bounds of an fp32 result."""
    N, H, D = q.shape
    Hk, page = kc.shape[1], kc.shape[2]
    q, lse, out = q.double(), lse.double(), w.double().clone()
    tol, terms = torch.zeros_like(out), torch.zeros_like(out)
    for n, s, e in tokens(starts, lens, table.shape[1] * page):
        lo = max(0, e - window + 1) if window else 0
        k = entries(kc, table[s], max(e + 1, 0))[lo:]
        if not len(k):
            continue
        for h in range(H):
            g = h * Hk // H
            x = scale * (k[:, g] @ q[n, h])
            size = abs(scale) * (k[:, g].abs() @ q[n, h].abs())
            y = x - lse[n, h]
            p = torch.exp(y)
            out[s, lo:e + 1] += p
            terms[s, lo:e + 1] += 1
            tol[s, lo:e + 1] += p * (size * (D + 4) + (x.abs() + lse[n, h].abs() + y.abs()) * 2 + 8) * 2.0 ** -24
    # the sum of the terms in fp32, in any order
    return out, tol + out.abs() * (terms + 4) * 2.0 ** -24 + 1e-30


def weight_whole(q, lse, kc, table, starts, lens, w, scale, window):
    """``weight`` a sequence and cache head at a time, for long ones."""
    H, D = q.shape[1:]
    Hk, page, cap = kc.shape[1], kc.shape[2], w.shape[1]
    out = w.double().clone()
    tol, terms = torch.zeros_like(out), torch.zeros_like(out)
    for s in range(len(lens)):
        a, n = starts[s], starts[s + 1] - starts[s]
        length = min(max(lens[s], 0), cap)
        if not n or not length:
            continue
        ids = table[s, :-(-length // page)].long()
        ids = torch.where((ids >= 0) & (ids < kc.shape[0]), ids, 0)
        k = kc[ids].transpose(1, 2).reshape(-1, Hk, D)[:length]
        e = torch.arange(length - n, length)[:, None]
        j = torch.arange(length)[None, :]
        sees = (j <= e) & (e - j < window) if window else j <= e
        for h in range(H):
            kh, qh = k[:, h * Hk // H].double(), q[a:a + n, h].double()
            l = lse[a:a + n, h].double()[:, None]
            x = scale * (qh @ kh.t())
            size = abs(scale) * (qh.abs() @ kh.abs().t())
            y = x - l
            p = torch.where(sees, torch.exp(y), 0.0)
            d = torch.where(sees, size * (D + 4) + (x.abs() + l.abs() + y.abs()) * 2 + 8, 0.0)
            out[s, :length] += p.sum(0)
            terms[s, :length] += sees.sum(0)
            tol[s, :length] += torch.where(sees, p * d, 0.0).sum(0) * 2.0 ** -24
    return out, tol + out.abs() * (terms + 4) * 2.0 ** -24 + 1e-30


def evict(kc, vc, table, lens, w, keep, recent, out_table):
    """-> index, new lens, weight, and the caches after the move."""
    page, cap = kc.shape[2], w.shape[1]
    k2, v2 = kc.clone(), vc.clone()
    index = torch.full((len(lens), keep), -1, dtype=torch.int32)
    left, out = [], torch.zeros_like(w)
    for s, length in enumerate(lens):
        length = min(max(length, 0), cap)
        last = min(recent, length, keep)
        old = length - last
        value = [(-math.inf if math.isnan(x) else x, math.isnan(x)) for x in w[s].tolist()]
        # NaN below every number, -inf included
        ranked = sorted(range(old), key=lambda e: (value[e][1], -value[e][0], e))
        kept = sorted(ranked[:min(keep, length) - last]) + list(range(old, length))
        left.append(len(kept))
        for i, e in enumerate(kept):
            index[s, i], out[s, i] = e, w[s, e]
            a, b = int(table[s, e // page]), int(out_table[s, i // page])
            a = a if 0 <= a < kc.shape[0] else 0
            if 0 <= b < kc.shape[0]:
                k2[b, :, i % page] = kc[a, :, e % page]
                v2[b, :, i % page] = vc[a, :, e % page]
    return index, torch.tensor(left, dtype=torch.int32), out, k2, v2
