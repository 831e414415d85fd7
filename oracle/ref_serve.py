"""Plain restatement of a serving step's operators, from their definitions: pages
given to sequences and taken back, one number at a time, and a token from a row of logits in
64 bits and more.  Test infrastructure."""

import math

import numpy as np

LEAST = 2.0 ** -40


def assign(table, lens, new, refs, page, rows):
    """Lists in, a dict of lists out."""
    table, refs = [list(r) for r in table], list(refs)
    cols = len(table[0]) if table else 0
    cap = cols * page
    free = [p for p, n in enumerate(refs) if n <= 0]
    asked_rows = asked_pages = 0
    out = {"starts": [0], "lens": [], "seq": [], "pos": [], "slot": []}
    taken = 0
    for s, row in enumerate(table):
        at, n = min(max(lens[s], 0), cap), max(new[s], 0)
        if at + n > cap:
            n = 0
        else:
            need = [c for c in range(cols) if c * page < at + n and (c + 1) * page > at
                    and not 0 <= row[c] < len(refs)] if n else []
            asked_rows += n
            asked_pages += len(need)
            if asked_rows > rows or (need and asked_pages > len(free)):
                n = 0
            else:
                for c in need:
                    row[c] = free[taken]
                    refs[row[c]] = 1
                    taken += 1
        for e in range(at, at + n):
            p = row[e // page]
            out["seq"].append(s)
            out["pos"].append(e)
            out["slot"].append(p * page + e % page)
        out["starts"].append(out["starts"][-1] + n)
        out["lens"].append(at + n)
    for name in ("seq", "pos", "slot"):
        out[name] += [-1] * (rows - len(out[name]))
    out["table"], out["refs"] = table, refs
    return out


def release(table, lens, refs, page):
    table, refs = [list(r) for r in table], list(refs)
    for row, n in zip(table, lens):
        for c in range(len(row)):
            if c * page >= n:
                if 0 <= row[c] < len(refs):
                    refs[row[c]] -= 1
                row[c] = -1
    return table, refs


def sample(row, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(index, log of its share) for one row of 32-bit numbers; the settings are taken
    as 32-bit numbers too.  Weights and sums in extended precision."""
    x = np.asarray(row, dtype=np.float64)
    u, temperature, top_p, min_p = (float(np.float32(v)) for v in (u, temperature, top_p, min_p))
    at = np.flatnonzero(x > -math.inf)   # a NaN is not above
    if not len(at):
        return -1, -math.inf
    v = x[at]
    top = v.max()
    if not temperature > 0:
        return int(at[v == top][0]), 0.0
    u = min(max(u, 0.0), 1.0 - 2.0 ** -24) if u == u else 0.0
    w = np.ones(len(v), dtype=np.longdouble)
    below = v != top
    with np.errstate(under="ignore"):
        w[below] = np.exp((v[below].astype(np.longdouble) - np.longdouble(top)) / np.longdouble(temperature))
    stay = w >= min(max(min_p, LEAST), 1.0)
    if 0 < top_k < len(x) and top_k <= len(v):
        stay &= v >= np.sort(v)[len(v) - top_k]
    at, v, w = at[stay], v[stay], w[stay]
    if top_p < 1.0:
        values, which = np.unique(-v, return_inverse=True)     # from the largest down
        mass = np.zeros(len(values), dtype=np.longdouble)
        np.add.at(mass, which, w)
        run = np.cumsum(mass)
        enough = int((run < np.longdouble(max(top_p, 0.0)) * run[-1]).sum())
        stay = v >= -values[min(enough, len(values) - 1)]
        at, v, w = at[stay], v[stay], w[stay]
    run = np.cumsum(w)
    pick = min(int((run <= np.longdouble(u) * run[-1]).sum()), len(at) - 1)
    return int(at[pick]), float(np.log(w[pick] / run[-1]))
