"""Attention behind a shared prefix where every weight is as far from a bf16 number as
one can be: a batch on which the weights' second halves show, with the bounds of results that
have them.  Here on the CPU: the bounds hold with both halves and not with one."""

import math

import pytest
import torch

import oracle.ref_paged as R

BF, I32 = torch.bfloat16, torch.int32
SCALE, TOP = 0.1, 5.0


def _key(target):
    """(x0, x1) in bf16 with SCALE (4 x0 + x1 / 64) nearest to target."""
    x0 = torch.arange(2.0, 5.0, 2.0 ** -6).to(BF).double().unique()
    x1 = torch.arange(-4.0, 4.0, 2.0 ** -6).to(BF).double().unique()
    s = SCALE * (4.0 * x0[:, None] + x1 / 64.0) - target
    i = int(s.abs().argmin())
    return float(x0[i // len(x1)]), float(x1[i % len(x1)])


class Halves:
    """S sequences of n new tokens (each with `own` entries of its own) behind `prefix`.
    Of 16 entries one has the largest score, weight 1 and no value; the others weigh
    0.5 (1 + 2^-8) (1 -+ 2^-10), a bf16 half-step above 0.5: a half of them, of value v, is rounded
    down by 2^-8 of it, the other half, of -v, up.  Exactly they cancel but for 2^-9; their
    first halves leave 2^-7 of one half's sum."""

    def __init__(self, S, n, own, prefix, H, Hk, D, page=64, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.S, self.H, self.n = S, H, n
        self.starts = [n * i for i in range(S + 1)]
        self.lens = [prefix + own + 3 * i for i in range(S)]
        cols = -(-max(self.lens) // page)
        full = prefix // page
        pages = full + 1 + S * (cols - full)
        order = torch.randperm(pages, generator=g).to(I32)
        self.ptable = order[:full + 1].view(1, -1)
        rest = order[full + 1:].view(S, cols - full)
        self.table = torch.cat((self.ptable[:, :full].expand(S, full), rest), 1).contiguous()
        self.plens, self.groups = [prefix], [0, S]
        half = math.log(0.5 * (1.0 + 2.0 ** -8))
        kinds = [(TOP, 0.0), _key(SCALE * 4.0 * TOP + half - 2.0 ** -10), _key(SCALE * 4.0 * TOP + half + 2.0 ** -10)]
        value = torch.randn(Hk, D, generator=g).abs() + 0.5
        self.k, self.v = torch.zeros(pages, Hk, page, D), torch.zeros(pages, Hk, page, D)
        for row in [*self.table.tolist(), self.ptable[0].tolist()]:
            for e in range(len(row) * page):
                kind = 0 if e % 16 == 0 else 1 + e % 2
                at = row[e // page], slice(None), e % page
                self.k[at][:, 0], self.k[at][:, 1] = kinds[kind]
                self.v[at] = value * (0.0, 1.0, -1.0)[kind]
        self.q = torch.zeros(S * n, H, D)
        self.q[:, :, 0], self.q[:, :, 1] = 4.0, 1.0 / 64.0
        self.k, self.v, self.q = self.k.to(BF), self.v.to(BF), self.q.to(BF)

    def widened(self):
        """The prefix's table so wide that the call shares it."""
        Hk, page, D = self.k.shape[1:]
        cols = -(-48_100_000 // ((self.S - 1) * Hk * D * 4 * page))
        wide = torch.full((1, max(cols, self.ptable.shape[1])), -1, dtype=I32)
        wide[:, :self.ptable.shape[1]] = self.ptable
        self.ptable = wide
        return self

    def expected(self):
        """out, lse and their bounds, all weights in two halves: 2^-16 of each."""
        args = self.table, self.starts, self.lens, SCALE, 0
        out, lse, tol, ltol = R.attention_whole(self.q, self.k, self.v, *args)
        if self.n * self.H // self.k.shape[1] > 16:    # where that oracle counts one half
            tol -= (2.0 ** -8 - 2.0 ** -16) * R.attention_whole(self.q, self.k, self.v.abs(), *args)[0]
        return out, lse, tol, ltol

    def rounded(self, halves):
        """The result with each weight, relative to the largest, in that many bf16 halves."""
        Hk, page, D = self.k.shape[1:]
        G = self.H // Hk
        out = torch.zeros(*self.q.shape, dtype=torch.float64)
        for s in range(self.S):
            k, v = (x[self.table[s].long()].transpose(1, 2).reshape(-1, Hk, D)[:self.lens[s]].double()
                    for x in (self.k, self.v))
            for i in range(self.n):
                r, e = self.starts[s] + i, self.lens[s] - self.n + i + 1
                for h in range(self.H):
                    x = SCALE * (k[:e, h // G] @ self.q[r, h].double())
                    p = torch.exp(x - x.max())
                    w = left = torch.zeros_like(p)
                    for _ in range(halves):
                        left = (p - w).to(BF).double()
                        w = w + left
                    out[r, h] = w @ v[:e, h // G] / p.sum()
        return out.to(BF).double()


SHAPES = [  # sequences, new, own, prefix, heads
    (3, 1, 40, 400, (2, 2, 128)), (3, 1, 40, 400, (2, 2, 64)), (4, 4, 50, 333, (6, 3, 128)),
    (2, 16, 30, 500, (8, 1, 64)), (2, 3, 3, 130, (8, 2, 128)), (2, 1, 300, 64, (1, 1, 128)),
]


@pytest.mark.parametrize("shape", SHAPES)
def test_bounds_tell_one_half_from_two(shape):
    S, n, own, prefix, (H, Hk, D) = shape
    s = Halves(S, n, own, prefix, H, Hk, D)
    ref, _, tol, _ = s.expected()
    assert ((s.rounded(2) - ref).abs() <= tol).all()
    assert ((s.rounded(1) - ref).abs() > 2.0 * tol).all()
