"""The serving step's plain implementations on cases worked out by hand."""

import math

import pytest

import oracle.ref_serve as R


def test_assign_by_hand():
    # pages of 16; page 2 is held by sequence 0, page 4 by others, 0, 1, 3 are free
    got = R.assign([[2, -1], [-1, -1], [-1, -1]], [15, 0, 0], [3, 17, 1], [0, 0, 1, 0, 1], 16, 32)
    # sequence 0 takes page 0; sequence 1 two pages (1, 3); sequence 2 finds none
    assert got["table"] == [[2, 0], [1, 3], [-1, -1]] and got["refs"] == [1, 1, 1, 1, 1]
    assert got["starts"] == [0, 3, 20, 20] and got["lens"] == [18, 17, 0]
    assert got["seq"][:4] == [0, 0, 0, 1] and got["seq"][20:] == [-1] * 12
    assert got["pos"][:4] == [15, 16, 17, 0] and got["slot"][:4] == [47, 0, 1, 16]
    assert got["slot"][19] == 48


def test_assign_serves_in_order():
    # one free page: the second asks for two, so the third, which asks for one, gets none
    # either; the fourth needs none
    table, refs = [[0], [-1], [-1], [1]], [1, 1, 0]
    got = R.assign([r + [-1] for r in table], [3, 0, 0, 4], [1, 17, 1, 1], refs, 16, 99)
    assert got["starts"] == [0, 1, 1, 1, 2] and got["refs"] == [1, 1, 0]
    # rows: the second passes them, and with it all behind
    got = R.assign([[0], [1], [2]], [0, 0, 0], [4, 9, 1], [1, 1, 1], 16, 12)
    assert got["starts"] == [0, 4, 4, 4]
    # one that its table row does not hold asks for nothing
    got = R.assign([[0], [1]], [10, 0], [7, 5], [1, 1], 16, 5)
    assert got["starts"] == [0, 0, 5] and got["lens"] == [10, 5]


def test_release_by_hand():
    assert R.release([[3, 1, -1], [3, 7, 0]], [17, 0], [1, 1, 0, 2], 16) == (
        [[3, 1, -1], [-1, -1, -1]], [0, 1, 0, 1])


@pytest.mark.parametrize("u,kw,want", [
    (0.0, {}, 0), (0.2, {}, 1), (0.6, {}, 1), (0.95, {}, 3),
    (0.99, {"top_k": 1}, 1), (0.99, {"top_k": 2}, 3), (0.5, {"top_p": 0.5}, 1),
    (0.2, {"temperature": 0.0}, 1), (0.0, {"min_p": 0.2}, 1), (0.99, {"min_p": 0.2}, 3),
])
def test_sample_by_hand(u, kw, want):
    # weights 1, 8, 0 and 2 of 11: sums 1/11, 9/11, 9/11, 1
    row = [math.log(1.0), math.log(8.0), -math.inf, math.log(2.0)]
    assert R.sample(row, u, **kw)[0] == want


def test_sample_shares_and_ties():
    row = [0.0, 1.0, 1.0, 1.0, math.nan, -math.inf]
    i, lp = R.sample(row, 0.5, top_k=2)       # equal entries stay together
    assert i == 2 and lp == pytest.approx(-math.log(3.0))
    i, lp = R.sample(row, 0.999, top_p=0.01)
    assert i == 3 and lp == pytest.approx(-math.log(3.0))
    assert R.sample(row, 0.5, temperature=0.0) == (1, 0.0)
    assert R.sample([-math.inf, math.nan], 0.5) == (-1, -math.inf)
    assert R.sample([math.inf, 3.0, math.inf], 0.9) == (2, pytest.approx(-math.log(2.0)))
    # far below the largest: never drawn
    assert R.sample([-30.0, 0.0], 0.0)[0] == 1
