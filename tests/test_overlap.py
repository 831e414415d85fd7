"""Operands that share memory: the test that the C ABI makes of strided operands
against every byte of small ones, and what it refuses through it."""

import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "attention_nn_amd", "csrc")

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include <set>
#include "overlap.h"
using namespace ann;

static std::set<int64_t> bytes(const Strided& x) {
  std::set<int64_t> s;
  for (int64_t i = 0; i < x.n; ++i)
    for (int64_t j = 0; j < x.m; ++j)
      for (int64_t b = 0; b < x.size; ++b) s.insert((intptr_t)x.at + i * x.row + j * x.col + b);
  return s;
}

int main() {
  srand(1);
  int met = 0, apart = 0;
  auto pick = [](int lo, int hi) { return (int64_t)(lo + rand() % (hi - lo + 1)); };
  for (int t = 0; t < 200000; ++t) {
    Strided x{(const void*)pick(1000, 1060), pick(0, 5), pick(-20, 40), pick(1, 4), pick(-9, 20), pick(0, 6)};
    Strided y{(const void*)pick(1000, 1060), pick(0, 4), t % 3 ? pick(-20, 40) : x.row, 1, 0, pick(0, 7)};
    if (t % 2) x.m = 1;
    bool want = false;
    const auto a = bytes(x);
    for (int64_t b : bytes(y)) want = want || a.count(b);
    if (overlap(x, y) != want) return 1;
    (want ? met : apart)++;
  }
  if (met < 20000 || apart < 20000) return 2;
  // strides and counts that pass 64 bits of bytes together
  const Strided far{(const void*)4096, 1 << 30, INT64_MAX / 4, 1, 0, 64}, near{(const void*)4096, 1, 0, 1, 0, 64};
  const Strided past{(const void*)8192, 1, 0, 1, 0, 64};
  return overlap(far, near) && !overlap(far, past) ? 0 : 3;
}
"""


def test_overlap_of_strided_operands(tmp_path):
    src, exe = tmp_path / "t.cpp", str(tmp_path / "t")
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I", CSRC, str(src), "-o", exe], check=True)
    assert subprocess.run([exe]).returncode == 0


FAKE = 1 << 40


def test_results_on_a_row_between_gaps_are_refused():
    """Queries (keys, values) whose rows lie further apart than the whole result:
    a result on one of them is refused as one on the first is."""
    from attention_nn_amd import _lib
    L = _lib.lib()
    c = _lib.AnnPaged(k=FAKE, v=FAKE, k_page=6 * 16 * 128, k_head=16 * 128, k_slot=128, v_page=6 * 16 * 128,
                      v_head=16 * 128, v_slot=128, table=FAKE, table_row=8, starts=FAKE, lens=FAKE, pages=64,
                      page_size=16, heads=6, head_dim=128, seqs=4, cols=8, rows=4)
    row = 1 << 20   # elements, of which 768 are a row
    for at in (row * 2, row * 6 + 5 * 256, row * 4 - 2 * 4 * 768 + 16, row * 2 + 767 * 2 - 14):
        assert L.ann_op_paged_attention(c, FAKE, row, 128, 6, 0.1, 0, FAKE + at, None, FAKE, 1 << 40,
                                        None) == _lib.ANN_E_ARG
        assert "overlaps" in L.ann_last_error().decode()
        for name in ("q", "k", "v"):
            r = _lib.AnnQkRows(q=FAKE << 1, k=FAKE << 2, v=FAKE << 3, q_out=FAKE + at, cs=FAKE, sn=FAKE, table_rows=64,
                               B=1, T=4, Hq=6, Hk=6, D=128, dtype=1, eps=1e-6)
            setattr(r, name, FAKE)
            for s in (r.q_stride, r.k_stride, r.v_stride):
                s[1], s[2] = row, 128
            assert L.ann_op_paged_append(c, r, None) == _lib.ANN_E_ARG
            assert "overlaps" in L.ann_last_error().decode()


def test_weights_that_overlap_in_part_are_refused():
    """New weights into memory that shares some rows with the old ones, or parts of
    rows, and into the log sums."""
    from attention_nn_amd import _lib
    L = _lib.lib()
    c = _lib.AnnPaged(k=FAKE, v=FAKE, k_page=6 * 16 * 128, k_head=16 * 128, k_slot=128, v_page=6 * 16 * 128,
                      v_head=16 * 128, v_slot=128, table=FAKE, table_row=8, starts=FAKE, lens=FAKE, pages=64,
                      page_size=16, heads=6, head_dim=128, seqs=4, cols=8, rows=4)

    def weight(w, wrow, out, orow, lse=FAKE << 2):
        return L.ann_op_paged_weight(c, FAKE, 768, 128, 6, lse, 0.1, 0, w, wrow, out, orow, None, 0, None)

    def evict(w, wrow, out, orow):
        return L.ann_op_paged_evict(c, FAKE, 8, 8, w, wrow, 100, 10, FAKE << 2, FAKE << 3, out, orow, None)

    # rows of 128 weights: one row on, half a row, the last one, a row of a broadcast
    # one, other strides that meet in row 2
    for w, wrow, out, orow in ((FAKE, 128, FAKE + 512, 128), (FAKE, 128, FAKE - 256, 128), (FAKE, 256, FAKE + 508, 256),
                               (FAKE, 128, FAKE + 3 * 512 + 508, 128), (FAKE, 0, FAKE - 1024, 128),
                               (FAKE, 300, FAKE + 800, 128), (FAKE, 128, FAKE, 128 + 4)):
        for call in (weight, evict):
            assert call(w, wrow, out, orow) == _lib.ANN_E_ARG, (w, wrow, out, orow)
            assert "weight" in L.ann_last_error().decode()
    for lse in (FAKE, FAKE + 2048 - 4, FAKE - 92):
        assert weight(FAKE << 3, 128, FAKE, 128, lse) == _lib.ANN_E_ARG
        assert "lse" in L.ann_last_error().decode()


def test_a_cache_that_is_written_has_rows_of_its_own():
    """Broadcast pages, heads or slots, and one tensor for keys and values, may be read,
    not appended to or evicted from."""
    from attention_nn_amd import _lib
    L = _lib.lib()
    plain = dict(k=FAKE, v=FAKE << 1, k_page=6 * 16 * 128, k_head=16 * 128, k_slot=128, v_page=6 * 16 * 128,
                 v_head=16 * 128, v_slot=128, table=FAKE, table_row=8, starts=FAKE, lens=FAKE, pages=64,
                 page_size=16, heads=6, head_dim=128, seqs=4, cols=8, rows=4)
    for kw in ({"k_page": 0}, {"k_head": 0}, {"k_slot": 0}, {"v_page": 0}, {"v_head": 0}, {"v_slot": 0}, {"v": FAKE}):
        c = _lib.AnnPaged(**{**plain, **kw})
        r = _lib.AnnQkRows(q=FAKE, k=FAKE, v=FAKE, q_out=FAKE, cs=FAKE, sn=FAKE, table_rows=64, B=1, T=4, Hq=6, Hk=6,
                           D=128, dtype=1, eps=1e-6)
        r.k, r.v = FAKE << 2, FAKE << 3
        for s in (r.q_stride, r.k_stride, r.v_stride):
            s[1], s[2] = 768, 128
        assert L.ann_op_paged_append(c, r, None) == _lib.ANN_E_ARG
        assert "share memory" in L.ann_last_error().decode()
        assert L.ann_op_paged_evict(c, FAKE, 8, 8, FAKE, 128, 100, 10, FAKE << 2, FAKE << 3, FAKE << 4, 128,
                                    None) == _lib.ANN_E_ARG
        assert "share memory" in L.ann_last_error().decode()
