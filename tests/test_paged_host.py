"""The paged cache without a GPU: where its addresses may go whatever the tables
hold (the kernels' own helpers, compiled for the host), what the C ABI refuses
before any launch, and what the Python layer does."""

import ctypes
import os
import subprocess

import pytest
import torch

from attention_nn_amd import _lib, kernels, paged

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "attention_nn_amd", "csrc")

PROGRAM = r"""
#include <cstdio>
#include <climits>
#include <initializer_list>
#include "paged.h"
using namespace ann;

int main() {
  const int odd[] = {INT_MIN, -70000, -1, 0, 1, 15, 16, 17, 63, 64, 70000, 1 << 30, INT_MAX};
  // a length never passes the table, whatever it says
  for (int cols : {0, 1, 3, 1 << 20})
    for (int sh : {4, 7, 10})
      for (int len : odd) {
        const int l = pg_len(len, cols, sh);
        if (l < 0 || l > (long long)cols << sh) return 1;
        if (len >= 0 && len <= (long long)cols << sh && l != len) return 2;
      }
  // new tokens never pass the rows
  for (int rows : {0, 1, 17, 70000})
    for (int a : odd)
      for (int b : odd) {
        const PgRange r = pg_range(a, b, rows);
        if (r.first < 0 || r.n < 0 || r.first + r.n > rows) return 3;
        if (0 <= a && a <= b && b <= rows && (r.first != a || r.n != b - a)) return 4;
      }
  // pages
  for (int pages : {1, 5, 1 << 30})
    for (int id : odd) {
      const bool is = id >= 0 && id < pages;
      if (pg_writable(id, pages) != is || pg_read(id, pages) != (is ? id : 0)) return 5;
    }
  // slots, past 2^31 elements
  if (pg_slot(35, 4, 128) != 3 * 128 || pg_slot(1023, 10, 1LL << 40) != 1023LL << 40) return 6;
  // quotients
  for (int d = 1; d < 70000; d = d < 300 ? d + 1 : d * 3 / 2 + 1) {
    const FastDiv f = FastDiv::of(d);
    for (int n : {0, 1, 2, 1000, 65535, 1 << 20, INT_MAX - 1, INT_MAX}) {
      if (f.div(n) != n / d) return 7;
      const int k = n / d * d;   // and on both sides of a multiple
      if (f.div(k) != k / d || (k && f.div(k - 1) != (k - 1) / d)) return 8;
    }
  }
  return 0;
}
"""


def test_addresses_stay_in_bounds(tmp_path):
    src = tmp_path / "t.cpp"
    src.write_text(PROGRAM)
    exe = str(tmp_path / "t")
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", CSRC, str(src), "-o", exe], check=True)
    assert subprocess.run([exe]).returncode == 0


FAKE = 1 << 40


def _paged(**kw):
    c = _lib.AnnPaged(k=FAKE, v=FAKE, k_page=6 * 16 * 128, k_head=16 * 128, k_slot=128,
                      v_page=6 * 16 * 128, v_head=16 * 128, v_slot=128, table=FAKE, table_row=8,
                      starts=FAKE, lens=FAKE, pages=64, page_size=16, heads=6, head_dim=128, seqs=4,
                      cols=8, rows=4)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def _attention(c, heads=6, q=FAKE, row=768, head=128, scale=0.1, window=0, out=FAKE, ws=FAKE, nws=1 << 40):
    return _lib.lib().ann_op_paged_attention(c, q, row, head, heads, scale, window, out, None, ws, nws, None)


@pytest.mark.parametrize("field,value,msg", [
    ("head_dim", 96, "head_dim"), ("heads", 0, "shape"), ("pages", 0, "shape"), ("seqs", -1, "shape"),
    ("seqs", 70000, "65535"), ("cols", -1, "shape"), ("rows", -2, "shape"), ("page_size", 8, "power of two"),
    ("page_size", 24, "power of two"), ("page_size", 2048, "power of two"), ("cols", 1 << 27, "2^30"),
    ("k", None, "null"), ("v", None, "null"), ("lens", None, "null"), ("table", None, "null"),
    ("starts", None, "null"), ("k", FAKE + 8, "aligned"), ("k_slot", 132, "aligned"), ("v_head", 4, "aligned"),
    ("k_slot", (1 << 25) + 8, "2^25"), ("v_slot", -8, "2^25"),
])
def test_cache_refusals(field, value, msg):
    assert _attention(_paged(**{field: value})) == _lib.ANN_E_ARG
    assert msg in _lib.lib().ann_last_error().decode()


@pytest.mark.parametrize("kw,msg", [
    ({"heads": 8}, "8 query heads over 6"), ({"heads": 0}, "query heads"), ({"q": None}, "null"),
    ({"q": FAKE + 2}, "aligned"), ({"row": 770}, "aligned"), ({"scale": float("nan")}, "finite"),
    ({"scale": float("inf")}, "finite"), ({"window": -1}, "window"), ({"out": None}, "out is null"),
    ({"row": 1 << 26}, "strides"), ({"head": 1 << 27}, "strides"), ({"row": -768}, "strides"),
    ({"out": FAKE + 4}, "aligned"), ({"heads": 600}, "2^30"),
    ({"scale": 3e38}, "finite"), ({"out": FAKE + 16}, "overlaps"), ({"out": FAKE + 4 * 768 * 2 - 16}, "overlaps"),
    ({"out": FAKE - 16}, "overlaps"), ({"row": 1536}, "overlaps"), ({"row": 0}, "overlaps"),
])
def test_attention_refusals(kw, msg):
    assert _attention(_paged(rows=1 << 22 if kw == {"heads": 600} else 4), **kw) == _lib.ANN_E_ARG
    assert msg in _lib.lib().ann_last_error().decode()
    assert _lib.lib().ann_op_paged_attention(None, FAKE, 768, 128, 6, 0.1, 0, FAKE, None, None, 0, None) == _lib.ANN_E_ARG


def test_weight_and_evict_refusals():
    L = _lib.lib()

    def weight(c, lse=FAKE, w=FAKE, wrow=128, out=FAKE, orow=128, heads=6):
        return L.ann_op_paged_weight(c, FAKE, 768, 128, heads, lse, 0.1, 0, w, wrow, out, orow, FAKE, 1 << 40, None)

    for kw in ({"lse": None}, {"w": None}, {"out": None}, {"orow": 256}, {"heads": 9}, {"out": FAKE + 4096, "orow": 120}):
        assert weight(_paged(), **kw) == _lib.ANN_E_ARG
    assert weight(_paged(starts=None)) == _lib.ANN_E_ARG

    def evict(c, table=FAKE, cols=8, w=FAKE, wrow=128, keep=100, recent=10, index=FAKE, lens=FAKE, out=FAKE, orow=128):
        return L.ann_op_paged_evict(c, table, 8, cols, w, wrow, keep, recent, index, lens, out, orow, None)

    for kw in ({"keep": 0}, {"recent": -1}, {"recent": 101}, {"table": None}, {"w": None}, {"index": None},
               {"lens": None}, {"out": None}, {"orow": 64}, {"out": FAKE + 4096, "orow": 120}):
        assert evict(_paged(), **kw) == _lib.ANN_E_ARG, kw
    for kw in ({"cols": 6}, {"cols": -1}, {"keep": 129}):
        assert evict(_paged(), **kw) == _lib.ANN_E_CAPACITY
    assert evict(_paged(v=None)) == _lib.ANN_E_ARG


def test_rows_refusals():
    L = _lib.lib()

    def rows(**kw):
        r = _lib.AnnQkRows(q=FAKE, k=FAKE, v=FAKE, gq=FAKE, gk=FAKE, q_out=FAKE, k_out=FAKE, cs=FAKE, sn=FAKE,
                           table_rows=64, B=1, T=4, Hq=6, Hk=6, D=128, dtype=1, eps=1e-6)
        for k, v in kw.items():
            setattr(r, k, v)
        return r

    bad = [{"D": 6}, {"D": 0}, {"B": -1}, {"T": -1}, {"Hq": -1}, {"dtype": 5}, {"eps": 0.0}, {"eps": float("nan")},
           {"q": None}, {"k": None}, {"q_out": None}, {"k_out": None}, {"cs": None}, {"table_rows": 0},
           {"pos0": -1}, {"pos0": 61}, {"Hq": 65535}]
    for kw in bad:
        assert L.ann_op_qk_norm_rope(rows(**kw), None) == _lib.ANN_E_ARG, kw
        assert L.ann_op_qk_norm_rope_bwd(rows(**kw), None) == _lib.ANN_E_ARG, kw
    assert L.ann_op_qk_norm_rope_bwd(rows(gq=None), None) == _lib.ANN_E_ARG
    assert L.ann_op_qk_norm_rope(None, None) == _lib.ANN_E_ARG
    for kw in [{"D": 64}, {"Hk": 3}, {"Hq": 0}, {"B": 2}, {"T": 5}, {"dtype": 0}, {"v": None}, {"pos": FAKE},
               {"q": FAKE + 4}, {"cs": FAKE + 4}, {"eps": -1.0}, {"q_out": FAKE + 16}, {"q_out": FAKE - 16}]:
        assert L.ann_op_paged_append(_paged(), rows(**kw), None) == _lib.ANN_E_ARG, kw
    odd = rows()
    odd.k_stride[1] = 4
    assert L.ann_op_paged_append(_paged(), odd, None) == _lib.ANN_E_ARG
    assert L.ann_op_paged_append(_paged(), None, None) == _lib.ANN_E_ARG


def test_nothing_to_do_launches_nothing():
    L = _lib.lib()
    assert _attention(_paged(rows=0)) == 0
    assert L.ann_op_paged_weight(_paged(seqs=0), FAKE, 768, 128, 6, FAKE, 0.1, 0, FAKE, 8, FAKE, 8, None, 0, None) == 0
    assert L.ann_op_paged_evict(_paged(seqs=0), FAKE, 8, 8, FAKE, 8, 4, 0, FAKE, FAKE, FAKE, 8, None) == 0


def test_python_layer_needs_gpu_tensors():
    x = torch.zeros(1, 1, 2, 64)
    t = torch.zeros(4, 16)
    with pytest.raises(ValueError, match="GPU tensor"):
        kernels.qk_norm_rope(x, x, t, t)
    with pytest.raises(ValueError, match="GPU tensor"):
        kernels.qk_norm_rope_bwd(x, x, x, x, t, t)
    q = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    c = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    i = torch.zeros(1, 2, dtype=torch.int32)
    for call in (lambda: paged.append(q, q, q, t, t, c, c, i, i[0], i[0, :1]),
                 lambda: paged.attention(q, c, c, i, i[0], i[0, :1], 0.1),
                 lambda: paged.attention_weight(q, t, c, i, i[0], i[0, :1], t, 0.1),
                 lambda: paged.evict(c, c, i, i[0, :1], t, 3)):
        with pytest.raises(ValueError, match="GPU tensor"):
            call()
