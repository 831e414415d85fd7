"""The operators of a serving step without a GPU: what the C ABI refuses before any
launch, what a call with nothing to do does, and what the Python layer asks for."""

import ctypes

import pytest
import torch

from attention_nn_amd import _lib, kernels, paged

FAKE = 1 << 40
MB = 1 << 20


def _where(i):
    return FAKE + i * MB


def _table(**kw):
    t = _lib.AnnPagedTable(table=_where(0), table_row=8, lens=_where(1), refs=_where(2), table_out=_where(3),
                           out_row=8, refs_out=_where(4), pages=64, page_size=16, seqs=4, cols=8)
    for k, v in kw.items():
        setattr(t, k, v)
    return t


def _assign(t, new=_where(5), rows=16, starts=_where(6), lens=_where(7), seq=_where(8), pos=_where(9),
            slot=_where(10), ws=_where(11), nws=1 << 40):
    return _lib.lib().ann_op_paged_assign(t, new, rows, starts, lens, seq, pos, slot, ws, nws, None)


def _said(msg):
    return msg in _lib.lib().ann_last_error().decode()


@pytest.mark.parametrize("field,value,msg", [
    ("pages", 0, "shape"), ("seqs", -1, "shape"), ("seqs", 65536, "65535"), ("cols", -1, "shape"),
    ("page_size", 0, "power of two"), ("page_size", 8, "power of two"), ("page_size", 24, "power of two"),
    ("page_size", 2048, "power of two"), ("page_size", -16, "power of two"), ("cols", (1 << 26) + 1, "2^30"),
    ("table", None, "null"), ("table_out", None, "null"), ("lens", None, "null"), ("refs", None, "null"),
    ("refs_out", None, "null"), ("out_row", 7, "rows of table_out overlap"), ("out_row", -8, "rows of table_out overlap"),
    ("refs_out", _where(3) + 4, "refs_out overlaps table_out"), ("refs_out", _where(2) + 4, "refs_out overlaps refs"),
    ("refs_out", _where(1) + 12, "refs_out overlaps lens"), ("refs_out", _where(0) - 252, "refs_out overlaps table"),
    ("table_out", _where(0) + 4, "table_out overlaps table"), ("table_out", _where(2) + 252, "table_out overlaps refs"),
    ("table_out", _where(1) - 124, "table_out overlaps lens"),
])
def test_tables_refused(field, value, msg):
    for call in (_assign, lambda t: _lib.lib().ann_op_paged_release(t, None)):
        assert call(_table(**{field: value})) == _lib.ANN_E_ARG
        assert _said(msg), _lib.lib().ann_last_error()


def test_in_place_only_as_it_lies():
    """A table in place with its rows elsewhere apart is an overlap."""
    for call in (_assign, lambda t: _lib.lib().ann_op_paged_release(t, None)):
        assert call(_table(table_out=_where(0), out_row=16)) == _lib.ANN_E_ARG
        assert _said("table_out overlaps table")
    assert _assign(_table(), lens=_where(1) + 4) == _lib.ANN_E_ARG and _said("new_lens overlaps lens")


@pytest.mark.parametrize("kw,msg", [
    ({"new": None}, "null"), ({"starts": None}, "null"), ({"lens": None}, "null"), ({"seq": None}, "null"),
    ({"pos": None}, "null"), ({"slot": None}, "null"), ({"rows": -1}, "rows=-1"), ({"rows": (1 << 30) + 1}, "2^30"),
    ({"starts": _where(5) + 12}, "starts overlaps new"), ({"starts": _where(7) - 16}, "starts overlaps new_lens"),
    ({"pos": _where(8) + 60}, "pos overlaps seq"), ({"slot": _where(9) - 124}, "slot overlaps pos"),
    ({"seq": _where(2)}, "seq overlaps refs"), ({"slot": _where(3) - 8}, "slot overlaps table_out"),
    ({"lens": _where(5)}, "new_lens overlaps new"),
])
def test_assign_refused(kw, msg):
    assert _assign(_table(), **kw) == _lib.ANN_E_ARG
    assert _said(msg), _lib.lib().ann_last_error()


def test_null_structs():
    L = _lib.lib()
    assert _assign(None) == _lib.ANN_E_ARG and L.ann_op_paged_release(None, None) == _lib.ANN_E_ARG
    assert L.ann_op_sample_logits(None, None) == _lib.ANN_E_ARG
    assert L.ann_op_paged_assign_ws_bytes(None, 4) == 0


def test_workspace_of_assign():
    """None of a small call; of others a bit a page and a few words a sequence and span,
    and a call with less is refused."""
    L = _lib.lib()
    assert L.ann_op_paged_assign_ws_bytes(_table(), 16) == 0
    for kw, rows in (({"pages": 1 << 20}, 16), ({"seqs": 4096}, 16), ({"cols": 1 << 20}, 16), ({}, 1 << 20),
                     ({"seqs": 65535, "cols": 1 << 14, "pages": 1 << 30}, 1 << 30)):
        t = _table(**kw)
        t.out_row = t.table_row = t.cols
        t.table, t.table_out = FAKE << 1, FAKE << 2
        t.refs, t.refs_out = FAKE << 3, FAKE << 4
        n = L.ann_op_paged_assign_ws_bytes(t, rows)
        spans = -(-t.cols * 16 // 4096)
        assert 0 < n <= t.pages // 8 + t.pages // 1024 + t.seqs * (spans + 4) * 4 + 64
        assert _assign(t, rows=rows, seq=FAKE << 5, pos=FAKE << 6, slot=FAKE << 7, nws=n - 1) not in (0, _lib.ANN_E_ARG)
        assert _said("workspace")
    assert L.ann_op_paged_assign_ws_bytes(_table(page_size=17), 16) == 0
    assert L.ann_op_paged_assign_ws_bytes(_table(), -1) == 0


# ---- attention behind a shared prefix ----------------------------------------------


def _paged(**kw):
    c = _lib.AnnPaged(k=FAKE, v=FAKE, k_page=6 * 16 * 128, k_head=16 * 128, k_slot=128,
                      v_page=6 * 16 * 128, v_head=16 * 128, v_slot=128, table=FAKE, table_row=8,
                      starts=FAKE, lens=FAKE, pages=64, page_size=16, heads=6, head_dim=128, seqs=4,
                      cols=8, rows=4)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def _prefix(**kw):
    x = _lib.AnnPagedPrefix(groups=FAKE, table=FAKE, row=8, lens=FAKE, count=2, cols=8)
    for k, v in kw.items():
        setattr(x, k, v)
    return x


def _shared(c, x, heads=6, q=FAKE, row=768, head=128, scale=0.1, window=0, out=FAKE << 1, ws=FAKE << 2, nws=1 << 40):
    return _lib.lib().ann_op_paged_attention_shared(c, x, q, row, head, heads, scale, window, out, None, ws, nws, None)


@pytest.mark.parametrize("kw,msg", [
    ({"count": -1}, "shape"), ({"count": 65536}, "65535"), ({"cols": -1}, "shape"), ({"cols": (1 << 26) + 1}, "2^30"),
    ({"groups": None}, "null"), ({"table": None}, "null"), ({"lens": None}, "null"),
])
def test_prefixes_refused(kw, msg):
    assert _shared(_paged(), _prefix(**kw)) == _lib.ANN_E_ARG
    assert _said(msg), _lib.lib().ann_last_error()
    assert _lib.lib().ann_op_paged_attention_shared_ws_bytes(_paged(), _prefix(**kw), 6, 0) == 0


@pytest.mark.parametrize("cache,kw,msg", [
    ({"head_dim": 96}, {}, "head_dim"), ({"page_size": 24}, {}, "power of two"), ({"k": None}, {}, "null"),
    ({"k": FAKE + 8}, {}, "aligned"), ({"starts": None}, {}, "null"), ({}, {"heads": 8}, "8 query heads over 6"),
    ({}, {"q": None}, "null"), ({}, {"q": FAKE + 2}, "aligned"), ({}, {"scale": float("nan")}, "finite"),
    ({}, {"window": -1}, "window"), ({}, {"out": None}, "out is null"), ({}, {"out": (FAKE << 1) + 4}, "aligned"),
    ({}, {"out": FAKE + 16}, "overlaps"), ({"rows": 1 << 22}, {"heads": 600}, "2^30"),
])
def test_attention_shared_refused(cache, kw, msg):
    assert _shared(_paged(**cache), _prefix(), **kw) == _lib.ANN_E_ARG
    assert _said(msg), _lib.lib().ann_last_error()


def test_attention_shared_needs_its_workspace():
    assert _shared(_paged(), None) == _lib.ANN_E_ARG and _said("prefix is null")
    c, x = _paged(seqs=64, rows=64, cols=640, table_row=640), _prefix(cols=512, row=512)
    n = _lib.lib().ann_op_paged_attention_shared_ws_bytes(c, x, 6, 0)
    assert n > 0
    assert _shared(c, x, nws=n - 1) not in (0, _lib.ANN_E_ARG) and _said("workspace")
    assert _shared(c, x, ws=None, nws=n) == _lib.ANN_E_ARG


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(6, 6), (8, 2), (64, 8)])
def test_workspace_of_shared_is_bounded(heads, kv_heads, dim):
    """Three kinds of parts of 2^28 bytes at most each, whatever the tables' widths, but for
    one part of each row."""
    for seqs in (1, 64, 1024, 65535):
        for rows in (1, 17, seqs, seqs + 511, 65536):
            for count in (0, 1, 7, 4096):
                for entries in (16, 1 << 14, 1 << 20, 1 << 30):
                    c = _paged(seqs=seqs, rows=rows, cols=entries // 16, table_row=entries // 16, heads=kv_heads,
                               head_dim=dim, pages=1 << 20)
                    x = _prefix(count=count, cols=entries // 16, row=entries // 16)
                    n = _lib.lib().ann_op_paged_attention_shared_ws_bytes(c, x, heads, 0)
                    one = rows * heads * (dim + 2) * 4
                    assert n <= 3 * max(1 << 28, one), (seqs, rows, count, entries, n)


def test_more_work_groups_than_a_launch_takes_are_refused():
    """2^26 rows behind a prefix would be joined by 2^24 work-groups of 256 threads."""
    c = _paged(seqs=65535, rows=1 << 26, cols=64, table_row=64, heads=1, head_dim=64, k_page=1024, v_page=1024, k_head=1024,
               v_head=1024, k_slot=64, v_slot=64)
    rc = _shared(c, _prefix(cols=64, row=64), heads=1, row=64, head=64, out=FAKE << 2, ws=FAKE << 3)
    assert rc not in (0, _lib.ANN_E_ARG) and _said("configuration")


# ---- tokens from logits ------------------------------------------------------------


def _rows(**kw):
    r = _lib.AnnLogitRows(logits=_where(0), stride=100, u=_where(1), temperature=None, top_k=None, top_p=None,
                          min_p=None, temperature_all=1.0, top_k_all=0, top_p_all=1.0, min_p_all=0.0, rows=4,
                          cols=100, dtype=0, ids=_where(2), logprob=_where(3))
    for k, v in kw.items():
        setattr(r, k, v)
    return r


@pytest.mark.parametrize("kw,msg", [
    ({"rows": -1}, "shape"), ({"cols": 0}, "shape"), ({"cols": (1 << 20) + 1}, "2^20"), ({"dtype": 7}, "dtype"),
    ({"dtype": -1}, "dtype"), ({"logits": None}, "null"), ({"u": None}, "null"), ({"ids": None}, "null"),
    ({"temperature_all": -0.5}, "temperature"), ({"temperature_all": float("nan")}, "temperature"),
    ({"top_p_all": -0.1}, "top_p"), ({"top_p_all": float("nan")}, "top_p"), ({"min_p_all": -1.0}, "min_p"),
    ({"min_p_all": float("nan")}, "min_p"), ({"top_k_all": -1}, "top_k"), ({"logits": _where(0) + 2}, "aligned"),
    ({"ids": _where(0) + 396}, "ids overlaps logits"), ({"ids": _where(0) + 400}, "ids overlaps logits"),
    ({"ids": _where(1) - 12}, "ids overlaps u"), ({"logprob": _where(2) + 8}, "logprob overlaps ids"),
    ({"logprob": _where(5), "top_k": _where(5)}, "logprob overlaps top_k"),
    ({"ids": _where(5), "min_p": _where(5) + 12}, "ids overlaps min_p"),
])
def test_rows_refused(kw, msg):
    assert _lib.lib().ann_op_sample_logits(_rows(**kw), None) == _lib.ANN_E_ARG
    assert _said(msg), _lib.lib().ann_last_error()


# ---- with nothing to do, and from Python ---------------------------------------------


def test_nothing_to_do_launches_nothing():
    assert _lib.lib().ann_op_sample_logits(_rows(rows=0, logits=None, u=None, ids=None), None) == 0
    assert _shared(_paged(rows=0), _prefix()) == 0


def test_structs_pack_as_they_lie():
    """``from_values`` writes what the fields read."""
    t = _lib.AnnPagedTable.from_values(*range(1, 12))
    assert [getattr(t, k) for k, _ in t._fields_] == list(range(1, 12))
    x = _lib.AnnPagedPrefix.from_values(*range(1, 7))
    assert [getattr(x, k) for k, _ in x._fields_] == list(range(1, 7))
    r = _lib.AnnLogitRows.from_values(*range(1, 17))
    assert [getattr(r, k) for k, _ in r._fields_] == list(range(1, 17))
    for c, n in ((_lib.AnnPagedTable, 72), (_lib.AnnPagedPrefix, 40), (_lib.AnnLogitRows, 104)):
        assert ctypes.sizeof(c) == n


def test_python_layer_needs_gpu_tensors():
    i = torch.zeros(1, 2, dtype=torch.int32)
    q = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    c = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    for call in (lambda: paged.assign(i, i[0, :1], i[0, :1], i[0], 16, 4),
                 lambda: paged.release(i, i[0, :1], i[0], 16),
                 lambda: paged.attention_shared(q, c, c, i, i[0], i[0, :1], i[0], i, i[0, :1], 0.1),
                 lambda: kernels.sample_logits(torch.zeros(1, 5), torch.zeros(1)),
                 lambda: kernels.sample_logits([1.0], torch.zeros(1))):
        with pytest.raises(ValueError, match="GPU tensor"):
            call()
