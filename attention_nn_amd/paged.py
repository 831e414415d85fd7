"""A key/value cache in pages that sequences of any lengths share, and the
attention of new tokens over it.

A layer's cache is two bf16 tensors (pages, kv_heads, page_size, head_dim);
entry ``e`` of sequence ``s`` is slot ``e % page_size`` of page
``table[s, e // page_size]``.  A call brings new tokens of every sequence behind
one another: those of sequence ``s`` are rows ``starts[s] .. starts[s + 1] - 1``,
and ``lens[s]`` counts the sequence's entries with these, so one call serves
prompts, chunks of prompts and single decoded tokens side by side::

    q = paged.append(q, k, v, cs, sn, k_cache, v_cache, table, starts, lens)
    y, lse = paged.attention(q, k_cache, v_cache, table, starts, lens, 0.1, want_lse=True)
    w = paged.attention_weight(q, lse, k_cache, table, starts, lens, w, 0.1)
    kept, lens, w = paged.evict(k_cache, v_cache, table, lens, w, keep=4096, recent=384)

(model.py:244-254 for one layer; the reference recomputes the context and has
no cache.)  ``table``, ``starts`` and ``lens`` are int32 GPU tensors that the
host does not look at, so every call can be captured into a graph and replayed
with new values.  An id that is no page is never written to and reads page 0;
a length past the table ends at it; ``starts`` must not fall.  Rows from
``starts[-1]`` on belong to no sequence and are left as they were.

The page size is a power of two from 16 to 1024, the head dimension 64 or 128.
The cache may have any strides over page, head and slot (multiples of 8), and a
head of it serves ``heads / kv_heads`` query heads behind one another.
Tensors live on one GPU, which need not be the current device; the work goes to
its current stream.
"""

import torch

from . import _lib

_BF16, _I32, _F32 = torch.bfloat16, torch.int32, torch.float32


def _check(name, x, dtype, dim, device=None):
    if not (isinstance(x, torch.Tensor) and x.is_cuda):
        raise ValueError(f"{name}: expected a GPU tensor")
    if x.dtype != dtype:
        raise TypeError(f"{name}: {x.dtype}, expected {dtype}")
    if x.dim() != dim:
        raise ValueError(f"{name}: expected {dim} dimensions, got shape {tuple(x.shape)}")
    if device is not None and x.device != device:
        raise ValueError(f"{name} is on {x.device}, not on {device}")
    return x


def _rows(name, x, device):
    """(rows, heads, head_dim) bf16 that 16-byte loads can read: x, or a copy."""
    _check(name, x, _BF16, 3, device)
    st = x.stride()
    if st[2] != 1 or (st[0] | st[1]) & 7 or x.data_ptr() & 15:
        x = x.clone(memory_format=torch.contiguous_format)
    return x


def _column(name, x, n, device):
    _check(name, x, _I32, 1, device)
    if x.shape[0] != n:
        raise ValueError(f"{name} has {x.shape[0]} elements, expected {n}")
    return x if x.stride(0) == 1 or n <= 1 else x.contiguous()


def _cache(k_cache, v_cache, table, lens, starts=None, rows=0):
    """AnnPaged of the call, and what has to outlive it."""
    device = _check("k_cache", k_cache, _BF16, 4).device
    pages, heads, page, dim = k_cache.shape
    _check("table", table, _I32, 2, device)
    S, cols = table.shape
    if cols > 1 and table.stride(1) != 1:
        table = table.contiguous()
    lens = _column("lens", lens, S, device)
    c = _lib.AnnPaged()
    keep = [table, lens]
    for name, x in (("k_cache", k_cache), ("v_cache", v_cache)):
        if x is None:
            continue
        _check(name, x, _BF16, 4, device)
        if tuple(x.shape) != (pages, heads, page, dim):
            raise ValueError(f"{name} {tuple(x.shape)} differs from {(pages, heads, page, dim)}")
        if x.stride(3) != 1:
            raise ValueError(f"{name}: the head dimension must be contiguous")
    c.k = k_cache.data_ptr()
    c.k_page, c.k_head, c.k_slot = k_cache.stride()[:3]
    if v_cache is not None:
        c.v = v_cache.data_ptr()
        c.v_page, c.v_head, c.v_slot = v_cache.stride()[:3]
    if starts is not None:
        starts = _column("starts", starts, S + 1, device)
        c.starts = starts.data_ptr()
        keep.append(starts)
    c.table, c.table_row, c.lens = table.data_ptr(), table.stride(0), lens.data_ptr()
    c.pages, c.page_size, c.heads, c.head_dim = pages, page, heads, dim
    c.seqs, c.cols, c.rows = S, cols, rows
    return c, device, keep


def _weight(name, weight, S, cap, device):
    _check(name, weight, _F32, 2, device)
    if tuple(weight.shape) != (S, cap):
        raise ValueError(f"{name} {tuple(weight.shape)} must be (sequences, table entries) = {(S, cap)}")
    return weight if weight.stride(1) == 1 or cap <= 1 else weight.contiguous()


def append(q, k, v, cs, sn, k_cache, v_cache, table, starts, lens, pos=None, eps=1e-6, out=None):
    """New tokens enter the cache: queries ``q`` (rows, heads, head_dim) and keys
    ``k`` (rows, kv_heads, head_dim) normalised and rotated as
    ``kernels.qk_norm_rope`` does, keys and values ``v`` to their entries.
    -> the queries, contiguous (``out``, where given).

    A token's position is its entry, or ``pos`` (rows,) int32 (after an eviction
    the positions run ahead of the entries); the tables ``cs``, ``sn`` (positions,
    head_dim / 4) end there (a position outside takes their nearest row)."""
    q = _rows("q", q, _check("k_cache", k_cache, _BF16, 4).device)
    N, H, D = q.shape
    c, device, keep = _cache(k_cache, v_cache, table, lens, starts, N)
    k, v = _rows("k", k, device), _rows("v", v, device)
    if tuple(k.shape) != (N, c.heads, c.head_dim) or k.shape != v.shape or D != c.head_dim:
        raise ValueError(f"k {tuple(k.shape)}, v {tuple(v.shape)} must be (rows, kv_heads, head_dim) "
                         f"= {(N, c.heads, c.head_dim)} beside q {tuple(q.shape)}")
    tabs = []
    for name, x in (("cs", cs), ("sn", sn)):
        _check(name, x, _F32, 2, device)
        if x.shape[1] != D // 4 or x.shape[0] < 1 or x.shape != cs.shape:
            raise ValueError(f"{name} {tuple(x.shape)} must be (positions, {D // 4})")
        tabs.append(x if x.is_contiguous() and not x.data_ptr() & 15 else
                    x.clone(memory_format=torch.contiguous_format))
    if out is None:
        out = torch.empty((N, H, D), dtype=_BF16, device=device)
    else:
        _check("out", out, _BF16, 3, device)
        if out.shape != q.shape or not out.is_contiguous():
            raise ValueError(f"out must be contiguous {tuple(q.shape)}")
    a = _lib.AnnQkRows()
    if pos is not None:
        pos = _column("pos", pos, N, device)
        a.pos, a.pos_each = pos.data_ptr(), 1
    a.q, a.k, a.v, a.q_out = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()
    a.q_stride[1], a.q_stride[2] = q.stride()[:2]
    a.k_stride[1], a.k_stride[2] = k.stride()[:2]
    a.v_stride[1], a.v_stride[2] = v.stride()[:2]
    a.cs, a.sn, a.table_rows = tabs[0].data_ptr(), tabs[1].data_ptr(), cs.shape[0]
    a.B, a.T, a.Hq, a.Hk, a.D, a.dtype, a.eps = 1, N, H, c.heads, D, _lib.DTYPE_BF16, eps
    _lib.launch(device, _lib.lib().ann_op_paged_append, c, a)
    return out


def _queries(q, k_cache, v_cache, table, starts, lens):
    q = _rows("q", q, _check("k_cache", k_cache, _BF16, 4).device)
    c, device, keep = _cache(k_cache, v_cache, table, lens, starts, q.shape[0])
    if q.shape[2] != c.head_dim:
        raise ValueError(f"q {tuple(q.shape)}: the cache's head dimension is {c.head_dim}")
    return q, c, device, keep


def attention(q, k_cache, v_cache, table, starts, lens, scale, window=0, want_lse=False, out=None):
    """Attention of new tokens ``q`` (rows, heads, head_dim), which ``append`` has
    entered, over their sequences' caches: the token at entry ``e`` sees the
    entries ``j <= e`` and, with ``window`` > 0, ``e - j < window``.
    -> (rows, heads, head_dim) bf16 (``out``, where given); with ``want_lse`` also
    (rows, heads) fp32, the log of each softmax sum.  A token that sees nothing
    gets 0 and -inf.  Weights enter the product with the values in bf16, as the
    framework's attention forms it; scores, softmax and sums are fp32."""
    q, c, device, keep = _queries(q, k_cache, v_cache, table, starts, lens)
    N, H, D = q.shape
    if out is None:
        out = torch.empty((N, H, D), dtype=_BF16, device=device)
    else:
        _check("out", out, _BF16, 3, device)
        if out.shape != q.shape or not out.is_contiguous():
            raise ValueError(f"out must be contiguous {tuple(q.shape)}")
    lse = torch.empty((N, H), dtype=_F32, device=device) if want_lse else None
    L = _lib.lib()
    nws = L.ann_op_paged_attention_ws_bytes(c, H, window)
    ws = torch.empty(nws, dtype=torch.uint8, device=device) if nws else None
    st = q.stride()
    _lib.launch(device, L.ann_op_paged_attention, c, q.data_ptr(), st[0], st[1], H, scale,
                window, out.data_ptr(), lse.data_ptr() if want_lse else None,
                ws.data_ptr() if nws else None, nws)
    return (out, lse) if want_lse else out


def attention_weight(q, lse, k_cache, table, starts, lens, weight, scale, window=0, out=None):
    """``weight`` (sequences, table entries) fp32 plus the attention weight that
    each entry receives from the new tokens ``q``, over all their heads; ``lse`` as
    ``attention`` returned it for the same tokens.  -> a new tensor, or ``out``,
    which may be ``weight``.  Entries behind a sequence keep their weight."""
    q, c, device, keep = _queries(q, k_cache, None, table, starts, lens)
    N, H, _ = q.shape
    _check("lse", lse, _F32, 2, device)
    if tuple(lse.shape) != (N, H):
        raise ValueError(f"lse {tuple(lse.shape)} must be {(N, H)}")
    lse = lse.contiguous()
    weight = _weight("weight", weight, c.seqs, c.cols * c.page_size, device)
    if out is None:
        out = torch.empty(weight.shape, dtype=_F32, device=device)
    elif _weight("out", out, c.seqs, c.cols * c.page_size, device) is not out:
        raise ValueError("out: rows must be contiguous")
    L = _lib.lib()
    nws = L.ann_op_paged_weight_ws_bytes(c, H)
    ws = torch.empty(nws, dtype=torch.uint8, device=device) if nws else None
    st = q.stride()
    _lib.launch(device, L.ann_op_paged_weight, c, q.data_ptr(), st[0], st[1], H, lse.data_ptr(),
                scale, window, weight.data_ptr(), weight.stride(0), out.data_ptr(),
                out.stride(0), ws.data_ptr() if nws else None, nws)
    return out


def evict(k_cache, v_cache, table, lens, weight, keep, recent=0, out_table=None):
    """Cut every sequence to ``keep`` entries: its last ``recent`` stay and, of the
    others, those of the largest ``weight`` (at equal weights the lower entry; a NaN
    is below every number).  They keep their order and move to entries 0 .. of
    the pages in ``out_table`` (sequences, pages), or in place.
    -> (index, lens, weight): the entry that each came from (sequences, keep)
    int32, -1 behind them; the new lengths; their weights, 0 behind them.

    ``out_table`` names pages that ``table`` does not (or is ``table``).  Keys hold
    their rotation, so later tokens go on at their own positions: pass ``pos`` to
    ``append``."""
    c, device, held = _cache(k_cache, v_cache, table, lens)
    cap = c.cols * c.page_size
    weight = _weight("weight", weight, c.seqs, cap, device)
    to = held[0] if out_table is None else _check("out_table", out_table, _I32, 2, device)
    if to.shape[0] != c.seqs:
        raise ValueError(f"out_table {tuple(to.shape)} must have {c.seqs} rows")
    if to.shape[1] > 1 and to.stride(1) != 1:
        to = to.contiguous()
    keep, recent = int(keep), int(recent)
    if keep < 1:
        raise ValueError(f"keep={keep} must be at least 1")
    if keep > to.shape[1] * c.page_size:
        raise ValueError(f"{to.shape[1]} pages of {c.page_size} do not hold keep={keep} entries")
    index = torch.empty((c.seqs, keep), dtype=_I32, device=device)
    left = torch.empty((c.seqs,), dtype=_I32, device=device)
    out = torch.empty((c.seqs, cap), dtype=_F32, device=device)
    _lib.launch(device, _lib.lib().ann_op_paged_evict, c, to.data_ptr(), to.stride(0), to.shape[1],
                weight.data_ptr(), weight.stride(0), keep, recent, index.data_ptr(),
                left.data_ptr(), out.data_ptr(), out.stride(0))
    return index, left, out
