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

``assign`` gives a step's tokens their pages and rows and ``release`` takes pages back, so
the tables too are made without the host; ``attention_shared`` reads entries that
sequences have in common once::

    a = paged.assign(table, lens, new, refs, page_size, rows)
    q = paged.append(q, k, v, cs, sn, k_cache, v_cache, a.table, a.starts, a.lens)
    y = paged.attention_shared(q, k_cache, v_cache, a.table, a.starts, a.lens, groups, prefix_table, prefix_lens, 0.1)
    ids = kernels.sample_logits(logits, u, temperature=0.8, top_p=0.95)
    table, refs = paged.release(a.table, lens, a.refs, page_size)

(model.py:244-254 for one layer; the reference recomputes the context and has
no cache.)  ``table``, ``starts`` and ``lens`` are int32 GPU tensors that the
host does not look at, so every call can be captured into a graph and replayed
with new values.  An id that is no page is never written to and reads page 0;
a length past the table ends at it; ``starts`` must not fall.  Rows from
``starts[-1]`` on belong to no sequence and are left as they were.

The page size is a power of two from 16 to 1024, the head dimension 64 or 128.
The cache may have any strides over page, head and slot (multiples of 8, slots at
most 2^25 elements apart), and a head of it serves ``heads / kv_heads`` query heads behind one another.
Tensors live on one GPU, which need not be the current device; the work goes to
its current stream.

A page that a call writes belongs to one sequence, and no two of its rows share
memory (an expanded cache can be read only); pages that are only read may be shared
by several (a common prefix).

These calls serve: autograd does not see them, and their results require no gradient.
"""

from typing import NamedTuple

import torch

from . import _lib
from ._stream import on_device

_BF16, _I32, _F32 = torch.bfloat16, torch.int32, torch.float32
_Tensor, _empty_strided, _parts = torch.Tensor, torch.empty_strided, torch.unsafe_split_with_sizes
_paged, _qk_rows = _lib.AnnPaged.from_values, _lib.AnnQkRows.from_values


def _refuse(name, x, dtype, dim, d):
    if not isinstance(x, _Tensor) or x.get_device() < 0:
        raise ValueError(f"{name}: expected a GPU tensor")
    if x.dtype != dtype:
        raise TypeError(f"{name}: {x.dtype}, expected {dtype}")
    if x.dim() != dim:
        raise ValueError(f"{name}: expected {dim} dimensions, got shape {tuple(x.shape)}")
    raise ValueError(f"{name} is on {x.device}, not on cuda:{d}")


def _check(name, x, dtype, dim, d):
    if not isinstance(x, _Tensor) or x.get_device() != d or x.dtype is not dtype or x.dim() != dim:
        _refuse(name, x, dtype, dim, d)


def _pool(k_cache):
    """The GPU that the cache is on."""
    if not isinstance(k_cache, _Tensor) or k_cache.get_device() < 0:
        raise ValueError("k_cache: expected a GPU tensor")
    return k_cache.get_device()


def _rows(name, x, d):
    """(rows, heads, head_dim) bf16 that 16-byte loads can read, x or a copy; and
    its address, row and head stride."""
    _check(name, x, _BF16, 3, d)
    a, b, c = x.stride()
    at = x.data_ptr()
    if c != 1 or (a | b) & 7 or at & 15:
        x = x.clone(memory_format=torch.contiguous_format)
        a, b, c = x.stride()
        at = x.data_ptr()
    return x, at, a, b


def _column(name, x, n, d):
    _check(name, x, _I32, 1, d)
    if x.shape[0] != n:
        raise ValueError(f"{name} has {x.shape[0]} elements, expected {n}")
    return x if x.is_contiguous() else x.contiguous()


def _new(shape, dtype, device):
    """A contiguous tensor (by its strides: a quarter faster than torch.empty)."""
    if len(shape) == 3:
        strides = (shape[1] * shape[2], shape[2], 1)
    else:
        strides = (shape[1], 1) if len(shape) == 2 else (1,)
    return _empty_strided(shape, strides, dtype=dtype, device=device)


def _out(out, like):
    _check("out", out, _BF16, 3, like.get_device())
    if out.shape != like.shape or not out.is_contiguous():
        raise ValueError(f"out must be contiguous {tuple(like.shape)}")
    return out


def _cache(d, k_cache, v_cache, table, lens, starts=None, rows=0):
    """AnnPaged of the call, (sequences, table columns, kv heads, page size, head
    dimension), the table, and what has to outlive the call."""
    # one expression for what is nearly always so; what is not is named below
    if not (k_cache.dtype is _BF16 and k_cache.dim() == 4 and isinstance(table, _Tensor)
            and table.dtype is _I32 and table.dim() == 2 and table.get_device() == d
            and isinstance(lens, _Tensor) and lens.dtype is _I32 and lens.dim() == 1
            and lens.get_device() == d):
        _check("k_cache", k_cache, _BF16, 4, d)
        _check("table", table, _I32, 2, d)
        _check("lens", lens, _I32, 1, d)
    shape = k_cache.shape
    pages, heads, page, dim = shape
    S, cols = table.shape
    ts, tc = table.stride()
    if tc != 1 and cols > 1:
        table = table.contiguous()
        ts = cols
    if lens.shape[0] != S or not lens.is_contiguous():
        lens = _column("lens", lens, S, d)
    kp, kh, ks, kd = k_cache.stride()
    if v_cache is None:
        v, vp, vh, vs, vd = 0, 0, 0, 0, 1
    else:
        _check("v_cache", v_cache, _BF16, 4, d)
        if v_cache.shape != shape:
            raise ValueError(f"v_cache {tuple(v_cache.shape)} differs from {tuple(shape)}")
        v = v_cache.data_ptr()
        vp, vh, vs, vd = v_cache.stride()
    if kd != 1 or vd != 1:
        raise ValueError("the caches' head dimension must be contiguous")
    first = 0
    if starts is not None:
        starts = _column("starts", starts, S + 1, d)
        first = starts.data_ptr()
    c = _paged(k_cache.data_ptr(), v, kp, kh, ks, vp, vh, vs, table.data_ptr(), ts, first,
               lens.data_ptr(), pages, page, heads, dim, S, cols, rows)
    return c, (S, cols, heads, page, dim), table, (lens, starts)


def _weight(name, weight, S, cap, d):
    _check(name, weight, _F32, 2, d)
    if weight.shape != (S, cap):
        raise ValueError(f"{name} {tuple(weight.shape)} must be (sequences, table entries) = {(S, cap)}")
    return weight if cap <= 1 or weight.stride(1) == 1 else weight.contiguous()


def _window(window):
    """As the C ABI's 32 bits hold it: 2^30 is past every table, -1 is refused there."""
    return window if 0 <= window < 1 << 30 else -1 if window < 0 else 1 << 30


def _angles(name, x, dim, d):
    _check(name, x, _F32, 2, d)
    n, m = x.shape
    if m != dim // 4 or n < 1:
        raise ValueError(f"{name} {tuple(x.shape)} must be (positions, {dim // 4})")
    if not x.is_contiguous() or x.data_ptr() & 15:
        x = x.clone(memory_format=torch.contiguous_format)
    return x


def append(q, k, v, cs, sn, k_cache, v_cache, table, starts, lens, pos=None, eps=1e-6, out=None):
    """New tokens enter the cache: queries ``q`` (rows, heads, head_dim) and keys
    ``k`` (rows, kv_heads, head_dim) normalised and rotated as
    ``kernels.qk_norm_rope`` does, keys and values ``v`` to their entries.
    -> the queries, contiguous (``out``, where given; it may be ``q``).

    A token's position is its entry, or ``pos`` (rows,) int32 (after an eviction
    the positions run ahead of the entries); the tables ``cs``, ``sn`` (positions,
    head_dim / 4) end there (a position outside takes their nearest row)."""
    d = _pool(k_cache)
    q, qp, qt, qh = _rows("q", q, d)
    k, kp, kt, kh = _rows("k", k, d)
    v, vp, vt, vh = _rows("v", v, d)
    N, H, D = q.shape
    c, (S, _, heads, _, dim), table, keep = _cache(d, k_cache, v_cache, table, lens, starts, N)
    if k.shape != (N, heads, dim) or v.shape != (N, heads, dim) or D != dim:
        raise ValueError(f"k {tuple(k.shape)}, v {tuple(v.shape)} must be (rows, kv_heads, head_dim) "
                         f"= {(N, heads, dim)} beside q {tuple(q.shape)}")
    cs, sn = _angles("cs", cs, D, d), _angles("sn", sn, D, d)
    if cs.shape != sn.shape:
        raise ValueError(f"cs {tuple(cs.shape)} and sn {tuple(sn.shape)} differ")
    out = _new((N, H, D), _BF16, q.device) if out is None else _out(out, q)
    at = 0
    if pos is not None:
        pos = _column("pos", pos, N, d)
        at = pos.data_ptr()
    a = _qk_rows(qp, kp, vp, 0, 0, out.data_ptr(), 0, 0, qt, qh, 0, kt, kh, 0, vt, vh, 0, 0, 0, 0, 0, 0,
                 cs.data_ptr(), sn.data_ptr(), at, 1, 0, cs.shape[0], 1, N, H, heads, D,
                 _lib.DTYPE_BF16, eps)
    rc = on_device(d, _lib.lib().ann_op_paged_append, c, a)
    if rc:
        _lib.check(rc)
    return out


def _queries(q, k_cache, v_cache, table, starts, lens):
    d = _pool(k_cache)
    rows = _rows("q", q, d)
    N, H, D = rows[0].shape
    if rows[2] > 1 << 25 or rows[3] * H > 1 << 28:   # a tile's offsets are 32 bits
        rows = _rows("q", rows[0].clone(memory_format=torch.contiguous_format), d)
    c, sizes, table, keep = _cache(d, k_cache, v_cache, table, lens, starts, N)
    if D != sizes[4]:
        raise ValueError(f"q {tuple(q.shape)}: the cache's head dimension is {sizes[4]}")
    return rows, N, H, D, d, c, sizes, (table, keep)


def attention(q, k_cache, v_cache, table, starts, lens, scale, window=0, want_lse=False, out=None):
    """Attention of new tokens ``q`` (rows, heads, head_dim), which ``append`` has
    entered, over their sequences' caches: the token at entry ``e`` sees the
    entries ``j <= e`` and, with ``window`` > 0, ``e - j < window``.
    -> (rows, heads, head_dim) bf16 (``out``, where given); with ``want_lse`` also
    (rows, heads) fp32, the log of each softmax sum.  A token that sees nothing
    gets 0 and -inf.  ``out`` may be ``q``.  Scores, softmax and sums are fp32; the
    weights enter the product with the values in two bf16 halves where a sequence
    has up to 16 rows (tokens times shared heads) or the call no more tokens than
    sequences, else in bf16, as in the framework's other attention."""
    (q, qp, qt, qh), N, H, D, d, c, _, keep = _queries(q, k_cache, v_cache, table, starts, lens)
    device = q.device
    out = _new((N, H, D), _BF16, device) if out is None else _out(out, q)
    window = _window(window)
    L = _lib.lib()
    nws = L.ann_op_paged_attention_ws_bytes(c, H, window)
    lse = _new((N, H), _F32, device) if want_lse else None
    ws = _new((nws,), torch.uint8, device) if nws else None
    rc = on_device(d, L.ann_op_paged_attention, c, qp, qt, qh, H, scale, window,
                   out.data_ptr(), lse.data_ptr() if want_lse else None,
                   ws.data_ptr() if nws else None, nws)
    if rc:
        _lib.check(rc)
    return (out, lse) if want_lse else out


def attention_shared(q, k_cache, v_cache, table, starts, lens, groups, prefix_table, prefix_lens, scale,
                     window=0, want_lse=False, out=None):
    """``attention`` of a batch whose sequences begin with the same entries: those of
    group ``g``, sequences ``groups[g] .. groups[g + 1] - 1``, with the first
    ``prefix_lens[g]`` entries of ``prefix_table[g]``.  Their own tables name the same
    pages there (or copies: of the page that a prefix ends in, say).  -> what ``attention`` gives.

    ``groups`` (groups + 1,), ``prefix_table`` (groups, columns) and ``prefix_lens`` (groups,)
    are int32 GPU tensors that the host does not look at; ``groups`` must not fall, and sequences of no
    group share nothing.  A prefix is read once for the tokens of all its sequences with up
    to 16 new ones; a sequence of more is on its own.  Where the tables are so narrow, or a
    window leaves so little of a prefix, that this saves too little, all goes as in
    ``attention``; else the weights enter the product with the values in two bf16 halves for
    sequences of up to 16 new tokens, in bf16 for those of more.  ``out`` may be ``q``."""
    (q, qp, qt, qh), N, H, D, d, c, (S, _, _, page, _), keep = _queries(q, k_cache, v_cache, table, starts, lens)
    _check("prefix_table", prefix_table, _I32, 2, d)
    count, cols = prefix_table.shape
    if cols > 1 and prefix_table.stride(1) != 1:
        prefix_table = prefix_table.contiguous()
    groups, prefix_lens = _column("groups", groups, count + 1, d), _column("prefix_lens", prefix_lens, count, d)
    x = _lib.AnnPagedPrefix.from_values(groups.data_ptr(), prefix_table.data_ptr(), prefix_table.stride(0),
                                        prefix_lens.data_ptr(), count, cols)
    device = q.device
    out = _new((N, H, D), _BF16, device) if out is None else _out(out, q)
    window = _window(window)
    L = _lib.lib()
    nws = L.ann_op_paged_attention_shared_ws_bytes(c, x, H, window)
    lse = _new((N, H), _F32, device) if want_lse else None
    ws = _new((nws,), torch.uint8, device) if nws else None
    rc = on_device(d, L.ann_op_paged_attention_shared, c, x, qp, qt, qh, H, scale, window, out.data_ptr(),
                   lse.data_ptr() if want_lse else None, ws.data_ptr() if nws else None, nws)
    if rc:
        _lib.check(rc)
    return (out, lse) if want_lse else out


def attention_weight(q, lse, k_cache, table, starts, lens, weight, scale, window=0, out=None):
    """``weight`` (sequences, table entries) fp32 plus the attention weight that
    each entry receives from the new tokens ``q``, over all their heads; ``lse`` as
    ``attention`` returned it for the same tokens.  -> a new tensor, or ``out``,
    which may be ``weight``.  Entries behind a sequence keep their weight."""
    (q, qp, qt, qh), N, H, _, d, c, (S, cols, _, page, _), keep = _queries(q, k_cache, None, table,
                                                                           starts, lens)
    _check("lse", lse, _F32, 2, d)
    if lse.shape != (N, H):
        raise ValueError(f"lse {tuple(lse.shape)} must be {(N, H)}")
    if not lse.is_contiguous():
        lse = lse.contiguous()
    weight = _weight("weight", weight, S, cols * page, d)
    if out is None:
        out = _new((S, cols * page), _F32, q.device)
    elif _weight("out", out, S, cols * page, d) is not out:
        raise ValueError("out: rows must be contiguous")
    rc = on_device(d, _lib.lib().ann_op_paged_weight, c, qp, qt, qh, H, lse.data_ptr(), scale, _window(window),
                   weight.data_ptr(), weight.stride(0), out.data_ptr(), out.stride(0), None, 0)
    if rc:
        _lib.check(rc)
    return out


def evict(k_cache, v_cache, table, lens, weight, keep, recent=0, out_table=None):
    """Cut every sequence to ``keep`` entries: its last ``recent`` stay and, of the
    others, those of the largest ``weight`` (at equal weights the lower entry; a NaN
    is below every number).  They keep their order and move to entries 0 .. of
    the pages in ``out_table`` (sequences, pages), or in place.
    -> (index, lens, weight): the entry that each came from (sequences, keep)
    int32, -1 behind them; the new lengths; their weights, 0 behind them.

    ``out_table`` names pages that ``table`` does not, each once (or is ``table``); in
    place, no two sequences share a page.  ``recent`` is at most ``keep``.  Keys hold
    their rotation, so later tokens go on at their own positions: pass ``pos`` to
    ``append``."""
    d = _pool(k_cache)
    c, (S, cols, _, page, _), table, held = _cache(d, k_cache, v_cache, table, lens)
    cap = cols * page
    weight = _weight("weight", weight, S, cap, d)
    if out_table is None:
        out_table = table
    else:
        _check("out_table", out_table, _I32, 2, d)
        if out_table.shape[0] != S:
            raise ValueError(f"out_table {tuple(out_table.shape)} must have {S} rows")
        if out_table.shape[1] > 1 and out_table.stride(1) != 1:
            out_table = out_table.contiguous()
    keep, recent = int(keep), int(recent)
    if keep < 1 or not 0 <= recent <= keep:
        raise ValueError(f"keep={keep} must be at least 1 and recent={recent} lie in [0, keep]")
    if keep > out_table.shape[1] * page:
        raise ValueError(f"{out_table.shape[1]} pages of {page} do not hold keep={keep} entries")
    device = k_cache.device
    index = _new((S, keep), _I32, device)
    left = _new((S,), _I32, device)
    out = _new((S, cap), _F32, device)
    rc = on_device(d, _lib.lib().ann_op_paged_evict, c, out_table.data_ptr(), out_table.stride(0),
                   out_table.shape[1], weight.data_ptr(), weight.stride(0), keep, recent,
                   index.data_ptr(), left.data_ptr(), out.data_ptr(), cap)
    if rc:
        _lib.check(rc)
    return index, left, out


class Assigned(NamedTuple):
    """A step's tables and row maps, as ``assign`` made them."""
    table: torch.Tensor    # (sequences, columns) int32
    refs: torch.Tensor     # (pages,) int32
    starts: torch.Tensor   # (sequences + 1,) int32; these four lie behind one another in one allocation
    lens: torch.Tensor     # (sequences,) int32
    seq: torch.Tensor      # (rows,) int32: the sequence of each row, -1 behind the last
    pos: torch.Tensor      # (rows,) int32: its entry, -1 behind
    slot: torch.Tensor     # (rows,) int64: page * page_size + place in the page, -1 behind


def _table_args(table, lens, refs, page_size, out, refs_out):
    """AnnPagedTable of the call, its outputs, (device, sequences), and what has to
    outlive the call."""
    if not isinstance(table, _Tensor) or table.get_device() < 0:
        raise ValueError("table: expected a GPU tensor")
    d = table.get_device()
    _check("table", table, _I32, 2, d)
    S, cols = table.shape
    _check("refs", refs, _I32, 1, d)
    device = table.device
    if out is None:
        if cols > 1 and table.stride(1) != 1:
            table = table.contiguous()
        out = _new((S, cols), _I32, device)
    else:
        _check("out", out, _I32, 2, d)
        if out.shape != (S, cols) or (cols > 1 and out.stride(1) != 1):
            raise ValueError(f"out {tuple(out.shape)} must be {(S, cols)}, rows contiguous")
        if cols > 1 and table.stride(1) != 1:
            table = table.contiguous()
    pages = refs.shape[0]
    if refs_out is None:
        refs_out = _new((pages,), _I32, device)
    else:
        _check("refs_out", refs_out, _I32, 1, d)
        if refs_out.shape[0] != pages or not refs_out.is_contiguous():
            raise ValueError(f"refs_out must be contiguous, {pages} elements")
    refs = _column("refs", refs, pages, d)
    lens = _column("lens", lens, S, d)
    t = _lib.AnnPagedTable.from_values(
        table.data_ptr(), table.stride(0), lens.data_ptr(), refs.data_ptr(), out.data_ptr(), out.stride(0),
        refs_out.data_ptr(), pages, _page_size(page_size), S, cols)
    return t, out, refs_out, d, S, (table, lens, refs)


def _page_size(n):
    """As the C ABI's 32 bits hold it: what is no page size is refused there."""
    return n if 0 <= n < 1 << 30 else 0


def assign(table, lens, new, refs, page_size, rows, out=None, refs_out=None, lens_out=None):
    """Pages for the next step: sequence ``s`` is to grow by ``new[s]`` tokens.
    -> ``Assigned``: the table with a page for every new entry, the pages' counts,
    ``starts`` and ``lens`` of the step as ``append`` and ``attention`` take them, and
    for each of its ``rows`` rows the sequence, the entry and the slot in the cache.

    ``refs`` (pages,) int32 counts the tables that name each page; a page is free
    where that is not above 0.  A column that names no page (-1) takes one once its entries
    are asked for, free pages in ascending order, and keeps it until ``release``: the
    same call again finds it there.  Sequences are served in order, whole or
    not at all: one whose entries do not fit its table row, or for which (with all
    asked for before it) the pages or the ``rows`` do not last, gets none and keeps
    its length.  One that needs no page needs only the rows.

    ``out``, ``refs_out`` and ``lens_out`` may be ``table``, ``refs`` and ``lens``: a step in
    place, which a captured graph replays on its own results."""
    t, out, refs_out, d, S, keep = _table_args(table, lens, refs, page_size, out, refs_out)
    new = _column("new", new, S, d)
    rows = int(rows)
    if not 0 <= rows <= 1 << 30:
        raise ValueError(f"rows={rows} must lie in [0, 2^30]")
    device = out.device
    # one allocation and its parts: half the time of four
    if lens_out is None:
        starts, lens_out, seq, pos = _parts(_new((2 * (S + rows) + 1,), _I32, device), (S + 1, S, rows, rows))
    else:
        _check("lens_out", lens_out, _I32, 1, d)
        if lens_out.shape[0] != S or not lens_out.is_contiguous():
            raise ValueError(f"lens_out must be contiguous, {S} elements")
        starts, seq, pos = _parts(_new((S + 2 * rows + 1,), _I32, device), (S + 1, rows, rows))
    slot = _new((rows,), torch.int64, device)
    L = _lib.lib()
    nws = L.ann_op_paged_assign_ws_bytes(t, rows)
    ws = _new((nws,), torch.uint8, device) if nws else None
    rc = on_device(d, L.ann_op_paged_assign, t, new.data_ptr(), rows, starts.data_ptr(), lens_out.data_ptr(),
                   seq.data_ptr(), pos.data_ptr(), slot.data_ptr(), ws.data_ptr() if nws else None, nws)
    if rc:
        _lib.check(rc)
    return Assigned(out, refs_out, starts, lens_out, seq, pos, slot)


def release(table, lens, refs, page_size, out=None, refs_out=None):
    """The pages behind each sequence's first ``lens[s]`` entries (0: of a sequence
    that ended; fewer: of one cut back) are given back.  -> (table, refs): -1 in their columns, one less
    in their counts.  ``out`` and ``refs_out`` may be ``table`` and ``refs``."""
    t, out, refs_out, d, _, keep = _table_args(table, lens, refs, page_size, out, refs_out)
    rc = on_device(d, _lib.lib().ann_op_paged_release, t)
    if rc:
        _lib.check(rc)
    return out, refs_out
