"""What attention over a paged cache asks for: by the rows there are and a fixed
bound, not by how wide its table is."""

import pytest

from attention_nn_amd import _lib

FAKE = 1 << 40


def _bytes(seqs, cols, rows, heads, kv_heads, dim, page, window=0):
    c = _lib.AnnPaged(k=FAKE, v=FAKE, k_page=kv_heads * page * dim, k_head=page * dim, k_slot=dim,
                      v_page=kv_heads * page * dim, v_head=page * dim, v_slot=dim, table=FAKE, table_row=cols,
                      starts=FAKE, lens=FAKE, pages=1 << 20, page_size=page, heads=kv_heads, head_dim=dim, seqs=seqs,
                      cols=cols, rows=rows)
    return _lib.lib().ann_op_paged_attention_ws_bytes(c, heads, window)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(6, 6), (8, 2), (64, 8)])
def test_bounded(heads, kv_heads, dim):
    """Both kinds of rows 2^28 bytes at most, whatever the table's width."""
    for seqs in (1, 3, 64, 1024, 65535):
        for rows in (1, 16, 17, seqs, seqs + 1, seqs + 511, 65536):
            for entries in (1024, 1 << 14, 1 << 17, 1 << 20, 1 << 30):
                for window in (0, 384, 5000):
                    n = _bytes(seqs, entries // 1024, rows, heads, kv_heads, dim, 1024, window)
                    assert n <= 2 << 28, (seqs, rows, entries, window, n)


def test_one_slot_a_row():
    """A mixed batch of decoding sequences takes a slot for each of its rows, where 16 a
    sequence are more; a step of a few sequences is bounded by nothing."""
    slot = (128 + 2) * 4
    for seqs, rows in ((1024, 1535), (64, 100)):
        n = _bytes(seqs, 64, rows, 8, 8, 128, 1024)
        assert n and n % (rows * 8 * slot) == 0 and n <= rows * 8 * slot * (64 + 64)
    assert _bytes(16, 8, 16, 6, 6, 128, 1024) == 16 * 6 * 5 * slot
    assert _bytes(1, 16, 2048, 12, 12, 128, 1024) == 2048 * 12 * 4 * slot


def test_more_work_groups_than_a_launch_takes_are_refused():
    """A mixed batch of 65,535 sequences of 512 cache heads would need 2^25 work-groups of
    256 threads: refused, not cut short."""
    c = _lib.AnnPaged(k=FAKE, v=FAKE, k_page=512 * 1024, k_head=1024, k_slot=64, v_page=512 * 1024, v_head=1024,
                      v_slot=64, table=FAKE, table_row=1, starts=FAKE, lens=FAKE, pages=1 << 20, page_size=16,
                      heads=512, head_dim=64, seqs=65535, cols=1, rows=65536)
    rc = _lib.lib().ann_op_paged_attention(c, FAKE, 512 * 64, 64, 512, 0.1, 0, FAKE << 1, None, FAKE, 1 << 40, None)
    assert rc not in (0, _lib.ANN_E_ARG) and "configuration" in _lib.lib().ann_last_error().decode()
