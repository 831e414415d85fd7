"""Which calls behind a shared prefix go as attention does, where a window leaves little of it
to read once or a launch would not hold them, by the workspace that a call asks for
(paged.attention_shared)."""

import pytest

from attention_nn_amd import _lib

FAKE = 1 << 40


def _bytes(seqs, rows, own, prefix, heads, kv_heads, dim, window, groups=1, page=64):
    """(of the call behind a prefix, of attention)."""
    L = _lib.lib()
    pcols = -(-prefix // page)
    cols = -(-(prefix + own) // page)
    c = _lib.AnnPaged(k=FAKE, v=FAKE, k_page=kv_heads * page * dim, k_head=page * dim, k_slot=dim,
                      v_page=kv_heads * page * dim, v_head=page * dim, v_slot=dim, table=FAKE, table_row=cols,
                      starts=FAKE, lens=FAKE, pages=1 << 16, page_size=page, heads=kv_heads, head_dim=dim, seqs=seqs,
                      cols=cols, rows=rows)
    x = _lib.AnnPagedPrefix(groups=FAKE, table=FAKE, row=pcols, lens=FAKE, count=groups, cols=pcols)
    return L.ann_op_paged_attention_shared_ws_bytes(c, x, heads, window), L.ann_op_paged_attention_ws_bytes(c, heads, window)


@pytest.mark.parametrize("shape", [
    # seqs, rows, own, prefix, heads, window: nothing of the prefix is left behind the own entries, or little
    (8, 8, 256, 8192, (6, 6, 128), 384), (16, 16, 700, 16384, (12, 12, 128), 384), (64, 64, 256, 8192, (12, 12, 128), 384),
    (16, 16, 700, 16384, (6, 6, 128), 4096), (96, 96, 700, 4096, (12, 12, 128), 384), (16, 16, 2500, 16384, (12, 12, 128), 4096),
    (96, 96, 1500, 4096, (8, 2, 128), 2048), (64, 64, 256, 8192, (8, 8, 64), 1024),
    # many tokens a sequence
    (24, 2400, 64, 4096, (12, 12, 128), 2048),
])
def test_little_left_goes_as_attention(shape):
    seqs, rows, own, prefix, heads, window = shape
    shared, alone = _bytes(seqs, rows, own, prefix, *heads, window)
    assert shared == alone
    assert _bytes(seqs, rows, own, prefix, *heads, 0)[0] > 0     # without the window the prefix is shared


@pytest.mark.parametrize("shape", [
    (64, 64, 100, 8192, (12, 12, 128), 1024), (96, 96, 32, 4096, (12, 12, 128), 384), (16, 16, 700, 16384, (12, 12, 128), 4096),
    (64, 1024, 100, 4096, (6, 6, 128), 2048), (96, 96, 32, 4096, (8, 2, 128), 2048),
    (64, 64, 100, 8192, (12, 12, 128), 8192 + 128), (64, 64, 100, 8192, (12, 12, 128), 1 << 30),
])
def test_much_left_is_shared(shape):
    seqs, rows, own, prefix, heads, window = shape
    shared, _ = _bytes(seqs, rows, own, prefix, *heads, window)
    slot = rows * heads[0] * (heads[2] + 2) * 4
    assert shared >= 2 * slot and shared % slot == 0


def test_a_window_past_every_entry_is_none():
    for window in (8192 + 256, 1 << 30, (1 << 31) - 1):
        assert _bytes(64, 64, 256, 8192, 12, 12, 128, window)[0] == _bytes(64, 64, 256, 8192, 12, 12, 128, 0)[0]


def test_more_work_groups_than_a_launch_takes():
    """2^21 new tokens of 128 heads would take more work-groups behind a prefix than one
    launch has, and go as attention does."""
    shared, alone = _bytes(1024, 1 << 21, 4096, 8192, 128, 128, 64, 0)
    assert shared == alone
    shared, _ = _bytes(1024, 1 << 15, 4096, 8192, 128, 128, 64, 0)
    assert shared >= 2 * (1 << 15) * 128 * (64 + 2) * 4
