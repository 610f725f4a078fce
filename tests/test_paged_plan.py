"""How a call's own keys are cut, as the workspace it asks for shows: none for whole sequences. The rule goes by the table's
width and the number of sequences and key/value heads; a card of 256 CUs, as where there is none."""
import ctypes

import pytest

from test_paged_host import _attention


def _pieces(batch, heads, keys, **kw):
    from lbw_amd import _lib
    width = keys // 16
    p = _attention(batch=batch, q_heads=heads, k_heads=heads, **{"cache.page_size": 16, "cache.table_width": width,
                                                                 "cache.table_stride": width, **kw})
    return _lib.load().lbw_attention_paged_workspace_size(ctypes.byref(p)) > 0


@pytest.mark.parametrize("batch", list(range(33, 49)))
def test_sequences_for_one_to_one_and_a_half_workgroups_a_cu_are_cut_alike(batch):
    """264 to 384 sequences x key/value heads: pieces above 1500 keys, for each number of them."""
    assert [_pieces(batch, 8, n) for n in (496, 1200, 1488, 1504, 1696, 2400, 3200, 4000)] == 3 * [False] + 5 * [True]


def test_fewer_and_more_of_them():
    assert not _pieces(32, 8, 4336) and _pieces(32, 8, 4352 + 16)        # one a CU: 4350
    assert not _pieces(50, 8, 3488) and _pieces(50, 8, 3504)             # more than three for two CUs: 3500
    assert not _pieces(1, 8, 1136) and _pieces(1, 8, 1168)
