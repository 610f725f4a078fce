"""Tables much wider than the lengths, as a captured serving step has them: the same results within the allowance, and to the
bit those of the narrow table where its columns are given."""
import pytest
import torch

import packed_ref as R
import paged_ref as P
from test_gpu_paged_attention import SCALE, Case, _i32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("prefix", [0, 40, 700, 2500])
@pytest.mark.parametrize("lens,hq,hk,page", [([1], 40, 8, 64), ([500, 0, 33], 12, 4, 16), ([40, 0, 5] * 12, 10, 2, 64),
                                             ([200, 17] * 20, 8, 8, 32), ([1900, 3, 64], 4, 1, 1024)])
def test_wide_tables_and_their_columns(prefix, lens, hq, hk, page):
    c = Case(lens, hq, hk, page, prefix=prefix, seed=len(lens))
    need = max(P.pages_of(n, page) for n in lens) + 1
    wide = torch.full((len(lens), 46800 // page), -9, dtype=torch.int32, device="cuda")
    wide[:, :need] = c.table
    sel = torch.arange(need, dtype=torch.int32).flip(0).expand(len(lens), hk, need).contiguous().cuda()
    for kw in ({}, {"selected": sel}):
        narrow = c.run(**kw)
        c.table = wide
        want, allow = P.attention(c.q, c.cache.k, c.cache.v, wide, lens, SCALE, c.prefix_table, prefix, kw.get("selected"))
        R.assert_within("wide", c.run(**kw), want, allow)
        c.table = wide[:, :need]
        assert not c.table.is_contiguous() or len(lens) == 1
        assert torch.equal(c.run(**kw), narrow)
        c.table = c.table.contiguous()


def test_one_row_for_every_query():
    """The tokens of a draft: one sequence's row of the table for all of them, not copied."""
    import lbw_amd
    c = Case([900], 12, 4, 16, seed=1)
    q = torch.randn(5, 12, 128, generator=torch.Generator().manual_seed(2)).to(c.q.dtype).cuda()
    lens = [896, 897, 898, 899, 900]
    rows = c.table.expand(5, -1)
    got = lbw_amd.attention_paged(q, c.cache, rows, _i32(lens))
    R.assert_within("out", got, *P.attention(q, c.cache.k, c.cache.v, rows.contiguous(), lens, SCALE))
    assert torch.equal(got, lbw_amd.attention_paged(q, c.cache, rows.contiguous(), _i32(lens)))
