"""paged_select where more pages score infinity than a list takes, beside negative, tiny and equal scores: the definition's
choice, and nothing written behind a list."""
import ctypes
import math

import pytest
import torch

import paged_ref as P

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
PAGE = 16


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _case(pages, infinite, low, step, width, how, seed=0):
    """Two sequences of `pages` pages each, one key/value head; a page's score is 128 times its bounds' value: from `low` up
    in steps, and infinite for `infinite` of them by `how`."""
    import lbw_amd
    g = torch.Generator().manual_seed(seed)
    total = 2 * pages
    table = torch.full((2, width), -1, dtype=torch.int32)
    table[:, :pages] = torch.randperm(total, generator=g).int().view(2, pages)
    value = (low + step * torch.arange(total, dtype=torch.float64)) / 128
    edge = value.to(BF)[:, None, None, None].expand(total, 1, 2, 128).clone()
    for b in range(2):
        for i, at in enumerate(torch.randperm(pages, generator=g)[:infinite].tolist()):
            kind = ("inf", "nan", "outside")[i % 3] if how == "all" else how
            if kind == "outside":
                table[b, at] = (-1, total, 2 ** 31 - 1, -2 ** 31)[i % 4]
            else:
                edge[int(table[b, at]), 0, :, i % 128] = math.inf if kind == "inf" else math.nan
    q = torch.ones(2, 1, 128, dtype=BF, device="cuda")
    pool = torch.zeros(1, 1, 1, 128, dtype=BF, device="cuda").expand(total, PAGE, 1, 128)   # (k and v are not read)
    return q, lbw_amd.PagedKV(pool, pool, edge.cuda()), table.cuda(), [pages * PAGE, pages * PAGE - 5]


def _guarded(q, cache, table, lens, count, first, last):
    """The lists of a call through the C entry, in a buffer with 4096 numbers behind them that have to stay."""
    from lbw_amd import _lib
    lib = _lib.load()
    p = _lib.PagedSelectParams()
    hk = cache.bounds.shape[1]
    n = q.shape[0] * hk * count
    sel = torch.full((n + 4096,), 12345, dtype=torch.int32, device="cuda")
    length = _i32(lens)
    p.cache.bounds, p.cache.pages, p.cache.page_size = cache.bounds.data_ptr(), cache.bounds.shape[0], cache.k.shape[1]
    p.cache.table, p.cache.table_stride, p.cache.table_width = table.data_ptr(), table.stride(0), table.shape[1]
    p.batch, p.q_heads, p.k_heads, p.head_dim = q.shape[0], q.shape[1], hk, 128
    p.q, p.q_stride_b, p.q_stride_h, p.lens = q.data_ptr(), q.stride(0), q.stride(1), length.data_ptr()
    p.count, p.first, p.last, p.selected = count, first, last, sel.data_ptr()
    size = lib.lbw_paged_select_workspace_size(ctypes.byref(p))
    ws = torch.empty(max(16, size), dtype=torch.uint8, device="cuda")
    rc = lib.lbw_paged_select(ctypes.byref(p), ctypes.c_void_p(ws.data_ptr()), size,
                              ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
    assert rc == 0, lib.lbw_last_error().decode()
    torch.cuda.synchronize()
    assert torch.all(sel[n:] == 12345)
    return sel[:n].view(q.shape[0], hk, count)


# one kernel (tables up to 233 pages of a group of one), and two
@pytest.mark.parametrize("pages,infinite,width", [(100, 9, 100), (100, 9, 1000), (200, 150, 200), (230, 9, 230), (500, 300, 500),
                                                  (1000, 600, 1000), (5000, 700, 5000), (5000, 4900, 5001)])
@pytest.mark.parametrize("low,step", [(-100.0, 0.25), (-20.0, 0.125), (-10.0, 0.0), (-5.0, 0.5), (-3.0, 0.0), (0.0, 0.0),
                                      (0.5, 0.0), (0.75, 0.0), (1.5, 0.5), (-1e30, 0.0)])
def test_more_infinite_pages_than_a_list_takes(pages, infinite, width, low, step):
    import lbw_amd
    q, cache, table, lens = _case(pages, infinite, low, step, width, "all", seed=pages)
    for count, first, last in ((1, 0, 0), (4, 0, 0), (7, 1, 2), (infinite, 0, 0), (infinite - 1, 0, 0),
                               (min(pages - 1, infinite + 3), 1, 1)):
        want = P.select(q, cache.bounds, table, lens, PAGE, count, first, last)
        assert torch.equal(_guarded(q, cache, table, lens, count, first, last).cpu(), want)
        assert torch.equal(lbw_amd.paged_select(q, cache, table, _i32(lens), count, first=first, last=last).cpu(), want)


@pytest.mark.parametrize("how", ["inf", "nan", "outside"])
@pytest.mark.parametrize("pages,width", [(150, 150), (700, 700)])
def test_each_way_to_be_infinite(how, pages, width):
    q, cache, table, lens = _case(pages, pages // 2, -10.0, 0.0625, width, how, seed=1)
    for count in (1, 5, pages // 2 - 1, pages // 2 + 1):
        want = P.select(q, cache.bounds, table, lens, PAGE, count, 0, 0)
        assert torch.equal(_guarded(q, cache, table, lens, count, 0, 0).cpu(), want)


def test_all_infinite_and_all_but_one():
    for pages in (120, 300, 5000):
        for infinite in (pages - 1, pages):
            q, cache, table, lens = _case(pages, infinite, -10.0, 0.0, pages, "all", seed=2)
            for count in (1, 60, pages - 1):
                want = P.select(q, cache.bounds, table, lens, PAGE, count, 0, 1)
                assert torch.equal(_guarded(q, cache, table, lens, count, 0, 1).cpu(), want)


def test_scores_of_minus_infinity():
    """An upper bound of -infinity under positive components of q: the lowest score there is, and a number's image."""
    q, cache, table, lens = _case(400, 3, -10.0, 0.0, 400, "inf", seed=3)
    finite = [int(p) for p in table[0] if torch.isfinite(cache.bounds[int(p)]).all()]
    cache.bounds[finite[50:300], :, 1] = -math.inf
    for count in (1, 3, 4, 150, 153, 154, 399):
        want = P.select(q, cache.bounds, table, lens, PAGE, count, 0, 0)
        assert torch.equal(_guarded(q, cache, table, lens, count, 0, 0).cpu(), want)
