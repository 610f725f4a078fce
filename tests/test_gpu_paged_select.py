"""paged_select against the definition on the host: the choice is exact."""
import math

import pytest
import torch

import paged_ref as P

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _case(lens, hq, hk, page, seed=0, width=None, spread=0.7):
    import lbw_amd
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(len(lens), hq, 128, generator=g) * 1.5).to(BF).cuda()
    table, _, total = P.make_table(lens, page, g, width=width)
    mid = torch.randn(total, hk, 1, 128, generator=g) * spread
    half = torch.rand(total, hk, 1, 128, generator=g) * 2
    edge = torch.cat((mid - half, mid + half), 2).to(BF).cuda()
    pool = torch.zeros(1, 1, 1, 128, dtype=BF, device="cuda").expand(total, page, hk, 128)   # (k and v are not read)
    return q, lbw_amd.PagedKV(pool, pool, edge), table.cuda()


def _check(q, cache, table, lens, count, first, last):
    import lbw_amd
    got = lbw_amd.paged_select(q, cache, table, _i32(lens), count, first=first, last=last)
    want = P.select(q, cache.bounds, table, lens, cache.k.shape[1], count, first, last)
    assert got.dtype == torch.int32 and torch.equal(got.cpu(), want)
    return got


@pytest.mark.parametrize("hq,hk", [(40, 8), (1, 1), (6, 3), (8, 1), (3, 3), (12, 4), (33, 1), (10, 2)])
@pytest.mark.parametrize("count,first,last", [(1, 0, 0), (4, 1, 1), (9, 0, 3), (9, 4, 5), (7, 2, 0)])
def test_heads_and_counts(hq, hk, count, first, last):
    lens = [1000, 0, 1, 16, 17, 145, 3000]
    _check(*_case(lens, hq, hk, 16, seed=hq), lens, count, first, last)


@pytest.mark.parametrize("page", [16, 64, 1024])
def test_page_sizes_and_wide_tables(page):
    lens = [20 * page, 20 * page - 1, 19 * page + 1, 5 * page, 6 * page, 7 * page]
    for count in (1, 6, 19, 20, 21, 64):
        _check(*_case(lens, 4, 2, page, seed=page, width=33), lens, count, min(2, count // 2), count // 3)


@pytest.mark.parametrize("pages", [1023, 1024, 1025, 4096, 4097, 9001])
def test_many_pages(pages):
    lens = [pages * 16, pages * 16 - 30]
    for count in (2, 100, pages // 2, pages - 1, pages):
        _check(*_case(lens, 2, 1, 16, seed=pages), lens, count, 1, 1)


def test_ties_go_to_the_lower_page():
    lens = [160, 800, 5000 * 16]
    for same in (1.0, 0.0, -0.0):
        q, cache, table = _case(lens, 4, 2, 16, seed=1)
        cache.bounds.fill_(same)
        for count in (1, 5, 9):
            got = _check(q, cache, table, lens, count, 1, 0)
            assert torch.equal(got.cpu(), torch.arange(count).int().expand(3, 2, count))
    # a few levels: the border lies within equal scores
    q, cache, table = _case(lens, 4, 2, 16, seed=2)
    g = torch.Generator().manual_seed(3)
    level = torch.randint(0, 3, (cache.bounds.shape[0], 1, 1, 1), generator=g).cuda().to(BF)
    cache.bounds.copy_(level.expand_as(cache.bounds))
    for count in (2, 7, 40):
        _check(q, cache, table, lens, count, 0, 1)


def test_scores_close_together_and_far_apart():
    """Scores that fp32 sums could not tell apart, and ones that span all exponents."""
    lens = [64 * 16]
    q, cache, table = _case(lens, 1, 1, 16, seed=4)
    q.fill_(1.0)
    cache.bounds.fill_(256.0)                             # a sum of 127 times 256 ...
    steps = torch.randperm(64, generator=torch.Generator().manual_seed(5)).double() * 2.0 ** -30
    cache.bounds[table[0, :64].long(), 0, :, 5] = steps.to(BF).cuda()[:, None]   # ... and the smallest differences
    for count in (1, 10, 33):
        got = _check(q, cache, table, lens, count, 0, 0)
        order = torch.sort(steps.to(BF).float(), descending=True, stable=True).indices[:count]
        assert torch.equal(got[0, 0].cpu(), torch.sort(order).values.int())
    lens = [3000 * 16]
    q, cache, table = _case(lens, 2, 2, 16, seed=6)
    g = torch.Generator().manual_seed(7)
    big = torch.exp2(torch.randint(-100, 100, (cache.bounds.shape[0], 1, 1, 1), generator=g).float()).cuda()
    cache.bounds.copy_((cache.bounds.float() * big).to(BF))
    for count in (3, 500, 2900):
        _check(q, cache, table, lens, count, 1, 2)


def test_nan_infinities_and_pages_outside_come_first():
    lens = [100 * 16, 50 * 16]
    q, cache, table = _case(lens, 6, 2, 16, seed=8)
    cache.bounds[table[0, 40].long(), 1, 0, 3] = float("nan")
    cache.bounds[table[0, 41].long(), 0, 1, 9] = math.inf
    cache.bounds[table[0, 42].long(), 0, 0, 9] = -math.inf
    table[0, 77], table[1, 20], table[1, 21] = -1, cache.bounds.shape[0], 2 ** 31 - 1
    for count in (1, 2, 4, 9):
        _check(q, cache, table, lens, count, 0, 0)
    got = _check(q, cache, table, lens, 6, 0, 0).cpu()
    assert {41, 42, 77} <= set(got[0, 0].tolist()) and {40, 77} <= set(got[0, 1].tolist())
    assert {20, 21} <= set(got[1, 0].tolist())
    q[1, 2] = float("nan")                                 # every page alike for its group
    _check(q, cache, table, lens, 5, 1, 1)


def test_lengths_outside_and_strided_q():
    lens = [-5, 2 ** 31 - 1, 33]
    q, cache, table = _case([160, 160, 33], 4, 2, 16, seed=9, width=10)
    _check(q, cache, table, lens, 4, 1, 1)
    buf = torch.zeros(3, 9, 128, dtype=BF, device="cuda")
    buf[:, 3:7] = q
    _check(buf[:, 3:7], cache, table, lens, 4, 1, 1)
    wide = torch.full((3, 30), -9, dtype=torch.int32, device="cuda")
    wide[:, 5:15] = table
    _check(q, cache, wide[:, 5:15], lens, 4, 1, 1)


def test_no_sequences_and_same_choice_every_run():
    import lbw_amd
    lens = [5000 * 16, 777]
    q, cache, table = _case(lens, 40, 8, 16, seed=10)
    assert lbw_amd.paged_select(q[:0], cache, table[:0], _i32([]), 5).shape == (0, 8, 5)
    first = _check(q, cache, table, lens, 50, 1, 4)
    for _ in range(5):
        assert torch.equal(lbw_amd.paged_select(q, cache, table, _i32(lens), 50, first=1, last=4), first)
    assert torch.all(lbw_amd.paged_select(q, cache, table[:, :0], _i32(lens), 5) == -1)


def test_bounds_hold_every_key_and_scores_every_product():
    """What the selection rests on: no key of a page scores above the page's score."""
    import lbw_amd
    g = torch.Generator().manual_seed(11)
    k, v = P.make_pool(8, 16, 2, 128, g)
    edge = torch.stack((k.amin(1), k.amax(1)), 2).contiguous()
    q = torch.randn(1, 6, 128, generator=g).to(BF).cuda()
    table = torch.arange(8, dtype=torch.int32)[None].cuda()
    best = (q[0].double().view(2, 3, 128)[:, None, :, None] *
            k.double().permute(2, 0, 1, 3)[:, :, None]).sum(-1).amax((2, 3))          # [heads, pages]
    qq = q[0].double().view(2, 3, 1, 128)
    e = edge.double().permute(1, 2, 0, 3)[:, :, None]
    score = (qq.clamp_min(0) * e[:, 1] + qq.clamp_max(0) * e[:, 0]).sum(-1).amax(1)
    assert torch.all(score >= best)
    sel = lbw_amd.paged_select(q, lbw_amd.PagedKV(k, v, edge), table, _i32([128]), 3, first=0, last=0)
    assert torch.equal(sel[0].cpu(), torch.sort(score.topk(3).indices, -1).values.int().cpu())


@pytest.mark.parametrize("hq,hk", [(1, 1), (2, 1), (3, 1), (4, 2), (5, 1), (7, 1), (12, 4), (64, 8)])
def test_short_tables_and_the_same_ones_widened(hq, hk):
    """A short table is scored and chosen from by one kernel, a wide one by two: the same choice, with ties, infinities, NaN
    and pages outside the cache among the scores."""
    import lbw_amd
    grp = hq // hk
    n = min(256, 700 // (grp + 2))           # the longest table that one kernel takes
    lens = [16 * n, 16 * n - 9, 16 * (n - 1), 16 * (n // 2) + 1, 16, 0]
    for width in (n, n + 1, 4 * n):
        q, cache, table = _case(lens, hq, hk, 16, seed=hq, width=4 * n)
        e = cache.bounds
        e[table[0, 3].long(), :, 0, 7] = float("-inf")
        e[table[0, 9].long(), :, 1, 5] = float("nan")
        e[table[1, 4:30].long()] = e[table[1, 4].long()].clone()
        table[2, 5] = e.shape[0]
        table[2, n - 3] = -7
        t = table[:, :width].contiguous()
        for count in (1, 8, n // 2, n - 1):
            _check(q, cache, t, lens, count, 0, 0)
            _check(q, cache, t, lens, count, count // 4, count // 3)
    # more sequences and heads than CUs: two kernels for short tables too
    many = [16 * 6 - i % 90 for i in range(300)]
    _check(*_case(many, grp, 1, 16, seed=3), many, 3, 1, 1)
