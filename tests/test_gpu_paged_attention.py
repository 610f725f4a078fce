"""attention_paged -- own keys, a common prefix, selected pages -- against the 64-bit definition."""
import math

import pytest
import torch

import packed_ref as R
import paged_ref as P

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
SCALE = 1 / math.sqrt(128)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Case:
    def __init__(self, lens, hq, hk, page, *, prefix=0, seed=0, head_major=True, heat=1.5, fill=-1, width=None):
        import lbw_amd
        g = torch.Generator().manual_seed(seed)
        self.lens, self.page = lens, page
        q = torch.randn(len(lens), hq, 128, generator=g) * (torch.rand(hq, 1, generator=g) * heat + 0.2)
        self.q = q.to(BF).cuda()
        need = P.pages_of(prefix, page)
        table, spare, total = P.make_table(lens, page, g, need + 3, width=width, fill=fill)
        self.table = table.cuda()
        self.cache = lbw_amd.PagedKV(*P.make_pool(total, page, hk, 128, g, head_major))
        self.prefix_table = spare[:need].contiguous().cuda() if prefix else None
        self.prefix = prefix

    def run(self, lens=None, **kw):
        import lbw_amd
        if self.prefix_table is not None:
            kw = {"prefix_table": self.prefix_table, "prefix_len": self.prefix, **kw}
        return lbw_amd.attention_paged(self.q, self.cache, self.table, _i32(self.lens if lens is None else lens), **kw)

    def check(self, scale=SCALE, **kw):
        sel = kw.get("selected")
        got = self.run(**kw)
        want, allow = P.attention(self.q, self.cache.k, self.cache.v, self.table, self.lens, scale,
                                  self.prefix_table, self.prefix, sel)
        R.assert_within("out", got, want, allow)
        return got


CASES = [  # lens, heads, kv heads, page
    ([1], 1, 1, 16), ([0], 2, 1, 16), ([5], 40, 8, 64), ([500], 40, 8, 64), ([31, 32, 33, 0, 64], 12, 4, 16),
    ([1000, 1, 129, 1023], 5, 1, 32), ([2000, 3], 6, 3, 128), ([700], 3, 3, 1024), ([100, 90], 66, 1, 16),
    ([97], 40, 1, 64), ([4096], 2, 2, 256), ([300] * 20, 4, 2, 16), ([7, 0, 40] * 50, 2, 1, 16),
    ([15, 16, 17, 47, 48, 49], 8, 2, 16), ([2600, 0, 1700], 4, 4, 16),
]


@pytest.mark.parametrize("lens,hq,hk,page", CASES)
@pytest.mark.parametrize("splits", [0, 1, 3])
def test_own_keys(lens, hq, hk, page, splits):
    Case(lens, hq, hk, page, seed=1).check(num_splits=splits)


@pytest.mark.parametrize("prefix", [1, 15, 16, 17, 33, 200, 1537])
@pytest.mark.parametrize("lens,hq,hk,page", [
    ([0], 4, 2, 16), ([7], 40, 8, 64), ([40, 0, 1, 17], 12, 4, 32), ([5] * 33, 5, 1, 16), ([100, 3] * 20, 3, 3, 64),
    ([10, 20], 66, 1, 16), ([1100, 0], 2, 1, 1024)])
def test_prefix(prefix, lens, hq, hk, page):
    Case(lens, hq, hk, page, prefix=prefix, seed=prefix).check()


@pytest.mark.parametrize("splits", [0, 1, 2, 7, 128])
def test_prefix_pieces_and_many_rows(splits):
    c = Case([60, 0, 300, 1] * 12, 10, 2, 64, prefix=3000, seed=5)
    c.check(num_splits=splits)
    Case([2000, 1, 1500], 8, 8, 16, prefix=700, seed=6).check(num_splits=splits)


def test_prefix_lengths_on_the_device():
    c = Case([20, 5], 12, 4, 32, prefix=100, seed=7)
    want = c.run()
    assert torch.equal(c.run(prefix_len=_i32([100])), want)
    full = c.run(prefix_len=None)
    assert torch.equal(c.run(prefix_len=_i32([10 ** 9])), full) and torch.equal(c.run(prefix_len=128), full)
    none = c.run(prefix_len=_i32([0]))
    assert torch.equal(c.run(prefix_len=_i32([-5])), none)
    c.prefix_table = None
    R.assert_within("no prefix", none, *P.attention(c.q, c.cache.k, c.cache.v, c.table, c.lens, SCALE))
    empty = c.run(prefix_table=_i32([]), prefix_len=None)
    assert torch.equal(empty, c.run())


def test_a_prefix_is_the_first_pages_of_every_table():
    """The same keys once as a prefix and once as the head of each sequence's own row (shared pages)."""
    page, prefix = 16, 160
    c = Case([30, 0, 77, 1], 12, 4, page, prefix=prefix, seed=8)
    want, allow = P.attention(c.q, c.cache.k, c.cache.v, c.table, c.lens, SCALE, c.prefix_table, prefix)
    R.assert_within("prefix", c.run(), want, allow)
    c.table = torch.cat((c.prefix_table[None].expand(4, -1), c.table), 1).contiguous()
    c.prefix_table = None
    R.assert_within("shared pages", c.run(lens=[n + prefix for n in c.lens]), want, allow)


@pytest.mark.parametrize("splits", [0, 1, 2, 5])
@pytest.mark.parametrize("page", [16, 64])
def test_selected(splits, page):
    c = Case([700, 0, 130, 1, 64], 8, 2, page, seed=9, width=60)
    sel = torch.full((5, 2, 6), -1, dtype=torch.int32)
    sel[0, 0] = torch.tensor([0, 2, 3, 5, 7, 10])
    sel[0, 1] = torch.tensor([10, 0, 10, 4, -1, 3])     # any order, one twice, ended early
    sel[1] = torch.arange(6)                             # no keys there
    sel[2, 0, :3] = torch.tensor([1, 0, 50])             # an entry past the length
    sel[2, 1] = torch.tensor([50, 51, 52, 53, 54, 1])    # ... whole tiles of them
    sel[3, 0, 0], sel[3, 1, :] = 0, 40                   # a single key; nothing but entries past the length
    sel[4, 0, :1] = 0                                    # (head 1: an empty list)
    c.check(selected=sel.cuda(), num_splits=splits)


def test_selected_of_one_odd_page_and_none():
    c = Case([333, 40], 6, 3, 16, seed=10)
    c.check(selected=torch.zeros(2, 3, 1, dtype=torch.int32, device="cuda"))
    c.check(selected=torch.tensor([[[20], [3], [1]], [[2], [0], [1]]], dtype=torch.int32, device="cuda"))
    assert torch.all(c.run(selected=torch.zeros(2, 3, 0, dtype=torch.int32, device="cuda")) == 0)
    assert torch.all(c.run(selected=torch.full((2, 3, 4), -1, dtype=torch.int32, device="cuda")) == 0)


def test_all_pages_selected_is_the_whole_sequence():
    c = Case([500, 33, 64], 12, 4, 32, seed=11)
    n = c.table.shape[1]
    sel = torch.arange(n, dtype=torch.int32).expand(3, 4, n).contiguous().cuda()
    assert torch.equal(c.run(selected=sel, num_splits=1), c.run(num_splits=1))


def test_selected_behind_a_prefix():
    c = Case([300, 64, 0], 8, 2, 16, prefix=100, seed=12)
    sel = torch.full((3, 2, 5), -1, dtype=torch.int32)
    sel[0, 0], sel[0, 1, :2], sel[1, 0, :4], sel[1, 1, 0] = torch.tensor([0, 3, 9, 17, 18]), torch.tensor([18, 1]), \
        torch.arange(4), 2
    c.check(selected=sel.cuda())
    c.check(selected=sel.cuda(), num_splits=3)


def test_many_pieces_scale_and_rising_scores():
    c = Case([3000, 2411], 8, 2, 64, seed=13)
    rise = torch.linspace(-2, 2, c.table.shape[1] * 64, device="cuda").view(-1, 64)
    for b in range(2):
        n = P.pages_of(c.lens[b], 64)
        at = c.table[b, :n].long()
        c.cache.k[at] = (c.cache.k[at] * 0.1 + rise[:n, :, None, None] * c.q[b, ::4]).to(BF)
    for splits in (0, 1, 2, 17, 128):
        c.check(scale=0.2, softmax_scale=0.2, num_splits=splits)


@pytest.mark.parametrize("kind", ["own", "prefix", "selected"])
def test_what_lies_behind_a_length_is_not_read(kind):
    """Rows behind a length, pages that belong to nobody and table entries behind a sequence may hold anything."""
    page = 64
    c = Case([300, 0, 41, 200, 64], 10, 2, page, prefix=100 if kind == "prefix" else 0, seed=14, width=9)
    kw = {}
    if kind == "selected":
        sel = torch.full((5, 2, 4), -1, dtype=torch.int32)
        sel[0], sel[1], sel[2, :, :2], sel[3], sel[4, :, 0] = torch.tensor([0, 2, 3, 4]), 0, torch.tensor([0, 5]), \
            torch.tensor([3, 0, 1, 8]), 0
        kw["selected"] = sel.cuda()
    for splits in (0, 1, 3):
        want = c.run(num_splits=splits, **kw)
        used = torch.zeros(c.cache.k.shape[0], page, dtype=torch.bool)
        lists = [(c.table[b], n) for b, n in enumerate(c.lens)]
        if kind == "prefix":
            lists.append((c.prefix_table, 100))
        for pages, n in lists:
            for r in range(n):
                used[int(pages[r // page]), r % page] = True
        k, v, table = c.cache.k.clone(), c.cache.v.clone(), c.table.clone()
        c.cache.k[~used] = float("nan")
        c.cache.v[~used] = float("inf")
        for b, n in enumerate(c.lens):
            c.table[b, P.pages_of(n, page):] = 2 ** 31 - 1 if b % 2 else -77
        lens = list(c.lens)
        lens[1] = -2 ** 31
        got = c.run(lens=lens, num_splits=splits, **kw)
        assert torch.equal(got, want)
        c.cache.k.copy_(k), c.cache.v.copy_(v), c.table.copy_(table)


def test_lengths_are_limited_to_the_table():
    c = Case([64, 32], 4, 2, 16, seed=15, width=4)
    want = c.run(lens=[64, 64])   # (the second one's entries behind its pages: outside the cache)
    got = c.run(lens=[2 ** 31 - 1, 10 ** 6])
    assert torch.equal(got[0], want[0]) and torch.isnan(got[1]).all() and torch.isnan(want[1]).all()


@pytest.mark.parametrize("splits", [0, 1, 3])
def test_pages_outside_the_cache_make_their_rows_nan(splits):
    for bad in (-1, -2 ** 31, 2 ** 31 - 1, "pages"):
        c = Case([300, 40, 0, 2000], 8, 2, 16, seed=16)
        want = c.run(num_splits=splits)
        bad = c.cache.k.shape[0] if bad == "pages" else bad
        c.table[0, 18] = bad        # its last page
        c.table[3, 5] = bad
        got = c.run(num_splits=splits)
        assert torch.isnan(got[[0, 3]]).all() and torch.equal(got[1:3], want[1:3])
        sel = torch.tensor([0, 1, 3, -1], dtype=torch.int32).expand(4, 2, 4).clone().cuda()
        assert torch.isfinite(c.run(selected=sel, num_splits=splits)).all()   # (not those pages)
        sel[0, 1, 2] = 18
        got = c.run(selected=sel, num_splits=splits)
        assert torch.isnan(got[0, 4:]).all() and torch.isfinite(got[0, :4]).all() and torch.isfinite(got[1:]).all()
    c = Case([10, 0], 4, 2, 16, prefix=40, seed=17)
    c.prefix_table[1] = 10 ** 6
    assert torch.isnan(c.run(num_splits=splits)).all()


@pytest.mark.parametrize("splits", [0, 1, 3, 128])
def test_nan_and_infinite_scores_stay_in_their_heads(splits):
    c = Case([2500, 0, 40, 1999], 8, 2, 64, seed=18)
    want = c.run(num_splits=splits)
    nan = torch.zeros(4, 8, dtype=torch.bool, device="cuda")
    c.q[0, 3] = float("nan")
    c.q[0, 5] = 3e38
    c.q[1, 0] = float("nan")                              # (no keys: 0 all the same)
    c.cache.k[c.table[2, 0].long(), :40, 1] = float("nan")
    c.cache.k[c.table[3, 8:20].long(), :, 0] = float("nan")
    c.cache.v[c.table[3, 25].long(), 3, 1] = float("nan")
    nan[0, 3] = nan[0, 5] = True
    nan[2, 4:] = True
    nan[3] = True
    got = c.run(num_splits=splits)
    assert torch.equal(torch.isnan(got).all(-1), nan) and torch.equal(torch.isnan(got).any(-1), nan)
    assert torch.equal(got[~nan], want[~nan])


def test_strided_pool_q_and_out():
    a, b = (Case([130, 64, 7], 6, 2, 16, seed=19, head_major=x) for x in (True, False))
    b.cache.k.copy_(a.cache.k), b.cache.v.copy_(a.cache.v)
    want = a.run()
    assert torch.equal(b.run(), want)
    qkv = torch.zeros(3, 10, 128, dtype=BF, device="cuda")
    qkv[:, 2:8] = a.q
    a.q = qkv[:, 2:8]
    buf = torch.full((3, 7, 136), 5.0, dtype=BF, device="cuda")
    out = buf[:, :6, :128]
    assert a.run(out=out) is out and torch.equal(out, want)
    out.fill_(5.0)
    assert torch.all(buf == 5.0)


def test_offsets_past_32_bits():
    import lbw_amd
    page, hk = 1024, 8
    pages = (1 << 31) // (page * hk * 128) + 3
    k = torch.zeros(pages, hk, page, 128, dtype=BF, device="cuda").transpose(1, 2)
    assert k.numel() > 1 << 31
    g = torch.Generator().manual_seed(20)
    k[pages - 1] = torch.randn(page, hk, 128, generator=g).to(BF).cuda()
    k[pages - 2, :500] = torch.randn(500, hk, 128, generator=g).to(BF).cuda()
    cache = lbw_amd.PagedKV(k, k)     # (one buffer for both: K = V)
    q = torch.randn(2, 2 * hk, 128, generator=g).to(BF).cuda()
    table, lens = _i32([[pages - 1, pages - 2], [pages - 1, pages - 2]]), [1524, 700]
    want, allow = P.attention(q, k, k, table, lens, SCALE)
    for splits in (0, 1, 4):
        R.assert_within("out", lbw_amd.attention_paged(q, cache, table, _i32(lens), num_splits=splits), want, allow)
    got = lbw_amd.attention_paged(q, cache, table[:, :0], _i32([0, 0]), prefix_table=table[0].contiguous(),
                                  prefix_len=1524)
    want, allow = P.attention(q, k, k, table, [1524, 1524], SCALE)
    R.assert_within("prefix", got, want, allow)
    sel = torch.tensor([1, -1], dtype=torch.int32).expand(2, hk, 2).contiguous().cuda()
    got = lbw_amd.attention_paged(q, cache, table, _i32([1524, 1524]), selected=sel)
    want, allow = P.attention(q, k, k, table[:, 1:].contiguous(), [500, 500], SCALE)
    R.assert_within("selected", got, want, allow)


def test_a_long_sequence():
    """400000 keys of one sequence, small pages."""
    c = Case([400000], 4, 2, 16, seed=21)
    got = c.run()
    k, v = (P.rows(x, c.table[0, :25000], 400000).transpose(0, 1).float() for x in (c.cache.k, c.cache.v))
    q = c.q[0].view(2, 2, 128).double()
    s = torch.bmm(q, k.double().transpose(1, 2).contiguous()) * SCALE
    p = torch.softmax(s, -1)
    want = torch.bmm(p, v.double()).view(4, 128)
    size = torch.bmm(p, v.double().abs()).view(4, 128)
    # P's and the output's roundings, and 2^-10 for the fp32 sums of 400000 terms in 12500 tiles
    R.assert_within("out", got[0], want, R.H * want.abs() + (R.H + 2 ** -10) * (1 + R.H) * size)


def test_no_sequences_and_refusals():
    import lbw_amd
    c = Case([20, 30], 4, 2, 16, seed=22)
    empty = lbw_amd.attention_paged(c.q[:0], c.cache, c.table[:0], _i32([]))
    assert empty.shape == (0, 4, 128)
    assert torch.all(lbw_amd.attention_paged(c.q, c.cache, c.table[:, :0], _i32([3, 3])) == 0)
    with pytest.raises(RuntimeError, match="overlaps"):
        c.run(out=c.q)
    with pytest.raises(RuntimeError, match="int32"):
        lbw_amd.attention_paged(c.q, c.cache, c.table, _i32([3, 3]).cpu())
    with pytest.raises(RuntimeError, match="contiguous"):
        c.run(selected=torch.zeros(2, 4, 2, dtype=torch.int32, device="cuda").transpose(1, 2))
    with pytest.raises(RuntimeError, match="int32"):
        c.run(prefix_table=c.table[0].cpu())
    k = c.cache.k.transpose(1, 3).contiguous().transpose(1, 3)
    with pytest.raises(RuntimeError, match="contiguous head dim"):
        lbw_amd.attention_paged(c.q, lbw_amd.PagedKV(k, c.cache.v), c.table, _i32([3, 3]))
    x = c.q.detach().requires_grad_()
    out = lbw_amd.attention_paged(x, c.cache, c.table, _i32([3, 3]))
    with pytest.raises(RuntimeError):
        out.float().sum().backward()
    with pytest.raises(NotImplementedError, match="not differentiable"):
        lbw_amd.attention_paged(x, c.cache, c.table, _i32([3, 3]), out=torch.empty_like(c.q))


@pytest.mark.parametrize("prefix", [1, 15, 16, 17, 31, 32, 33, 47, 100, 449, 1000])
@pytest.mark.parametrize("lens,hq,hk,page", [
    ([0, 1, 15, 16, 17, 33, 90], 12, 4, 16), ([64, 70, 0], 66, 1, 64), ([5, 60], 6, 3, 1024), ([40, 1] * 70, 4, 2, 32)])
def test_short_prefixes_walked_by_each_sequence_and_apart(prefix, lens, hq, hk, page):
    c = Case(lens, hq, hk, page, prefix=prefix, seed=prefix)
    for splits in (0, 1, 2):
        c.check(num_splits=splits)
    n = P.pages_of(max(lens), page)
    sel = torch.full((len(lens), hk, n + 1), -1, dtype=torch.int32)
    sel[..., :n] = torch.arange(n, dtype=torch.int32).flip(0)
    sel[0] = -1
    for splits in (0, 1):
        c.check(num_splits=splits, selected=sel.cuda())
    # lengths of it that the device holds
    for m in (0, 1, 18, prefix, prefix + 1, 2 ** 31 - 1, -5):
        kw = {"prefix_table": c.prefix_table, "prefix_len": _i32([m])}
        got = c.run(**kw)
        want, allow = P.attention(c.q, c.cache.k, c.cache.v, c.table, lens, SCALE, c.prefix_table,
                                  max(0, min(m, len(c.prefix_table) * page)))
        R.assert_within("out", got, want, allow)


def test_a_bad_page_of_a_short_prefix_reaches_all_and_of_a_sequence_only_it():
    for splits in (0, 1):
        c = Case([20, 0, 50], 4, 2, 16, prefix=60, seed=90)
        want = c.run(num_splits=splits)
        c.table[2, 1] = -9
        got = c.run(num_splits=splits)
        assert torch.isnan(got[2]).all() and torch.equal(got[:2], want[:2])
        c.prefix_table[3] = c.cache.k.shape[0]
        assert torch.isnan(c.run(num_splits=splits)).all()
