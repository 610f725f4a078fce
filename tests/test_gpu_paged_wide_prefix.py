"""A common prefix for more than 96 query rows a key/value head, 128 at a time over shared tiles: lengths on the device, what
lies behind them, pages outside the cache, offsets past 32 bits, replays."""
import math

import pytest
import torch

import packed_ref as R
import paged_ref as P
from test_gpu_paged_attention import SCALE, Case, _i32

pytestmark = pytest.mark.gpu
BF = torch.bfloat16

# lens, heads, kv heads, page: 97, 129, 160 and 260 rows a key/value head (waves and workgroups with some rows and none)
WIDE = [([30, 0, 5] * 32 + [1], 2, 2, 16), ([7] * 43, 6, 2, 64), ([90, 0, 16, 33] * 8, 10, 2, 32), ([3, 60] * 65, 2, 1, 1024)]


def _used(c, own=True):
    """Which rows of the pool belong to the prefix's first c.prefix keys or to a sequence."""
    used = torch.zeros(c.cache.k.shape[:2], dtype=torch.bool)
    lists = [(c.prefix_table.cpu(), c.prefix)] + [(c.table[b].cpu(), n) for b, n in enumerate(c.lens) if own]
    for pages, n in lists:
        for r in range(n):
            used[int(pages[r // c.page]), r % c.page] = True
    return used


@pytest.mark.parametrize("lens,hq,hk,page", WIDE)
@pytest.mark.parametrize("splits", [0, 1, 3, 128])
def test_lengths_on_the_device(lens, hq, hk, page, splits):
    c = Case(lens, hq, hk, page, prefix=2500, seed=len(lens))
    reach = len(c.prefix_table) * page
    for n in (0, 1, 15, 16, 63, 64, 65, 1000, 1537, 2499, 2500, reach, reach + 1, 2 ** 31 - 1, -7):
        got = c.run(prefix_len=_i32([n]), num_splits=splits)
        keys = max(0, min(n, reach))
        some = [0, 1, len(lens) // 2, len(lens) - 1]
        want, allow = P.attention(c.q[some], c.cache.k, c.cache.v, c.table[some], [lens[b] for b in some], SCALE,
                                  c.prefix_table, keys)
        R.assert_within(f"{n} keys", got[some], want, allow)


@pytest.mark.parametrize("lens,hq,hk,page", WIDE)
@pytest.mark.parametrize("prefix", [1500, 1537, 2111])
@pytest.mark.parametrize("splits", [0, 1, 5])
def test_what_lies_behind_the_prefix_is_not_read(lens, hq, hk, page, prefix, splits):
    c = Case(lens, hq, hk, page, prefix=prefix, seed=prefix)
    c.prefix_table = torch.cat((c.prefix_table, _i32([0, 1, 2]))).contiguous()
    kw = {"prefix_len": _i32([prefix]), "num_splits": splits}
    want = c.run(**kw)
    used = _used(c).cuda()
    c.cache.k[~used] = math.nan
    c.cache.v[~used] = math.inf
    c.cache.v[~used] *= torch.tensor([1.0, math.nan], dtype=BF, device="cuda").repeat(64)
    need = P.pages_of(prefix, page)
    c.prefix_table[need:] = _i32([-1, 2 ** 31 - 1, c.cache.k.shape[0]])
    assert torch.equal(c.run(**kw), want)


@pytest.mark.parametrize("lens,hq,hk,page", WIDE)
@pytest.mark.parametrize("splits", [0, 1, 3, 128])
@pytest.mark.parametrize("bad", [-1, -2 ** 31, 2 ** 31 - 1, "pages"])
def test_pages_outside_the_cache(lens, hq, hk, page, splits, bad):
    """Every row whose prefix holds such a page is NaN; a length that ends before it leaves it out."""
    c = Case(lens, hq, hk, page, prefix=2500, seed=3)
    n_pages = len(c.prefix_table)
    bad = c.cache.k.shape[0] if bad == "pages" else bad
    for at in {0, n_pages // 2, n_pages - 1}:
        old = int(c.prefix_table[at])
        kw = {"prefix_len": _i32([at * page]), "num_splits": splits}
        clean = c.run(**kw)
        c.prefix_table[at] = bad
        assert torch.equal(c.run(**kw), clean)
        for n in (at * page + 1, 2500):
            assert torch.isnan(c.run(prefix_len=_i32([n]), num_splits=splits)).all()
        c.prefix_table[at] = old
    assert torch.isfinite(c.run(num_splits=splits)).all()


def test_bad_pages_beside_sequences_own():
    """One of a sequence's pages, and a selection behind the prefix."""
    c = Case([40, 0, 33] * 20, 12, 4, 16, prefix=2000, seed=4)
    old = int(c.table[3, 1])
    for splits in (0, 1, 4):
        want = c.run(num_splits=splits)
        c.table[3, 1] = -5
        got = c.run(num_splits=splits)
        assert torch.isnan(got[3]).all() and torch.equal(got[:3], want[:3]) and torch.equal(got[4:], want[4:])
        sel = torch.tensor([0, 2, -1], dtype=torch.int32).expand(60, 4, 3).contiguous().cuda()
        assert torch.isfinite(c.run(num_splits=splits, selected=sel)).all()
        sel[3, 2, 2] = 1
        got = c.run(num_splits=splits, selected=sel)
        assert torch.isnan(got[3, 6:9]).all() and torch.isfinite(got[3, :6]).all() and torch.isfinite(got[4:]).all()
        c.table[3, 1] = old


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
    q = torch.randn(52, 2 * hk, 128, generator=g).to(BF).cuda()
    table = _i32([[pages - 2]]).expand(52, 1).contiguous()
    lens = [0, 1, 300, 500] * 13
    for splits in (0, 1, 4):
        got = lbw_amd.attention_paged(q, cache, table, _i32(lens), prefix_table=_i32([pages - 1, pages - 2]), prefix_len=1524,
                                      num_splits=splits)
        want, allow = P.attention(q[:8], k, k, table[:8], lens[:8], SCALE, _i32([pages - 1, pages - 2]), 1524)
        R.assert_within("out", got[:8], want, allow)
        assert torch.isfinite(got).all()


@pytest.mark.parametrize("selected", [False, True])
def test_replays_follow_the_device(selected):
    c = Case([40, 0, 33, 300] * 12, 12, 4, 16, prefix=3000, seed=6)
    n = _i32([3000])
    lens = _i32(c.lens)
    import lbw_amd
    sel = torch.tensor([0, 2, 1, -1], dtype=torch.int32).expand(48, 4, 4).contiguous().cuda()
    kw = {"prefix_table": c.prefix_table, "prefix_len": n, **({"selected": sel} if selected else {})}

    def call():
        return lbw_amd.attention_paged(c.q, c.cache, c.table, lens, **kw)

    call()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call()
        graphs.append((g, out))
    for i, keys in enumerate((3000, 0, 17, 2048, 9999, 1)):
        n.fill_(keys)
        lens.copy_(_i32([(x * (i + 1)) % 301 for x in c.lens]))
        c.q.normal_()
        for g, out in graphs:
            g.replay()
            want = call()
            torch.cuda.synchronize()
            # (lengths past a sequence's pages meet entries of -1: NaN in both)
            assert torch.allclose(out.float(), want.float(), rtol=0, atol=0, equal_nan=True)
