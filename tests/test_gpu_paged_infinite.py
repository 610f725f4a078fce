"""attention_paged with infinities among the keys and values, as the formula has them: an infinite value makes its component
infinite and nothing else changes, a score of -infinity has the weight 0, scores that are all of it give NaN."""
import math

import pytest
import torch

import packed_ref as R
import paged_ref as P
from test_gpu_paged_attention import SCALE, Case, _i32

pytestmark = pytest.mark.gpu
LENS = [1, 5, 15, 16, 17, 31, 32, 33, 47, 63, 64, 65, 100, 0, 700]


def _lists(c, seed=0):
    """A selection of all of a sequence's pages in any order, -1 behind them."""
    g = torch.Generator().manual_seed(seed)
    need = [P.pages_of(n, c.page) for n in c.lens]
    sel = torch.full((len(need), c.cache.k.shape[2], max(need) + 1), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        for h in range(sel.shape[1]):
            sel[b, h, :n] = torch.randperm(n, generator=g).int()
    return sel.cuda()


# lens, heads, kv heads, page, prefix: whole sequences and pieces; prefixes walked by each sequence, 32 and 128 rows at a time
FORMS = [(LENS, 12, 4, 16, 0), (LENS, 5, 1, 64, 0), ([4100, 3000, 33], 40, 8, 64, 0), (LENS, 12, 4, 16, 21),
         (LENS[:5], 12, 4, 32, 2000), (LENS, 66, 1, 16, 90), ([40, 0, 3] * 20, 12, 4, 16, 1537),
         ([7, 0, 90] * 12, 10, 2, 64, 3001), ([33] * 100, 2, 1, 1024, 1030), (LENS * 8, 8, 8, 16, 2047)]


@pytest.mark.parametrize("lens,hq,hk,page,prefix", FORMS)
@pytest.mark.parametrize("splits", [0, 1, 3])
@pytest.mark.parametrize("selected", [False, True])
def test_an_infinite_value_is_its_own_component_s(lens, hq, hk, page, prefix, splits, selected):
    """In the last key of every sequence, of the prefix, and in a key in the middle."""
    c = Case(lens, hq, hk, page, prefix=prefix, seed=len(lens) + prefix)
    kw = {"num_splits": splits, **({"selected": _lists(c)} if selected else {})}
    clean = c.run(**kw)
    mark = torch.zeros(len(lens), hq, 128, dtype=torch.float32, device="cuda")
    grp = hq // hk

    def put(page_of, row, b, head, d, value):
        c.cache.v[int(page_of[row // page]), row % page, head, d] = value
        mark[b, head * grp:(head + 1) * grp, d] = value

    for b, n in enumerate(lens):
        if n:
            put(c.table[b], n - 1, b, 0, b % 50, math.inf)
            put(c.table[b], n // 2, b, hk - 1, 50 + b % 50, -math.inf)
    if prefix:
        put(c.prefix_table, prefix - 1, slice(None), hk - 1, 127, -math.inf)
        put(c.prefix_table, prefix // 3, slice(None), 0, 126, math.inf)
    got = c.run(**kw).float()
    assert torch.equal(got[mark != 0], mark[mark != 0])
    assert torch.equal(got[mark == 0], clean.float()[mark == 0])


@pytest.mark.parametrize("lens,hq,hk,page,prefix", FORMS)
@pytest.mark.parametrize("splits", [0, 1, 3])
@pytest.mark.parametrize("selected", [False, True])
def test_scores_of_minus_infinity(lens, hq, hk, page, prefix, splits, selected):
    c = Case(lens, hq, hk, page, prefix=prefix, seed=len(lens) + prefix + 1)
    c.q[..., 9] = 1.0
    kw = {"num_splits": splits, **({"selected": _lists(c)} if selected else {})}
    # the second half of every sequence, and the first half of the prefix: as if they were not there
    keep = [n - n // 2 for n in lens]
    for b, n in enumerate(lens):
        for row in range(keep[b], n):
            c.cache.k[int(c.table[b, row // page]), row % page, :, 9] = -math.inf
    behind = prefix // 2
    first = [(int(c.prefix_table[r // page]), r % page) for r in range(prefix)] if prefix else []
    for at in first[:behind]:
        c.cache.k[at[0], at[1], :, 9] = -math.inf
    got = c.run(**kw)
    ks, vs = ([x[at] for at in first[behind:]] for x in (c.cache.k, c.cache.v))
    none = torch.zeros(0, hk, 128, dtype=c.q.dtype, device="cuda")
    ks, vs = (torch.stack(x) if x else none for x in (ks, vs))
    for b, n in enumerate(keep):
        own = [P.rows(x, c.table[b, :P.pages_of(n, page)], n) for x in (c.cache.k, c.cache.v)]
        k, v = torch.cat((ks, own[0])), torch.cat((vs, own[1]))
        if len(k) == 0:
            assert torch.all(got[b] == 0)
            continue
        r = R.attention(c.q[b:b + 1], k, v, [1], [len(k)], False, SCALE)
        R.assert_within("out", got[b:b + 1], r["out"], r["out_a"])
    # all of them: NaN where there are keys, of one's own or the prefix
    if prefix:
        for at in first[behind:]:
            c.cache.k[at[0], at[1], :, 9] = -math.inf
    for b, n in enumerate(lens):
        if b % 2:
            for row in range(keep[b]):
                c.cache.k[int(c.table[b, row // page]), row % page, :, 9] = -math.inf
    got = c.run(**kw)
    for b, n in enumerate(lens):
        if n and b % 2 == 0:
            own = [P.rows(x, c.table[b, :P.pages_of(keep[b], page)], keep[b]) for x in (c.cache.k, c.cache.v)]
            r = R.attention(c.q[b:b + 1], *own, [1], [keep[b]], False, SCALE)
            R.assert_within("out", got[b:b + 1], r["out"], r["out_a"])
        elif n or prefix:
            assert torch.isnan(got[b]).all()
        else:
            assert torch.all(got[b] == 0)


def test_a_score_of_infinity_is_nan():
    for prefix, splits in ((0, 0), (0, 3), (40, 0), (2000, 1)):
        c = Case([50, 20, 0, 3000], 8, 2, 16, prefix=prefix, seed=3)
        c.q[..., 9] = 1.0
        c.cache.k[int(c.table[0, 3]), 1, 1, 9] = math.inf         # its last key but one, of one head
        c.cache.k[int(c.table[3, 100]), 7, 0, 9] = math.inf
        got = c.run(num_splits=splits)
        nan = torch.zeros(4, 8, dtype=torch.bool, device="cuda")
        nan[0, 4:] = nan[3, :4] = True
        assert torch.equal(torch.isnan(got).all(-1), nan) and torch.equal(torch.isnan(got).any(-1), nan)


def test_lengths_of_a_prefix_that_end_inside_a_tile():
    """An infinite value in the last key of every length of the prefix that the device may hold."""
    c = Case([20, 0, 3] * 20, 12, 4, 16, prefix=1000, seed=4)
    for n in (1, 2, 15, 16, 17, 31, 33, 48, 63, 64, 65, 127, 129, 700, 999, 1000):
        at = (int(c.prefix_table[(n - 1) // 16]), (n - 1) % 16)
        clean = c.run(prefix_len=_i32([n]))
        old = c.cache.v[at].clone()
        c.cache.v[at[0], at[1], 2, 5] = math.inf
        got = c.run(prefix_len=_i32([n]))
        assert torch.all(got[:, 6:9, 5] == math.inf)
        got[:, 6:9, 5] = clean[:, 6:9, 5]
        assert torch.equal(got, clean)
        c.cache.v[at] = old
