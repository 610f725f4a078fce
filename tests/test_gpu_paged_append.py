"""paged_append_ against the 64-bit definition: rows, pages, bounds, what is left alone."""
import math

import pytest
import torch

import packed_ref as R
import paged_ref as P

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
POSITIONS = 4096   # rows of the rotation table, at least


def _rope(dim, rot, axes, inter, positions, device="cuda"):
    import lbw_amd
    n = rot // 2
    split = {1: (n,), 2: (n - n // 2, n // 2), 3: (n - 2 * (n // 3), n // 3, n // 3)}[axes]
    ang = torch.outer(torch.arange(positions, dtype=torch.float64),
                      100.0 ** (-torch.arange(n, dtype=torch.float64) / max(1, n)))
    return lbw_amd.axis_rope(ang, split, interleaved=inter, device=device), ang.to(device), split


class Case:
    def __init__(self, new, old, *, hq=4, hk=2, dim=128, rot=None, axes=1, inter=True, page=16, weights=None, eps=None,
                 bounds=True, decode=False, head_major=True, seed=0, spare_tokens=0, scales=(1.0, 1.0)):
        import lbw_amd
        g = torch.Generator().manual_seed(seed)
        self.new, self.old, self.page, self.eps, self.scales = new, old, page, eps, scales
        T = sum(new) + spare_tokens
        # (a row for every token of a sequence: the definition looks its angles up there)
        self.rope, self.ang, self.split = _rope(dim, dim if rot is None else rot, axes, inter,
                                                max(POSITIONS, *(o + n for o, n in zip(old, new))))
        self.inter = inter
        qkv = (torch.randn(T, hq + 2 * hk, dim, generator=g) * 1.7).to(BF).cuda()
        self.q, self.k, self.v = qkv.split([hq, hk, hk], 1)
        self.w = None
        if weights is not None:
            self.w = [(1 + 0.1 * torch.randn(dim, generator=g)).to(weights).cuda() for _ in range(2)]
        table, _, total = P.make_table([o + n for o, n in zip(old, new)], page, g)
        self.table = table.cuda()
        k, v = P.make_pool(total, page, hk, dim, g, head_major)
        edge = None
        if bounds:
            edge = torch.stack((k.amin(1), k.amax(1)), 2).contiguous()
        self.cache = lbw_amd.PagedKV(k, v, edge)
        self.lens = torch.tensor(old, dtype=torch.int32).cuda()
        self.starts = None if decode else torch.tensor([sum(new[:i]) for i in range(len(new) + 1)],
                                                       dtype=torch.int32).cuda()
        self.rows = [o + i for o, n in zip(old, new) for i in range(n)]
        self.pos = None if axes == 1 else torch.randint(0, POSITIONS, (T, axes), generator=g, dtype=torch.int32).cuda()

    def run(self, **kw):
        import lbw_amd
        wq, wk = self.w if self.w else (None, None)
        return lbw_amd.paged_append_(self.cache, self.q, self.k, self.v, self.table, self.lens, self.rope, self.pos,
                                     starts=self.starts, wq=wq, wk=wk, eps=self.eps, q_scale=self.scales[0],
                                     k_scale=self.scales[1], **kw)

    def want(self):
        n = len(self.rows)
        pos = torch.tensor(self.rows, device="cuda")[:, None] if self.pos is None else self.pos[:n]
        assert self.pos is not None or max(self.rows, default=0) < len(self.ang)
        ang = R.token_angles(self.ang, self.split, pos)
        wq, wk = self.w if self.w else (None, None)
        return (P.turned(self.q[:n], wq, ang, self.inter, self.eps, self.scales[0]),
                P.turned(self.k[:n], wk, ang, self.inter, self.eps, self.scales[1]))

    def check(self, before):
        """`before`: copies of the cache's tensors. Rows, then bounds, then everything else untouched."""
        q_out = self.got
        wq, wk = self.want()
        R.assert_within("q", q_out[:len(self.rows)], wq, R.head_norm_allow(wq))
        k, v, edge = before
        k, v = k.clone(), v.clone()
        table = self.table.cpu()
        t = 0
        for b, (o, n) in enumerate(zip(self.old, self.new)):
            fresh = {}
            for r in range(o, o + n):
                page, at = int(table[b, r // self.page]), r % self.page
                got = self.cache.k[page, at]
                R.assert_within(f"k of token {t}", got, wk[t], R.head_norm_allow(wk[t]))
                k[page, at], v[page, at] = got, self.v[t]
                lo, hi = fresh.get(page, (None, None))
                fresh[page] = (got, got) if lo is None else (torch.minimum(lo, got), torch.maximum(hi, got))
                t += 1
            if edge is not None:
                for page, (lo, hi) in fresh.items():
                    first = (table[b, :P.pages_of(o + n, self.page)].tolist()).index(page) * self.page
                    if first < o:   # begun before: joined with what was there
                        lo, hi = torch.minimum(lo, edge[page, :, 0]), torch.maximum(hi, edge[page, :, 1])
                    edge[page] = torch.stack((lo, hi), 1)
        assert torch.equal(self.cache.k, k) and torch.equal(self.cache.v, v)
        if edge is not None:
            assert torch.equal(self.cache.bounds, edge)

    def go(self, **kw):
        c = self.cache
        before = (c.k.clone(), c.v.clone(), None if c.bounds is None else c.bounds.clone())
        self.got = self.run(**kw)
        self.check(before)
        return self


@pytest.mark.parametrize("dim", [32, 64, 128, 256])
@pytest.mark.parametrize("eps,weights", [(None, None), (1e-6, None), (1e-6, BF), (1e-5, torch.float32)])
@pytest.mark.parametrize("inter,axes", [(True, 1), (False, 1), (True, 3), (False, 2)])
def test_one_token_per_sequence(dim, eps, weights, inter, axes):
    old = [0, 15, 16, 33, 700]
    Case([1] * 5, old, dim=dim, eps=eps, weights=weights, inter=inter, axes=axes, decode=True, seed=dim + axes).go()


@pytest.mark.parametrize("page", [16, 64, 1024])
@pytest.mark.parametrize("new,old", [
    ([1], [0]), ([17, 1, 60, 0, 33], [0, 63, 5, 40, 1000]), ([0, 0, 5], [3, 0, 0]), ([130], [15]),
    ([16, 16, 32], [0, 16, 8]), ([1] * 70, list(range(70))), ([3, 0] * 100, [5, 9] * 100), ([1100], [1000])])
def test_prompts(page, new, old):
    Case(new, old, page=page, eps=1e-6, weights=BF, seed=page).go()


@pytest.mark.parametrize("hq,hk,dim", [(40, 8, 128), (12, 12, 128), (5, 1, 64), (6, 3, 256), (33, 11, 32), (1, 1, 128)])
@pytest.mark.parametrize("decode", [True, False])
def test_heads(hq, hk, dim, decode):
    new = [1, 1, 1] if decode else [40, 7, 1]
    Case(new, [20, 0, 47], hq=hq, hk=hk, dim=dim, inter=False, decode=decode, seed=hq).go()


@pytest.mark.parametrize("decode", [True, False])
def test_half_a_head_turned_scales_no_bounds_and_strided_pages(decode):
    new = [1, 1] if decode else [30, 2]
    Case(new, [10, 31], rot=64, inter=False, scales=(0.3, 1.5), bounds=False, head_major=False, decode=decode).go()
    Case(new, [10, 31], rot=24, inter=True, head_major=False, decode=decode, seed=1).go()


def test_many_tokens():
    """More tokens than waves, a wave per token."""
    Case([9000, 7500, 1], [3, 100, 0], hq=2, hk=1, page=64, axes=3, eps=1e-6, weights=BF).go()


def test_tokens_behind_the_last_sequence_are_left_alone():
    c = Case([5, 0, 20], [0, 3, 30], spare_tokens=9)
    out = torch.full_like(c.q.contiguous(), 7.0)
    c.go(q_out=out)
    assert torch.all(out[25:] == 7.0)
    # and ahead of the first
    c = Case([5, 4], [0, 30], spare_tokens=3)
    c.q, c.k, c.v = (x.roll(3, 0) for x in (c.q, c.k, c.v))
    c.starts += 3
    out = torch.full_like(c.q, 7.0)
    before = (c.cache.k.clone(), c.cache.v.clone(), c.cache.bounds.clone())
    c.run(q_out=out)
    assert torch.all(out[:3] == 7.0)
    c.q, c.k, c.v, c.got = (x.roll(-3, 0) for x in (c.q, c.k, c.v, out))
    c.check(before)


@pytest.mark.parametrize("decode", [True, False])
def test_q_in_place_and_wide_tables(decode):
    c = Case([1] * 4 if decode else [20, 1, 0, 9], [0, 40, 3, 15], decode=decode)
    want = c.run()
    buf = torch.full((4, 50), -1, dtype=torch.int32, device="cuda")   # rows of a wider table
    buf[:, 3:3 + c.table.shape[1]] = c.table
    c.table = buf[:, 3:3 + c.table.shape[1]]
    q = c.q.clone()
    c.q = q
    assert c.run(q_out=q) is q and torch.equal(q, want)


@pytest.mark.parametrize("decode", [True, False])
def test_rows_and_pages_outside_are_not_written(decode):
    import lbw_amd
    n = [1] * 6 if decode else [2] * 6
    c = Case(n, [5] * 6, decode=decode, page=16)
    width, pages = c.table.shape[1], c.cache.k.shape[0]
    want = c.run()
    before = (c.cache.k.clone(), c.cache.v.clone(), c.cache.bounds.clone())
    # a page outside the cache, rows outside the table
    c.table[1, 0] = pages
    c.table[2, 0] = -1
    c.lens[3] = width * 16
    c.lens[4] = -10
    c.lens[5] = 2 ** 31 - 1
    pos = torch.full((sum(n),), 5, dtype=torch.int32, device="cuda")
    if not decode:
        pos[1::2] = 6
    c.pos = pos                                   # (as before: positions that do not follow the rows)
    got = c.run()
    assert torch.equal(got, want)                 # q is turned all the same
    for x, y in zip(before, (c.cache.k, c.cache.v, c.cache.bounds)):
        assert torch.equal(x, y)                  # the first sequence's rows are as they were, no other is touched
    # starts that lead nowhere
    if not decode:
        for bad in ([0] * 7, [100] * 7, [-5, -4, -3, -2, -1, 0, 0]):
            c.starts = torch.tensor(bad, dtype=torch.int32, device="cuda")
            lbw_amd.paged_append_(c.cache, c.q, c.k, c.v, c.table, c.lens, c.rope, c.pos, starts=c.starts)
            for x, y in zip(before, (c.cache.k, c.cache.v, c.cache.bounds)):
                assert torch.equal(x, y)


@pytest.mark.parametrize("decode", [True, False])
def test_positions_outside_the_table_and_nan(decode):
    c = Case([1, 1] if decode else [3, 40], [4, 10], decode=decode)
    c.pos = torch.arange(c.q.shape[0], dtype=torch.int32, device="cuda")
    c.pos[0], c.pos[1] = -1, POSITIONS
    out = c.run()
    assert torch.isnan(out[:2]).all() and torch.isfinite(out[2:]).all()
    page = int(c.table[0, 0])
    assert torch.isnan(c.cache.k[page, 4]).all() and torch.equal(c.cache.v[page, 4], c.v[0])
    assert torch.isnan(c.cache.bounds[page]).all()        # a key of NaN leaves no bounds
    # a single component, and infinities
    c = Case([1] if decode else [20], [3], decode=decode, hq=2, hk=2)
    c.pos = torch.zeros(c.q.shape[0], dtype=torch.int32, device="cuda")
    c.k = c.k.clone()
    c.k[-1, 0, 6] = float("inf")
    c.k[-1, 1, 8] = float("nan")
    c.run()
    page = int(c.table[0, (2 + c.q.shape[0]) // 16])
    edge = c.cache.bounds[page].float()
    assert edge[0, 1, 6] == math.inf and torch.isnan(edge[1, :, 8]).all()
    assert torch.isfinite(edge[1, :, :8]).all() and torch.isfinite(edge[0, :, 9:]).all()


def test_same_bits_on_every_run_and_again_on_the_same_rows():
    c = Case([33, 200, 1], [20, 7, 64], eps=1e-6, weights=BF)
    out = c.run()
    first = [x.clone() for x in (c.cache.k, c.cache.v, c.cache.bounds)]
    for _ in range(5):
        assert torch.equal(c.run(), out)
        for x, y in zip(first, (c.cache.k, c.cache.v, c.cache.bounds)):
            assert torch.equal(x, y)


def test_one_by_one_is_all_at_once():
    """A prompt in one call, in pieces, and token by token: the same bits, bounds too."""
    import lbw_amd
    c = Case([75], [0], eps=1e-6, weights=BF, page=16)
    out = c.run()
    first = [x.clone() for x in (c.cache.k, c.cache.v, c.cache.bounds)]
    for step in (1, 7, 32):
        for x in (c.cache.k, c.cache.v, c.cache.bounds):
            x.fill_(3.0)
        for t in range(0, 75, step):
            n = min(step, 75 - t)
            s = slice(t, t + n)
            starts = None if step == 1 else torch.tensor([0, n], dtype=torch.int32, device="cuda")
            got = lbw_amd.paged_append_(c.cache, c.q[s], c.k[s], c.v[s], c.table,
                                        torch.tensor([t], dtype=torch.int32, device="cuda"), c.rope, starts=starts,
                                        wq=c.w[0], wk=c.w[1], eps=1e-6)
            assert torch.equal(got, out[s])
        for b in range(5):
            page, n = int(c.table[0, b]), min(16, 75 - 16 * b)
            assert torch.equal(c.cache.k[page, :n], first[0][page, :n])
            assert torch.equal(c.cache.v[page, :n], first[1][page, :n])
            assert torch.equal(c.cache.bounds[page], first[2][page])


def test_offsets_past_32_bits():
    import lbw_amd
    page, hk = 1024, 8
    pages = (1 << 31) // (page * hk * 128) + 3
    cache = lbw_amd.paged_kv(pages, page, hk, bounds=True)
    assert cache.k.numel() > 1 << 31
    rope, ang, split = _rope(128, 128, 1, True, 64)
    g = torch.Generator().manual_seed(3)
    qkv = torch.randn(30, 4 * hk, 128, generator=g).to(BF).cuda()
    q, k, v = qkv.split([2 * hk, hk, hk], 1)
    table = torch.tensor([[pages - 1, 0], [pages - 2, 0]], dtype=torch.int32).cuda()
    lens = torch.tensor([1000, 900], dtype=torch.int32).cuda()
    starts = torch.tensor([0, 20, 30], dtype=torch.int32).cuda()
    pos = torch.arange(30, dtype=torch.int32).cuda()
    lbw_amd.paged_append_(cache, q, k, v, table, lens, rope, pos, starts=starts)
    want = P.turned(k, None, R.token_angles(ang, split, pos), True, None, 1.0)
    got = torch.cat((cache.k[pages - 1, 1000:1020], cache.k[pages - 2, 900:910]))
    R.assert_within("far rows", got, want, R.head_norm_allow(want))
    assert torch.equal(cache.v[pages - 1, 1000:1020], v[:20])
    assert torch.all(cache.k[:pages - 2, ::97] == 0) and torch.all(cache.k[pages - 1, :1000] == 0)
    assert torch.equal(cache.bounds[pages - 1, :, 1], torch.cat((cache.k[pages - 1, 1000:1020],
                                                                torch.zeros_like(k[:1]))).amax(0))


def test_no_tokens_and_refusals():
    import lbw_amd
    c = Case([3, 4], [1, 2])
    none = torch.zeros(3, dtype=torch.int32, device="cuda")
    out = lbw_amd.paged_append_(c.cache, c.q[:0], c.k[:0], c.v[:0], c.table, c.lens, c.rope, starts=none)
    assert out.shape == (0, 4, 128)
    args = (c.cache, c.q, c.k, c.v, c.table, c.lens, c.rope)
    with pytest.raises(RuntimeError, match="overlaps"):
        lbw_amd.paged_append_(*args, starts=c.starts, q_out=c.q.as_strided(c.q.shape, (8 * 128, 128, 1), 128))
    with pytest.raises(RuntimeError, match="overlaps"):
        lbw_amd.paged_append_(lbw_amd.PagedKV(c.cache.k, c.cache.k, c.cache.bounds), *args[1:], starts=c.starts)
    with pytest.raises(RuntimeError, match="several elements"):
        lbw_amd.paged_append_(lbw_amd.PagedKV(c.cache.k, c.cache.v[:, :1].expand(-1, 16, -1, -1), c.cache.bounds),
                              *args[1:], starts=c.starts)
    with pytest.raises(RuntimeError, match="int32"):
        lbw_amd.paged_append_(*args[:5], c.lens.cpu(), c.rope, starts=c.starts)
    with pytest.raises(RuntimeError, match="contiguous rows"):
        lbw_amd.paged_append_(*args[:4], c.table.T.contiguous().T, c.lens, c.rope, starts=c.starts)
    w = torch.ones(128, dtype=BF, device="cuda", requires_grad=True)
    with pytest.raises(NotImplementedError, match="not differentiable"):
        lbw_amd.paged_append_(*args, starts=c.starts, wq=w, wk=w, eps=1e-6)
    with torch.no_grad():
        lbw_amd.paged_append_(*args, starts=c.starts, wq=w, wk=w, eps=1e-6)
    # a write is counted
    x = c.cache.k.detach()
    n = x._version
    lbw_amd.paged_append_(*args, starts=c.starts)
    assert c.cache.k._version > n and c.cache.bounds._version > 0


@pytest.mark.parametrize("hq,hk,dim,inter", [(3, 3, 128, True), (10, 5, 64, False), (7, 7, 32, True), (6, 3, 256, False)])
@pytest.mark.parametrize("page,new", [(16, [1500, 0, 1100]), (32, [2600, 900]), (64, [7000, 33]), (128, [300, 90]), (16, [9, 40])])
def test_many_pages_and_few_with_odd_heads(hq, hk, dim, inter, page, new):
    """Pages whose keys are looked after one head and two at a time, an odd one last, or by a kernel of its own."""
    Case(new, [5 + 30 * i for i in range(len(new))], hq=hq, hk=hk, dim=dim, inter=inter, page=page, eps=1e-6, weights=BF,
         seed=dim + page).go()


@pytest.mark.parametrize("page", [16, 64, 128])
@pytest.mark.parametrize("new,old", [
    ([20, 0, 40, 1], [3, 9, 0, 16]), ([150, 300], [70, 0]), ([0] * 70 + [5] + [0] * 130 + [3, 0], [1] * 203),
    ([16, 0, 64, 128, 127], [0, 0, 64, 128, 1]), ([33] * 80, list(range(80))), ([0, 0, 0], [5, 0, 1])])
def test_tokens_before_the_first_sequence_are_left_alone(page, new, old):
    """The same tokens behind others that belong to nobody, to the bit; among empty sequences too."""
    import lbw_amd
    lead = 9
    c = Case(new, old, page=page, spare_tokens=lead + 4, axes=2, eps=1e-6, weights=BF, seed=page)
    args = (c.table, c.lens, c.rope)
    outs, caches = [], []
    for shift in (0, lead):
        cache = lbw_amd.PagedKV(c.cache.k.clone(), c.cache.v.clone(), c.cache.bounds.clone())
        part = slice(lead - shift, None)
        q = c.q[part]
        out = torch.full(q.shape, 3.0, dtype=BF, device="cuda")
        lbw_amd.paged_append_(cache, q, c.k[part], c.v[part], *args, c.pos[part], starts=c.starts + shift, q_out=out,
                              wq=c.w[0], wk=c.w[1], eps=1e-6)
        assert (out[:shift] == 3).all() and (out[shift + sum(new):] == 3).all()
        outs.append(out[shift:])
        caches.append(cache)
    assert torch.equal(*outs)
    for n in ("k", "v", "bounds"):
        assert torch.equal(getattr(caches[0], n), getattr(caches[1], n))
    # and as the definition has it
    c.q, c.k, c.v, c.pos = (x[lead:] for x in (c.q, c.k, c.v, c.pos))
    if sum(new):
        c.go()
