"""paged_append_ on a slice of a longer packed batch: sequences that begin before the slice's first token or end behind its
last one, as the same tokens with starts inside it."""
import pytest
import torch

import packed_ref as R
import paged_ref as P

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _append(tokens, starts, lens, page, width, hk=3, dim=128, bounds=True, seed=0):
    """A call's arguments, and what it leaves: (q, k pages, v pages, bounds)."""
    import lbw_amd
    g = torch.Generator().manual_seed(seed)
    q, k, v = torch.randn(tokens, 4 * hk, dim, generator=g).to(BF).cuda().split([2 * hk, hk, hk], 1)
    pages = len(lens) * width + 2
    table = torch.randperm(pages, generator=g).int()[:len(lens) * width].view(len(lens), width).cuda()
    pool = P.make_pool(pages, page, hk, dim, g)
    cache = lbw_amd.PagedKV(*pool, torch.stack((pool[0].amin(1), pool[0].amax(1)), 2).contiguous() if bounds else None)
    ang = torch.outer(torch.arange(500, dtype=torch.float64), 100.0 ** (-torch.arange(dim // 2, dtype=torch.float64) / dim))
    pos = torch.randint(0, 500, (tokens,), generator=g, dtype=torch.int32).cuda()
    out = torch.full((tokens, 2 * hk, dim), 7.0, dtype=BF, device="cuda")
    lbw_amd.paged_append_(cache, q, k, v, table, _i32(lens), lbw_amd.axis_rope(ang, device="cuda"), pos, starts=_i32(starts),
                          q_out=out, eps=1e-6)
    want = P.turned(k, None, R.token_angles(ang.cuda(), (dim // 2,), pos[:, None]), True, 1e-6, 1.0)
    return (out, cache.k, cache.v) + ((cache.bounds,) if bounds else ()), table.cpu(), (k, v, want)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 1024])
@pytest.mark.parametrize("bounds", [True, False])
@pytest.mark.parametrize("tokens,starts,lens", [
    (100, [-5, 100], [0]), (100, [-200, 100], [3]), (4, [-2, 2], [5]), (2, [-1, 1, 2], [15, 40]), (90, [-30, -7, 41, 90], [0, 9, 5]),
    (700, [-3, 300, 301, 900], [20, 0, 7]), (130, [-100, 200], [11]), (40, [-2 ** 31, -2 ** 31 + 5, 30, 40], [0, 0, 16])])
def test_starts_before_the_first_token(page, bounds, tokens, starts, lens):
    # row of token t: len + t - start
    inside = [min(max(s, 0), tokens) for s in starts]
    moved = [n + max(0, min(stop, tokens) - start) - max(0, min(stop, tokens) - max(start, 0)) if stop > 0 else n
             for n, start, stop in zip(lens, starts, starts[1:])]
    far = max(moved)
    if far > 100000:           # (rows past every table: nothing to be written there)
        width = 3
    else:
        width = P.pages_of(far + tokens, page) + 1
    got, table, (k, v, want) = _append(tokens, starts, lens, page, width, bounds=bounds)
    same, _, _ = _append(tokens, inside, moved, page, width, bounds=bounds)
    for a, b in zip(got, same):
        assert torch.equal(a, b)
    # and every token's row where the formula has it
    for b, (start, stop) in enumerate(zip(starts, starts[1:])):
        for t in range(max(start, 0), min(stop, tokens)):
            row = lens[b] + t - start
            if row // page >= width:
                continue
            at = int(table[b, row // page])
            R.assert_within(f"k of token {t}", got[1][at, row % page], want[t], R.head_norm_allow(want[t]))
            assert torch.equal(got[2][at, row % page], v[t])
            if bounds:
                assert (got[3][at, :, 0] <= got[1][at, row % page]).all() and (got[3][at, :, 1] >= got[1][at, row % page]).all()


def test_a_batch_in_slices_is_the_batch():
    """The tokens of three sequences in one call, and in calls over slices of them that share the starts' tensor."""
    import lbw_amd
    page, lens, starts = 16, [5, 0, 40], [0, 61, 80, 150]
    width = 9
    g = torch.Generator().manual_seed(4)
    q, k, v = torch.randn(150, 8, 128, generator=g).to(BF).cuda().split([4, 2, 2], 1)
    table = torch.arange(3 * width, dtype=torch.int32, device="cuda").view(3, width)
    rope = lbw_amd.axis_rope(lbw_amd.wan_rope_freqs(128, 512).cuda())
    caches = []
    for size in (150, 1, 7, 50, 149):
        cache = lbw_amd.paged_kv(3 * width, page, 2, bounds=True)
        for x in (cache.k, cache.v, cache.bounds):
            x.fill_(3.0)
        outs = []
        for at in range(0, 150, size):
            s = slice(at, min(150, at + size))
            outs.append(lbw_amd.paged_append_(cache, q[s], k[s], v[s], table, _i32(lens), rope,
                                              starts=_i32(starts) - at, eps=1e-6))
        caches.append((torch.cat(outs), cache.k, cache.v, cache.bounds))
    for c in caches[1:]:
        for a, b in zip(c, caches[0]):
            assert torch.equal(a, b)


@pytest.mark.parametrize("page", [16, 64, 128, 256])
@pytest.mark.parametrize("tokens", [1, 65, 100, 1000])
@pytest.mark.parametrize("bounds", [True, False])
def test_tokens_without_sequences_are_left_alone(page, tokens, bounds):
    import lbw_amd
    cache = lbw_amd.paged_kv(3, page, 2, bounds=bounds)
    q, k, v = torch.ones(tokens, 8, 128, dtype=BF, device="cuda").split([4, 2, 2], 1)
    rope = lbw_amd.axis_rope(lbw_amd.wan_rope_freqs(128, 2048).cuda())
    out = torch.full((tokens, 4, 128), 7.0, dtype=BF, device="cuda")
    table, none = torch.zeros(0, 2, dtype=torch.int32, device="cuda"), _i32([])
    assert lbw_amd.paged_append_(cache, q, k, v, table, none, rope, starts=_i32([0]), q_out=out) is out
    assert torch.all(out == 7) and not cache.k.any() and not cache.v.any() and (not bounds or not cache.bounds.any())
