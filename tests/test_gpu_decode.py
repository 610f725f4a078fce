"""attention_decode against the 64-bit definition."""
import math

import pytest
import torch

import packed_ref as R

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
SCALE = 1 / math.sqrt(128)


def _data(B, hq, hk, cap, seed, heat=1.5):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(B, hq, 128, generator=g) * (torch.rand(hq, 1, generator=g) * heat + 0.2)
    kv = torch.randn(2, B, cap, hk, 128, generator=g).to(BF).cuda()
    return q.to(BF).cuda(), kv[0], kv[1]


def _lens(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


CASES = [  # lens, capacity, heads, kv heads
    ([1], 1, 1, 1), ([0], 8, 2, 1), ([5], 8, 40, 8), ([500], 1024, 40, 8), ([31, 32, 33, 0, 64], 64, 12, 4),
    ([1000, 1, 129, 1023], 1024, 5, 1), ([2000, 3], 2048, 6, 3), ([700], 700, 3, 3), ([100, 90], 100, 66, 1),
    ([97], 128, 40, 1), ([4096], 5000, 2, 2), ([300] * 20, 301, 4, 2),
    ([7, 0, 40] * 50, 64, 2, 1),
]


@pytest.mark.parametrize("lens,cap,hq,hk", CASES)
@pytest.mark.parametrize("splits", [0, 1, 3])
def test_against_the_definition(lens, cap, hq, hk, splits):
    import lbw_amd
    q, k, v = _data(len(lens), hq, hk, cap, 1)
    out = lbw_amd.attention_decode(q, k, v, _lens(lens), num_splits=splits)
    want, allow = R.decode(q, k, v, lens, SCALE)
    R.assert_within("out", out, want, allow)


def test_many_pieces_scale_and_rising_scores():
    import lbw_amd
    q, k, v = _data(2, 8, 2, 3000, 2)
    k = (k * 0.1 + torch.linspace(-2, 2, 3000, device="cuda")[:, None, None] * q[:, None, ::4]).to(BF)
    for splits in (2, 17, 128):
        out = lbw_amd.attention_decode(q, k, v, _lens([3000, 2411]), softmax_scale=0.2, num_splits=splits)
        want, allow = R.decode(q, k, v, [3000, 2411], 0.2)
        R.assert_within("out", out, want, allow)


def test_lengths_outside_the_cache_are_limited_and_rows_behind_them_unread():
    import lbw_amd
    q, k, v = _data(4, 10, 2, 300, 3)
    lens = [300, 0, 41, 200]
    want = lbw_amd.attention_decode(q, k, v, _lens(lens))
    for b, n in enumerate(lens):
        k[b, n:] = float("nan")
        v[b, n:] = float("inf")
    got = lbw_amd.attention_decode(q, k, v, _lens([301, -7, 41, 200]))
    assert torch.equal(got, want) and torch.all(got[1] == 0)
    got = lbw_amd.attention_decode(q, k, v, _lens([2 ** 31 - 1, -2 ** 31, 41, 200]))
    assert torch.equal(got, want)


def test_strided_caches_and_out():
    import lbw_amd
    q, k, v = _data(3, 6, 2, 130, 4)
    want = lbw_amd.attention_decode(q, k, v, _lens([130, 64, 7]))
    big = torch.zeros(2, 3, 2, 140, 128, dtype=BF, device="cuda")     # head-major caches
    big[0, :, :, 3:133], big[1, :, :, 3:133] = k.transpose(1, 2), v.transpose(1, 2)
    k2, v2 = big[0, :, :, 3:133].transpose(1, 2), big[1, :, :, 3:133].transpose(1, 2)
    buf = torch.full((3, 7, 136), 5.0, dtype=BF, device="cuda")
    out = buf[:, :6, :128]
    assert lbw_amd.attention_decode(q, k2, v2, _lens([130, 64, 7]), out=out) is out
    assert torch.equal(out, want)
    out.fill_(5.0)
    assert torch.all(buf == 5.0)


def test_offsets_past_32_bits():
    """A cache of over 2^31 elements: the last sequence's rows lie past a 32-bit offset."""
    import lbw_amd
    cap, hk = 140000, 8
    q = torch.randn(17, 8, 128, device="cuda").to(BF)
    k = torch.zeros(17, cap, hk, 128, dtype=BF, device="cuda")
    assert k.numel() > 1 << 31
    v = k  # (one buffer for both: K = V)
    lens = [0] * 16 + [200]
    k[16, :200] = torch.randn(200, hk, 128, device="cuda").to(BF)
    out = lbw_amd.attention_decode(q, k, v, _lens(lens))
    want, allow = R.decode(q[16:], k[16:, :200], v[16:, :200], [200], SCALE)
    R.assert_within("out", out[16:], want, allow)
    assert torch.all(out[:16] == 0)
    # and far rows of one sequence
    k1 = k.view(1, 17 * cap, hk, 128)
    n = 17 * cap
    k1[0, -100:] = torch.randn(100, hk, 128, device="cuda").to(BF) * 3
    out = lbw_amd.attention_decode(q[:1], k1, k1, _lens([n]))
    qh, kh = q[0].double(), k1[0].transpose(0, 1)
    s = torch.stack([(kh[h].float() @ qh[h].float()) for h in range(hk)]).double() * SCALE
    p = torch.softmax(s, -1)
    want = torch.stack([(p[h, :, None].float() * kh[h].float()).double().sum(0) for h in range(hk)])
    size = torch.stack([(p[h, :, None].float() * kh[h].float().abs()).double().sum(0) for h in range(hk)])
    # P's and the output's roundings; the fp32 steps of 74000 tiles' additions, of order 2^-8 at most
    R.assert_within("far rows", out[0], want, R.H * want.abs() + 2 * R.H * size + 1e-6)


def test_no_sequences_and_refusals():
    import lbw_amd
    q, k, v = _data(2, 4, 2, 40, 5)
    assert lbw_amd.attention_decode(q[:0], k[:0], v[:0], _lens([])).shape == (0, 4, 128)
    assert torch.all(lbw_amd.attention_decode(q, k[:, :0], v[:, :0], _lens([3, 3])) == 0)
    with pytest.raises(RuntimeError, match="overlaps"):
        lbw_amd.attention_decode(q, k, v, _lens([3, 3]), out=q)
    with pytest.raises(RuntimeError, match="int32"):
        lbw_amd.attention_decode(q, k, v, _lens([3, 3]).cpu())
    with pytest.raises(RuntimeError, match="contiguous head dim"):
        lbw_amd.attention_decode(q, k.transpose(1, 3).contiguous().transpose(1, 3), v, _lens([3, 3]))
    x = q.detach().requires_grad_()
    out = lbw_amd.attention_decode(x, k, v, _lens([3, 3]))
    with pytest.raises(RuntimeError):
        out.float().sum().backward()


@pytest.mark.parametrize("splits", [0, 1, 3, 128])
def test_nan_and_infinite_scores_stay_in_their_heads(splits):
    """A query, keys or values that are not finite give NaN in the heads that read them, cut into pieces or
    not, and leave the bits of the others."""
    import lbw_amd
    lens = [2500, 0, 40, 1999]
    q, k, v = _data(4, 8, 2, 2500, 6)
    run = lambda q, k, v: lbw_amd.attention_decode(q, k, v, _lens(lens), num_splits=splits)  # noqa: E731
    want = run(q, k, v)
    q, k, v = q.clone(), k.clone(), v.clone()
    nan = torch.zeros(4, 8, dtype=torch.bool, device="cuda")
    q[0, 3] = float("nan")
    q[0, 5] = 3e38                            # scores of both infinities
    q[1, 0] = float("nan")                    # (no keys: 0 all the same)
    k[2, :40, 1] = float("nan")               # every key of kv head 1
    k[3, 512:1500, 0] = float("nan")          # whole pieces of kv head 0
    v[3, 1600, 1] = float("nan")
    nan[0, 3] = nan[0, 5] = True
    nan[2, 4:] = True
    nan[3] = True
    got = run(q, k, v)
    assert torch.equal(torch.isnan(got).all(-1), nan) and torch.equal(torch.isnan(got).any(-1), nan)
    assert torch.equal(got[~nan], want[~nan])
    # every key of every sequence
    k[:] = float("nan")
    got = run(*_data(4, 8, 2, 2500, 6)[:1], k, v)
    assert torch.isnan(got[[0, 2, 3]]).all() and torch.all(got[1] == 0)
