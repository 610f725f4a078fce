"""attention_packed and its gradient against the 64-bit definition."""
import math

import pytest
import torch

import packed_ref as R

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
SCALE = 1 / math.sqrt(128)


def _data(ql, kl, hq, hk, seed, heat=1.5):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda n, h: torch.randn(n, h, 128, generator=g)  # noqa: E731
    t = torch.rand(hq, 1, generator=g) * heat + 0.2
    q, k, v, do = rnd(sum(ql), hq) * t, rnd(sum(kl), hk), rnd(sum(kl), hk), rnd(sum(ql), hq)
    return [x.to(BF).cuda() for x in (q, k, v, do)]


def _run(q, k, v, do, ql, kl, causal, scale=None):
    import lbw_amd
    plan = lbw_amd.packed_plan(ql, kl, causal=causal)
    out, lse = lbw_amd.attention_packed(q, k, v, plan, softmax_scale=scale, return_lse=True)
    grads = lbw_amd.attention_packed_backward(do, q, k, v, out, lse, plan, softmax_scale=scale)
    return dict(zip(("out", "lse", "dq", "dk", "dv"), (out, lse) + tuple(grads)))


def _compare(got, want):
    for n in ("out", "dq", "dk", "dv"):
        R.assert_within(n, got[n], want[n], want[n + "_a"])
    empty = want["lse"] == -math.inf
    assert torch.equal(got["lse"] == -math.inf, empty)
    R.assert_within("lse", got["lse"][~empty], want["lse"][~empty], want["lse_a"][~empty])


CASES = [  # q_lens, k_lens, heads, kv heads, causal
    ([1], [1], 1, 1, True), ([17, 1, 60, 0, 33], None, 3, 1, True), ([128], None, 2, 2, True),
    ([129, 64, 65], None, 2, 1, True), ([127, 128, 256, 63], None, 5, 1, False),
    ([1, 1, 1], [700, 1, 64], 4, 2, True), ([300], [1000], 2, 2, True), ([511, 37], None, 6, 3, True),
    ([200, 5], [37, 0], 2, 1, True), ([200, 5], [37, 0], 2, 1, False), ([0, 3], [9, 200], 2, 2, True),
    ([2, 130], [130, 2], 3, 3, True), ([640], [641], 1, 1, True), ([64, 32, 96], [64, 96, 32], 2, 1, True),
    ([1025, 3, 258], None, 8, 2, True), ([33] * 40, None, 1, 1, True),
    # few rows over many keys, many queries over few keys: items cut into pieces (up to 16)
    ([16], [3000], 2, 1, True), ([5, 2, 130], [2500, 10, 700], 1, 1, False), ([2200], [70], 6, 1, False),
    ([1, 129], [9000, 129], 1, 1, True), ([5000, 40], [33, 40], 1, 1, True),
    # few items of keys: 64 of them per workgroup, whole and in pieces; items of 64 and 65 keys
    ([448, 65], None, 3, 1, True), ([449], [320], 4, 2, False), ([1300], None, 8, 1, True),
    # equal items, more than run at once: those of the last round are cut
    ([129, 300], [4100, 4200], 130, 130, True), ([4200], [385], 65, 65, False),
]


@pytest.mark.parametrize("ql,kl,hq,hk,causal", CASES)
def test_forward_and_gradient(ql, kl, hq, hk, causal):
    kl = ql if kl is None else kl
    q, k, v, do = _data(ql, kl, hq, hk, 1)
    _compare(_run(q, k, v, do, ql, kl, causal),
             R.attention(q, k, v, ql, kl, causal, SCALE, do))


@pytest.mark.parametrize("scale", [0.003, 1.0])
def test_other_scales_with_peaked_rows(scale):
    ql = kl = [150, 90]
    q, k, v, do = _data(ql, kl, 4, 2, 2, heat=3.0)
    _compare(_run(q, k, v, do, ql, kl, True, scale), R.attention(q, k, v, ql, kl, True, scale, do))


@pytest.mark.parametrize("causal", [True, False])
def test_rising_scores_move_the_reference_late(causal):
    """Keys sorted by their score: the running reference moves in every tile, by hundreds at the end."""
    ql = kl = [400]
    q, k, v, do = _data(ql, kl, 2, 1, 3)
    q = torch.ones_like(q) * q[:1]
    k = (k * 0.1 + torch.linspace(-3, 3, 400, device="cuda")[:, None, None] * q[:1, :1]).to(BF)
    _compare(_run(q, k, v, do, ql, kl, causal), R.attention(q, k, v, ql, kl, causal, SCALE, do))


def test_strided_views_of_a_fused_projection():
    ql = kl = [70, 131]
    hq, hk = 6, 2
    g = torch.Generator().manual_seed(4)
    qkv = torch.randn(201, hq + 2 * hk, 128, generator=g).to(BF).cuda()
    q, k, v = qkv.split([hq, hk, hk], 1)
    do = torch.randn(hq, 201, 128, generator=g).to(BF).cuda().transpose(0, 1)
    _compare(_run(q, k, v, do, ql, kl, True), R.attention(q, k, v, ql, kl, True, SCALE, do))


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_a_sequence_never_reaches_its_neighbours(bad):
    ql, kl = [70, 50, 65], [100, 50, 65]
    q, k, v, do = _data(ql, kl, 4, 2, 5)
    want = _run(q, k, v, do, ql, kl, True)
    qs, ks = slice(70, 120), slice(100, 150)
    for x, s in ((q, qs), (k, ks), (v, ks), (do, qs)):
        x[s] = bad
    got = _run(q, k, v, do, ql, kl, True)
    for n in ("out", "dq"):
        assert torch.equal(got[n][:70], want[n][:70]) and torch.equal(got[n][120:], want[n][120:])
    for n in ("dk", "dv"):
        assert torch.equal(got[n][:100], want[n][:100]) and torch.equal(got[n][150:], want[n][150:])


def test_rows_around_the_packed_ones_are_left_alone():
    """Through the C entry: outputs inside larger buffers keep what is around them."""
    import ctypes
    import lbw_amd
    from lbw_amd import _lib
    ql, kl = [70, 31], [70, 90]
    q, k, v, do = _data(ql, kl, 4, 2, 6)
    plan = lbw_amd.packed_plan(ql, kl)
    want = _run(q, k, v, do, ql, kl, True)

    def framed(t):
        b = torch.full((t.shape[0] + 9, t.shape[1] + 1, 136), 3.0, dtype=BF, device="cuda")
        return b, b[4:4 + t.shape[0], :t.shape[1], :128]
    out_b, out = framed(q)
    dq_b, dq = framed(q)
    dk_b, dk = framed(k)
    dv_b, dv = framed(v)
    lse = torch.empty(4, 101, device="cuda")
    p = _lib.PackedParams(q_heads=4, k_heads=2, head_dim=128, q_tokens=101, k_tokens=160,
                          lse=lse.data_ptr(), q_items=plan.q_items.data_ptr(),
                          n_q_items=plan.q_items.shape[0], k_items=plan.k_items.data_ptr(),
                          n_k_items=plan.k_items.shape[0])
    g = _lib.PackedGrads()
    for s, n, t in ((p, "q", q), (p, "k", k), (p, "v", v), (p, "out", out), (g, "dout", do), (g, "dq", dq),
                    (g, "dk", dk), (g, "dv", dv)):
        setattr(s, n, t.data_ptr())
        setattr(s, n + "_stride_l", t.stride(0))
        setattr(s, n + "_stride_h", t.stride(1))
    lib = _lib.load()
    stream = _lib.stream_ptr()
    assert lib.lbw_attention_packed_workspace_size(ctypes.byref(p)) == 0  # (no tile counts: never cut)
    _lib.check(lib.lbw_attention_packed_fwd(ctypes.byref(p), None, 0, stream), "fwd")
    n = lib.lbw_attention_packed_bwd_workspace_size(ctypes.byref(p))
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    assert lib.lbw_attention_packed_bwd(ctypes.byref(p), ctypes.byref(g), ws.data_ptr(), n - 1, stream) == 4
    _lib.check(lib.lbw_attention_packed_bwd(ctypes.byref(p), ctypes.byref(g), ws.data_ptr(), n, stream), "bwd")
    for name, b, t in (("out", out_b, out), ("dq", dq_b, dq), ("dk", dk_b, dk), ("dv", dv_b, dv)):
        assert torch.equal(t, want[name])
        t.fill_(3.0)
        assert torch.all(b == 3.0)
    assert torch.equal(lse, want["lse"])


def test_same_bits_every_run():
    ql = kl = [333, 128, 700]
    q, k, v, do = _data(ql, kl, 6, 2, 7)
    first = _run(q, k, v, do, ql, kl, True)
    for _ in range(3):
        again = _run(q, k, v, do, ql, kl, True)
        assert all(torch.equal(first[n], again[n]) for n in first)


def test_autograd_gives_the_explicit_gradients():
    import lbw_amd
    ql = kl = [90, 200]
    q, k, v, do = _data(ql, kl, 4, 2, 8)
    want = _run(q, k, v, do, ql, kl, True)
    plan = lbw_amd.packed_plan(ql)
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    out = lbw_amd.attention_packed(*leaves, plan)
    assert torch.equal(out, want["out"])
    out.backward(do)
    for x, n in zip(leaves, ("dq", "dk", "dv")):
        assert torch.equal(x.grad, want[n])
    # a gradient broadcast over the rows; v alone wanted
    out, lse = lbw_amd.attention_packed(q, k, leaves[2], plan, return_lse=True)
    assert not lse.requires_grad
    row = do[:1]
    gv, = torch.autograd.grad(out, leaves[2], row.expand_as(out))
    ref = lbw_amd.attention_packed_backward(row.expand_as(out).contiguous(), q, k, v, want["out"],
                                            want["lse"], plan)[2]
    assert torch.equal(gv, ref)
    # no second derivatives
    out = lbw_amd.attention_packed(*leaves, plan)
    g, = torch.autograd.grad(out.float().square().sum(), leaves[0], create_graph=True)
    with pytest.raises(RuntimeError):
        g.float().sum().backward()
    with torch.no_grad():
        assert not lbw_amd.attention_packed(*leaves, plan).requires_grad


def test_head_dim_that_is_not_contiguous_is_copied():
    import lbw_amd
    ql = kl = [40, 9]
    q, k, v, do = _data(ql, kl, 4, 2, 11)
    want = _run(q, k, v, do, ql, kl, True)
    leaves = [x.transpose(1, 2).contiguous().requires_grad_() for x in (q, k, v)]
    out = lbw_amd.attention_packed(*[x.transpose(1, 2) for x in leaves], lbw_amd.packed_plan(ql))
    assert torch.equal(out, want["out"])
    for g, n in zip(torch.autograd.grad(out, leaves, do), ("dq", "dk", "dv")):
        assert torch.equal(g.transpose(1, 2), want[n])


def test_more_than_2_31_elements():
    """Many sequences whose packed rows pass 2^31 elements of q: the last one against the definition."""
    import lbw_amd
    lens, hq = [90] * 3000, 63
    n = sum(lens)
    q = torch.empty(n, hq, 128, dtype=BF, device="cuda").normal_()
    assert q.numel() > 1 << 31
    k, v = torch.randn(n, 1, 128, device="cuda").to(BF), torch.randn(n, 1, 128, device="cuda").to(BF)
    plan = lbw_amd.packed_plan(lens)
    out, lse = lbw_amd.attention_packed(q, k, v, plan, return_lse=True)
    dq, dk, dv = lbw_amd.attention_packed_backward(out, q, k, v, out, lse, plan)  # (dout = out)
    s = slice(n - 90, n)
    r = R.attention(q[s], k[s], v[s], [90], [90], True, SCALE, out[s])
    R.assert_within("out", out[s], r["out"], r["out_a"])
    for name, x in (("dq", dq), ("dk", dk), ("dv", dv)):
        R.assert_within(name, x[s], r[name], r[name + "_a"])


def test_nothing_to_do():
    import lbw_amd
    q, k, v, do = _data([0], [5], 4, 2, 9)
    got = _run(q, k, v, do, [0], [5], True)
    assert got["out"].shape == (0, 4, 128) and torch.all(got["dk"] == 0) and torch.all(got["dv"] == 0)
    got = _run(do.new_ones(3, 4, 128), k[:0], v[:0], do.new_ones(3, 4, 128), [3], [0], False)
    assert torch.all(got["out"] == 0) and torch.all(got["dq"] == 0) and torch.all(got["lse"] == -math.inf)
    plan = lbw_amd.packed_plan([])
    assert lbw_amd.attention_packed(q, k[:0], v[:0], plan).shape == (0, 4, 128)


def test_one_tensor_as_keys_and_values_and_heads_that_are_expanded():
    import lbw_amd
    ql = [70, 33]
    q, k, _, do = _data(ql, ql, 4, 2, 13)
    plan = lbw_amd.packed_plan(ql)
    want = R.attention(q, k, k, ql, ql, True, SCALE, do)
    x = k.detach().requires_grad_()
    g, = torch.autograd.grad(lbw_amd.attention_packed(q, x, x, plan), x, do)
    # two gradients, each within its allowance, and the rounding of their sum
    total = want["dk"] + want["dv"]
    R.assert_within("dk + dv", g, total, (1 + R.H) * (want["dk_a"] + want["dv_a"]) + R.H * total.abs())
    one = k[:, :1].detach().requires_grad_()
    wide = one.expand(-1, 2, -1)  # head stride 0
    out = lbw_amd.attention_packed(q, wide, wide, plan)
    same = lbw_amd.attention_packed(q, wide.detach().contiguous(), wide.detach().contiguous(), plan)
    assert torch.equal(out, same)
    g, = torch.autograd.grad(out, one, do)
    assert g.shape == one.shape and torch.isfinite(g).all()


def test_a_plan_of_other_lengths_stays_inside_the_tensors():
    """An op cannot see whose table it gets: items that do not fit are skipped, not followed."""
    import lbw_amd
    big = lbw_amd.packed_plan([4000, 100])
    q, k, v, _ = _data([60], [60], 2, 1, 10)
    info = (60, 60) + big.info[2:]
    out, _ = torch.ops.lbw.attention_packed(q, k, v, big.q_items, big.k_items, info, 0.0, True)
    torch.cuda.synchronize()
    assert out.shape == q.shape
    with pytest.raises(RuntimeError, match="the plan is for 4100"):
        torch.ops.lbw.attention_packed(q, k, v, big.q_items, big.k_items, big.info, 0.0, True)
    with pytest.raises(ValueError, match="the plan"):
        lbw_amd.attention_packed(q, k, v, big)
    with pytest.raises(ValueError, match="plan is on"):
        lbw_amd.attention_packed(q, k, v, lbw_amd.packed_plan([60], device="cpu"))


@pytest.mark.parametrize("ql,kl", [([70], [70]), ([16], [3000]), ([200, 5], [37, 2])])
def test_a_query_that_is_nan_has_a_nan_lse(ql, kl):
    """Only a query that sees no key has lse -inf; the other rows stay within their allowance."""
    import lbw_amd
    q, k, v, _ = _data(ql, kl, 2, 1, 14)
    want = R.attention(q, k, v, ql, kl, True, SCALE)
    plan = lbw_amd.packed_plan(ql, kl)
    rows = [0, ql[0] - 1]
    q = q.clone()
    q[rows, 1] = float("nan")
    out, lse = lbw_amd.attention_packed(q, k, v, plan, return_lse=True)
    for r in rows:
        if want["lse"][1, r] == -math.inf:    # sees no key
            assert lse[1, r] == -math.inf and torch.all(out[r, 1] == 0)
        else:
            assert torch.isnan(lse[1, r]) and torch.isnan(out[r, 1]).all()
    keep = torch.ones(2, sum(ql), dtype=torch.bool, device="cuda")
    keep[1, rows] = False
    R.assert_within("out", out[keep.T], want["out"][keep.T], want["out_a"][keep.T])
    keep &= want["lse"] != -math.inf
    R.assert_within("lse", lse[keep], want["lse"][keep], want["lse_a"][keep])


def test_head_dim_that_is_not_contiguous_is_copied_without_autograd_too():
    import lbw_amd
    ql = kl = [40, 9]
    q, k, v, do = _data(ql, kl, 4, 2, 11)
    want = _run(q, k, v, do, ql, kl, True)
    plan = lbw_amd.packed_plan(ql)
    with torch.inference_mode():
        xs = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v)]
        out, lse = lbw_amd.attention_packed(*xs, plan, return_lse=True)
        grads = lbw_amd.attention_packed_backward(do.clone(), *xs, out, lse, plan)
    for n, x in zip(("out", "lse", "dq", "dk", "dv"), (out, lse) + tuple(grads)):
        assert torch.equal(x, want[n])


@pytest.mark.parametrize("scale", [1e-30, 1e-6, 1e3, 1e6, 1e8])
def test_rows_without_keys_at_every_scale(scale):
    import lbw_amd
    ql, kl = [200, 5], [37, 2]
    q, k, v, _ = _data(ql, kl, 4, 2, 15)
    if scale > 1e6:  # ordinary scores times it leave what fp32 holds of an exponent: 0 and NaN
        with pytest.raises(RuntimeError, match="softmax_scale"):
            lbw_amd.attention_packed(q, k, v, lbw_amd.packed_plan(ql, kl), softmax_scale=scale)
        return
    out, lse = lbw_amd.attention_packed(q, k, v, lbw_amd.packed_plan(ql, kl), softmax_scale=scale, return_lse=True)
    none = torch.zeros(205, dtype=torch.bool, device="cuda")
    none[:163] = none[200:203] = True
    assert torch.all(out[none] == 0) and torch.equal(lse == -math.inf, none.expand(4, 205))
