"""qk_head_norm_rope and its gradient against the 64-bit definition."""
import pytest
import torch

import packed_ref as R

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _data(T, hq, hk, d, seed, w_dtype=BF, gain=2.0):
    g = torch.Generator().manual_seed(seed)
    qkv = (torch.randn(T, (hq + 2 * hk) * d, generator=g) * gain).to(BF).cuda()
    q = qkv[:, :hq * d].unflatten(1, (hq, d))
    k = qkv[:, hq * d:(hq + hk) * d].unflatten(1, (hk, d))
    v = qkv[:, (hq + hk) * d:].unflatten(1, (hk, d))
    w = [(1 + 0.2 * torch.randn(d, generator=g)).to(w_dtype).cuda() for _ in range(2)]
    return q, k, v, w


def _rope(axes, rows, inter, seed=0):
    import lbw_amd
    g = torch.Generator().manual_seed(100 + seed)
    ang = (torch.rand(rows, sum(axes), generator=g) * 50 - 25).cuda()
    return ang, lbw_amd.axis_rope(ang, axes, interleaved=inter)


def _pos(T, axes, rows, seed=0):
    g = torch.Generator().manual_seed(200 + seed)
    return torch.randint(0, rows, (T, len(axes)), generator=g, dtype=torch.int32).cuda()


CASES = [  # T, hq, hk, d, axes, interleaved, weights
    (1, 1, 1, 32, (16,), True, BF), (3, 5, 1, 64, (8,), False, BF), (67, 40, 8, 128, (22, 21, 21), True, BF),
    (130, 12, 12, 128, (64,), False, torch.float32), (257, 6, 3, 256, (40, 24), False, BF),
    (9, 3, 3, 128, (5, 1, 4, 3), True, torch.float32), (33, 7, 7, 64, (0, 32), True, None),
    (5000, 2, 1, 128, (30, 10), True, BF), (4, 33, 11, 32, (0,), True, BF),
]


@pytest.mark.parametrize("T,hq,hk,d,axes,inter,wd", CASES)
def test_forward_and_gradient(T, hq, hk, d, axes, inter, wd):
    import lbw_amd
    q, k, _, w = _data(T, hq, hk, d, T + d, wd or BF)
    w = w if wd is not None else [None, None]
    ang, rope = _rope(axes, 50, inter)
    pos = _pos(T, axes, 50)
    qs, ks, eps = 0.7, 1.0, 1e-5
    q, k = q.detach().requires_grad_(), k.detach().requires_grad_()
    for x in w:
        if x is not None:
            x.requires_grad_()
    q2, k2 = lbw_amd.qk_head_norm_rope(q, k, w[0], w[1], rope, pos, eps, q_scale=qs, k_scale=ks)
    g = torch.Generator().manual_seed(7)
    # gradients as a network hands them back: another layout, and one broadcast over the heads
    dq2 = torch.randn(hq, T, d, generator=g).to(BF).cuda().transpose(0, 1)
    dk2 = torch.randn(T, 1, d, generator=g).to(BF).cuda().expand(T, hk, d)
    leaves = [x for x in (q, k, *w) if x is not None]
    grads = torch.autograd.grad((q2, k2), leaves, (dq2, dk2))
    a = R.token_angles(ang, axes, pos)
    for n, (x, y, dy, ww, s) in enumerate(((q, q2, dq2, w[0], qs), (k, k2, dk2, w[1], ks))):
        X = x.detach().double().requires_grad_()
        W = ww.detach().double().requires_grad_() if ww is not None else None
        Y = R.head_norm(X, W, a, inter, eps, s)
        R.assert_within("qk"[n] + "'", y, Y.detach(), R.head_norm_allow(Y.detach()))
        G = torch.autograd.grad(Y, [X] if W is None else [X, W], dy.double())
        # r (g w - x r mean(g w x r)): before the one rounding an fp32 sum over the head (d <= 256 terms)
        # of products; 2^10 E of the sizes of the two terms
        r = torch.rsqrt(X.detach().square().mean(-1, keepdim=True) + eps)
        gw = R.rotate(dy.double(), a.cos(), -a.sin(), inter).abs() * s
        gw = gw * (W.detach().abs() if W is not None else 1)
        size = r * (gw.amax(-1, keepdim=True) +
                    (X.detach().abs() * r).amax(-1, keepdim=True) *
                    (gw * X.detach().abs() * r).mean(-1, keepdim=True))
        R.assert_within("d" + "qk"[n], grads[n], G[0], R.H * G[0].abs() + 2 ** 10 * R.E * size)
        if W is not None:
            terms = (R.rotate(dy.double(), a.cos(), -a.sin(), inter) * s * X.detach() * r).abs().sum((0, 1))
            half = R.H if ww.dtype == BF else R.E
            # each lane adds its tokens in turn, then lanes, waves and workgroups: no term passes
            # through more than T + 200 additions
            R.assert_within("dw" + "qk"[n], grads[2 + n], G[1],
                            half * G[1].abs() + (T + 200) * R.E * terms)


def test_same_bits_every_run():
    import lbw_amd
    q, k, _, w = _data(3001, 12, 4, 128, 5)
    _, rope = _rope((64,), 3001, False)
    pos = torch.arange(3001, dtype=torch.int32, device="cuda")
    leaves = [x.detach().requires_grad_() for x in (q, k, *w)]
    out = []
    for _ in range(3):
        y = lbw_amd.qk_head_norm_rope(*leaves, rope, pos)
        out.append(y + torch.autograd.grad(y, leaves, (y[0].detach(), y[1].detach())))
    for o in out[1:]:
        assert all(torch.equal(x, y) for x, y in zip(out[0], o))


def test_only_one_output_used_and_int_edges():
    import lbw_amd
    q, k, _, w = _data(8, 4, 2, 64, 6)
    _, rope = _rope((32,), 8, True)
    pos = torch.arange(8, dtype=torch.int32, device="cuda")
    leaves = [x.detach().requires_grad_() for x in (q, k, *w)]
    y = lbw_amd.qk_head_norm_rope(*leaves, rope, pos)
    g = torch.autograd.grad(y[0], leaves, torch.ones_like(y[0]))
    assert torch.all(g[1] == 0) and torch.all(g[3] == 0) and g[0].abs().max() > 0
    # no tokens
    y = lbw_amd.qk_head_norm_rope(leaves[0][:0], leaves[1][:0], leaves[2], leaves[3], rope, pos[:0])
    assert y[0].shape == (0, 4, 64)
    g = torch.autograd.grad(y[0].sum() + y[1].sum(), leaves[2:])
    assert all(torch.all(x == 0) for x in g)


def test_position_outside_the_table_is_nan_only_there():
    import lbw_amd
    q, k, _, w = _data(4, 2, 2, 128, 8)
    _, rope = _rope((20, 12), 10, True)
    pos = torch.tensor([[3, 3], [10, 3], [3, -1], [9, 0]], dtype=torch.int32, device="cuda")
    y, _ = lbw_amd.qk_head_norm_rope(q, k, *w, rope, pos)
    nan = torch.isnan(y)
    assert not nan[0].any() and not nan[3].any()
    assert nan[1, :, :40].all() and not nan[1, :, 40:].any()
    assert nan[2, :, 40:64].all() and not nan[2, :, :40].any() and not nan[2, :, 64:].any()


@pytest.mark.parametrize("T,hq,hk,d", [(1, 40, 8, 128), (64, 12, 4, 128), (7, 3, 3, 64), (5, 6, 2, 256)])
def test_write_form_into_cache_rows(T, hq, hk, d):
    import lbw_amd
    q, k, v, w = _data(T, hq, hk, d, 9)
    ang, rope = _rope((d // 4,), 40, False)
    cap = 33
    buf = torch.full((2, T, cap + 1, hk, d), 7.0, dtype=BF, device="cuda")
    kc, vc = buf[0][:, :cap], buf[1][:, :cap]      # (strided: the caches end before their buffers)
    rows = torch.arange(T, dtype=torch.int32, device="cuda") * 5 % cap
    if T > 3:
        rows[1], rows[2] = -1, cap               # not written
    pos = torch.arange(T, dtype=torch.int32, device="cuda") % 40
    qo = torch.empty(T, hq, d, dtype=BF, device="cuda")
    lbw_amd.qk_head_norm_rope_(q, k, *w, rope, pos, q_out=qo, k_out=kc, v=v, v_out=vc, rows=rows)
    q2, k2 = lbw_amd.qk_head_norm_rope(q, k, *w, rope, pos)
    assert torch.equal(qo, q2)
    want = torch.full_like(buf, 7.0)
    for t, r in enumerate(rows.tolist()):
        if 0 <= r < cap:
            want[0, t, r], want[1, t, r] = k2[t], v[t]
    assert torch.equal(buf, want)


def test_write_form_in_place_and_strided():
    import lbw_amd
    q, k, v, w = _data(50, 10, 5, 128, 10)
    _, rope = _rope((64,), 50, False)
    pos = torch.arange(50, dtype=torch.int32, device="cuda")
    want = lbw_amd.qk_head_norm_rope(q, k, *w, rope, pos)
    v0 = v.clone()
    lbw_amd.qk_head_norm_rope_(q, k, *w, rope, pos, q_out=q, k_out=k)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(v, v0)


def test_outputs_that_share_memory_with_other_tensors_are_refused():
    import lbw_amd
    T, h, d = 6, 2, 64
    _, rope = _rope((32,), 8, True)
    pos = torch.zeros(T, dtype=torch.int32, device="cuda")
    buf = torch.zeros(T, 3 * h, d, dtype=BF, device="cuda")
    q, k, v = buf.split([h, h, h], 1)
    go = lambda q_, k_, qo, ko, **kw: lbw_amd.qk_head_norm_rope_(  # noqa: E731
        q_, k_, None, None, rope, pos, q_out=qo, k_out=ko, **kw)
    new = lambda: torch.zeros(T, h, d, dtype=BF, device="cuda")  # noqa: E731
    go(q, k, q, k)                              # in place, column blocks of one buffer
    go(q, k, new(), v)                          # k's result into v's columns (v is not read)
    for bad in (lambda: go(q, q, q, new()),     # q's result over k, which other waves still read
                lambda: go(q, k, k, new()), lambda: go(q, k, new(), q), lambda: go(q, k, v, v),
                lambda: go(q, k, buf[:, 1:3], new()), lambda: go(q, k, new(), new(), v=v, v_out=q),
                lambda: go(q, k, q, k, v=v, v_out=k)):
        with pytest.raises(RuntimeError, match="overlaps"):
            bad()
    cache = torch.zeros(T, 9, h, d, dtype=BF, device="cuda")
    rows = torch.zeros(T, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="overlaps"):
        go(q, k, new(), cache, v=v, v_out=cache, rows=rows)
    with pytest.raises(RuntimeError, match="one place"):
        go(q, k, new(), cache[:1].expand(T, 9, h, d), rows=rows)


def test_more_than_2_31_elements():
    import lbw_amd
    T, hq, d = 270000, 63, 128
    q = torch.zeros(T, hq, d, dtype=BF, device="cuda")
    assert q.numel() > 1 << 31
    q[-3:] = torch.randn(3, hq, d, device="cuda").to(BF)
    k = torch.zeros(T, 1, d, dtype=BF, device="cuda")
    ang, rope = _rope((64,), 50, True)
    pos = torch.full((T,), 7, dtype=torch.int32, device="cuda")
    q2, _ = lbw_amd.qk_head_norm_rope(q, k, None, None, rope, pos)
    want = R.head_norm(q[-3:].double(), None, R.token_angles(ang, (64,), pos[-3:]), True, 1e-6, 1.0)
    R.assert_within("q'", q2[-3:], want, R.head_norm_allow(want))
    assert torch.all(q2[:-3] == 0)


def test_refusals_on_the_device():
    import lbw_amd
    q, k, v, w = _data(8, 4, 2, 128, 11)
    _, rope = _rope((64,), 8, True)
    pos = torch.zeros(8, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="overlaps"):
        buf = torch.zeros(9, 4, 128, dtype=BF, device="cuda")
        lbw_amd.qk_head_norm_rope_(buf[:8], k, *w, rope, pos, q_out=buf[1:], k_out=k.clone())
    with pytest.raises(RuntimeError, match="one place"):
        lbw_amd.qk_head_norm_rope_(q, k, *w, rope, pos, q_out=q[:1].expand(8, 4, 128), k_out=k.clone())
    with pytest.raises(RuntimeError, match="multiples of 8"):
        lbw_amd.qk_head_norm_rope(torch.zeros(8, 4 * 129, dtype=BF, device="cuda").unflatten(1, (4, 129))[..., :128],
                                  k, *w, rope, pos)
    with pytest.raises(ValueError, match="another device"):
        lbw_amd.qk_head_norm_rope(q, k, *w, lbw_amd.axis_rope(torch.zeros(8, 64)), pos)
    with pytest.raises(RuntimeError, match="pos"):
        lbw_amd.qk_head_norm_rope(q, k, *w, rope, pos.cpu())
    x = q.detach().requires_grad_()
    y = lbw_amd.qk_head_norm_rope(x, k, *w, rope, pos)[0]
    g, = torch.autograd.grad(y.float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.float().sum().backward()  # no second derivatives


def test_no_rotation_and_a_column_of_positions():
    import lbw_amd
    q, k, _, w = _data(9, 4, 2, 128, 12)
    none = lbw_amd.axis_rope(torch.empty(5, 0), device="cuda")
    pos3 = torch.arange(27, dtype=torch.int32, device="cuda").view(9, 3)
    got = lbw_amd.qk_head_norm_rope(q, k, *w, none, pos3[:, 1])
    for y, x, wt in zip(got, (q, k), w):
        want = R.head_norm(x.double(), wt.double(), torch.zeros(9, 0, dtype=torch.float64, device="cuda"), True, 1e-6, 1.0)
        R.assert_within("y", y, want, R.head_norm_allow(want))
    rope = lbw_amd.axis_rope(torch.randn(30, 64, generator=torch.Generator().manual_seed(1)), device="cuda")
    a = lbw_amd.qk_head_norm_rope(q, k, *w, rope, pos3[:, 1])
    b = lbw_amd.qk_head_norm_rope(q, k, *w, rope, pos3[:, 1:2].contiguous())
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def _gradient_allowance(X, W, a, inter, eps, s, dy):
    """As in test_forward_and_gradient: 2^10 E of the sizes of the two terms, and the one rounding."""
    r = torch.rsqrt(X.square().mean(-1, keepdim=True) + eps)
    gw = R.rotate(dy.double(), a.cos(), -a.sin(), inter).abs() * s * W.abs()
    size = r * (gw.amax(-1, keepdim=True) + (X.abs() * r).amax(-1, keepdim=True) *
                (gw * X.abs() * r).mean(-1, keepdim=True))
    terms = (R.rotate(dy.double(), a.cos(), -a.sin(), inter) * s * X * r).abs().sum((0, 1))
    return 2 ** 10 * R.E * size, terms


@pytest.mark.parametrize("hq,hk,d", [(4, 1, 128), (6, 3, 32), (5, 5, 256), (12, 4, 64)])
def test_gradient_with_eps_0(hq, hk, d):
    """Lanes past the last head hold zeros, whose rsqrt(0) must not reach the weights' gradient."""
    import lbw_amd
    T = 21
    q, k, _, w = _data(T, hq, hk, d, 15)
    ang, rope = _rope((d // 2,), 50, True)
    pos = _pos(T, (d // 2,), 50)
    leaves = [x.detach().requires_grad_() for x in (q, k, *w)]
    y = lbw_amd.qk_head_norm_rope(*leaves, rope, pos, 0.0)
    dy = [torch.randn(x.shape, generator=torch.Generator().manual_seed(n)).to(BF).cuda() for n, x in enumerate(y)]
    grads = torch.autograd.grad(y, leaves, dy)
    a = R.token_angles(ang, (d // 2,), pos)
    for n in range(2):
        X, W = leaves[n].detach().double().requires_grad_(), leaves[2 + n].detach().double().requires_grad_()
        Y = R.head_norm(X, W, a, True, 0.0, 1.0)
        R.assert_within("y", y[n], Y.detach(), R.head_norm_allow(Y.detach()))
        G = torch.autograd.grad(Y, (X, W), dy[n].double())
        allow, terms = _gradient_allowance(X.detach(), W.detach(), a, True, 0.0, 1.0, dy[n])
        R.assert_within("dx", grads[n], G[0], R.H * G[0].abs() + allow)
        R.assert_within("dw", grads[2 + n], G[1], R.H * G[1].abs() + (T + 200) * R.E * terms)


def _cache_layouts(T, cap, hk, d):
    new = lambda *s: torch.full(s, 7.0, dtype=BF, device="cuda")  # noqa: E731
    a, b, c, e = new(T, cap, 2, hk, d), new(T, cap, hk, 2, d), new(T, 2, hk, cap, d), new(hk, cap, 2, T, d)
    return {"K and V of a token": (a, a[:, :, 0], a[:, :, 1]), "K and V of a head": (b, b[..., 0, :], b[..., 1, :]),
            "heads first": (c, c[:, 0].transpose(1, 2), c[:, 1].transpose(1, 2)),
            "sequences last": (e, e[:, :, 0].permute(2, 1, 0, 3), e[:, :, 1].permute(2, 1, 0, 3))}


@pytest.mark.parametrize("layout", ["K and V of a token", "K and V of a head", "heads first", "sequences last"])
def test_write_form_into_interleaved_caches(layout):
    import lbw_amd
    T, hq, hk, d, cap = 5, 4, 2, 64, 9
    q, k, v, w = _data(T, hq, hk, d, 16)
    _, rope = _rope((32,), 40, False)
    pos = torch.arange(T, dtype=torch.int32, device="cuda")
    rows = torch.tensor([0, 8, 3, -1, 5], dtype=torch.int32, device="cuda")
    buf, kc, vc = _cache_layouts(T, cap, hk, d)[layout]
    qo = torch.empty(T, hq, d, dtype=BF, device="cuda")
    lbw_amd.qk_head_norm_rope_(q, k, *w, rope, pos, q_out=qo, k_out=kc, v=v, v_out=vc, rows=rows)
    q2, k2 = lbw_amd.qk_head_norm_rope(q, k, *w, rope, pos)
    assert torch.equal(qo, q2)
    want, wk, wv = _cache_layouts(T, cap, hk, d)[layout]
    for t, r in enumerate(rows.tolist()):
        if r >= 0:
            wk[t, r], wv[t, r] = k2[t], v[t]
    assert torch.equal(buf, want)


def test_write_form_in_place_in_an_interleaved_projection():
    import lbw_amd
    T, h, d = 11, 3, 128
    _, rope = _rope((64,), 40, True)
    pos = torch.arange(T, dtype=torch.int32, device="cuda")
    g = torch.Generator().manual_seed(17)
    buf = torch.randn(T, h, 3, d, generator=g).to(BF).cuda()
    want = buf.clone()
    want[:, :, 0], want[:, :, 1] = lbw_amd.qk_head_norm_rope(buf[:, :, 0], buf[:, :, 1], None, None, rope, pos)
    lbw_amd.qk_head_norm_rope_(buf[:, :, 0], buf[:, :, 1], None, None, rope, pos, q_out=buf[:, :, 0], k_out=buf[:, :, 1])
    assert torch.equal(buf, want)


def test_outputs_are_refused_exactly_when_they_share_an_element():
    import random
    import lbw_amd
    rng = random.Random(18)
    _, rope = _rope((16,), 8, True)
    store = torch.zeros(8192, dtype=BF, device="cuda")
    none = torch.zeros(8, 4, 32, dtype=BF, device="cuda")

    def layout(own):
        while True:
            T, h = rng.randint(1, 6), rng.randint(1, 3)
            s = [8 * rng.randint(0 if not own else 4, rng.choice([10, 60])) for _ in range(2)]
            at = 8 * rng.randint(0, 100)
            place = [at + t * s[0] + i * s[1] + x for t in range(T) for i in range(h) for x in range(32)]
            if not own or len(set(place)) == len(place):
                return (T, h, 32), (*s, 1), at, set(place)
    seen = [0, 0]
    for _ in range(300):
        size, stride, at, mine = layout(True)
        T, h, _ = size
        _, kstride, kat, _ = layout(False)
        place = {kat + t * kstride[0] + x for t in range(T) for x in range(32)}
        q_out, k = store.as_strided(size, stride, at), store.as_strided((T, 1, 32), kstride, kat)
        pos = torch.zeros(T, dtype=torch.int32, device="cuda")
        call = lambda: lbw_amd.qk_head_norm_rope_(none[:T, :h], k, None, None, rope, pos, q_out=q_out,  # noqa: E731
                                                  k_out=torch.empty(T, 1, 32, dtype=BF, device="cuda"))
        shared = bool(mine & place)
        seen[shared] += 1
        if shared:
            with pytest.raises(RuntimeError, match="overlaps"):
                call()
        else:
            call()
    assert min(seen) > 20


def test_more_tokens_than_2_21():
    import lbw_amd
    T, d = (1 << 21) + 77, 32
    g = torch.Generator(device="cuda").manual_seed(19)
    q, k, dq, dk = (torch.randn(T, 1, d, generator=g, device="cuda").to(BF) for _ in range(4))
    w = [(1 + 0.1 * torch.randn(d, generator=g, device="cuda")).to(BF) for _ in range(2)]
    ang, rope = _rope((16,), 50, True)
    pos = (torch.arange(T, device="cuda") % 50).int()
    leaves = [x.requires_grad_() for x in (q, k, *w)]
    y = lbw_amd.qk_head_norm_rope(*leaves, rope, pos, 1e-6)
    grads = torch.autograd.grad(y, leaves, (dq, dk))
    a = R.token_angles(ang, (16,), pos)
    # each lane adds the tokens of its wave in turn: those of a quarter of a workgroup, at least one a CU for q and k
    deep = T // (4 * torch.cuda.get_device_properties(0).multi_processor_count) + 200
    for n, dy in enumerate((dq, dk)):
        X, W = leaves[n].detach().double().requires_grad_(), leaves[2 + n].detach().double().requires_grad_()
        Y = R.head_norm(X, W, a, True, 1e-6, 1.0)
        R.assert_within("y", y[n], Y.detach(), R.head_norm_allow(Y.detach()))
        G = torch.autograd.grad(Y, (X, W), dy.double())
        allow, terms = _gradient_allowance(X.detach(), W.detach(), a, True, 1e-6, 1.0, dy)
        R.assert_within("dx", grads[n], G[0], R.H * G[0].abs() + allow)
        R.assert_within("dw", grads[2 + n], G[1], R.H * G[1].abs() + deep * R.E * terms)


def test_gradients_with_far_heads_are_copied():
    """Heads 2^26 elements apart, as a head-major gradient of 524288 tokens has them."""
    import lbw_amd
    T, d, far = 6, 128, 1 << 26
    q, k, _, w = _data(T, 2, 2, d, 20)
    _, rope = _rope((64,), 8, True)
    pos = torch.arange(T, dtype=torch.int32, device="cuda")
    leaves = [x.detach().requires_grad_() for x in (q, k, *w)]
    y = lbw_amd.qk_head_norm_rope(*leaves, rope, pos)
    dy = torch.randn(T, 2, d, generator=torch.Generator().manual_seed(21)).to(BF).cuda()
    g = torch.empty(far + T * d, dtype=BF, device="cuda").as_strided((T, 2, d), (d, far, 1))
    g.copy_(dy)
    want = torch.autograd.grad(y, leaves, (dy, dy), retain_graph=True)
    got = torch.autograd.grad(y, leaves, (g, g))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
