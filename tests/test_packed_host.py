"""CPU checks of the operators on packed sequences: the plan covers every row and pair once, the
oracle's gradients against differences, refusals of arguments, struct layouts."""
import ctypes
import random

import pytest
import torch

import packed_ref as R
from test_capi import HEADER, _header_struct, _header_struct_fields, _layout  # noqa: F401


def lbw():
    import lbw_amd
    return lbw_amd


LENS = [([300, 1, 0, 129], [300, 5, 3, 20], True), ([128, 256, 127], [128, 256, 127], True),
        ([5], [5], False), ([0, 0], [0, 7], True), ([7, 3], [0, 0], False), ([], [], True),
        ([64, 200], [1000, 30], True), ([64, 200], [1000, 30], False)]


@pytest.mark.parametrize("ql,kl,causal", LENS)
def test_plan_covers_every_row_once_and_bounds_what_is_seen(ql, kl, causal):
    p = lbw().packed_plan(ql, kl, causal=causal, device="cpu")
    assert (p.q_tokens, p.k_tokens) == (sum(ql), sum(kl))
    q_at = [sum(ql[:s]) for s in range(len(ql))]
    k_at = [sum(kl[:s]) for s in range(len(kl))]
    rows = []
    for row0, n, pos, other0, other, bound, shift, _ in p.q_items.tolist():
        assert 0 < n <= 128
        s = max(x for x in range(len(ql)) if q_at[x] == row0 - pos and ql[x] > 0 and pos < ql[x])
        assert (other0, other) == (k_at[s], kl[s]) and pos + n <= ql[s]
        for i in range(pos, pos + n):
            seen = [j for j in range(kl[s]) if not causal or j <= i + kl[s] - ql[s]]
            assert seen == [j for j in range(kl[s]) if j <= i + shift]
            assert not seen or seen[-1] < bound
        assert bound == (seen[-1] + 1 if seen else 0)
        rows += range(row0, row0 + n)
    assert sorted(rows) == list(range(sum(ql)))
    keys = []
    for row0, n, pos, other0, other, bound, shift, _ in p.k_items.tolist():
        assert 0 < n <= 128
        s = max(x for x in range(len(kl)) if k_at[x] == row0 - pos and kl[x] > 0 and pos < kl[x])
        assert (other0, other) == (q_at[s], ql[s]) and pos + n <= kl[s]
        sees = [i for i in range(ql[s]) if pos <= i + shift]
        assert bound == (sees[0] if sees else ql[s])
        keys += range(row0, row0 + n)
    assert sorted(keys) == list(range(sum(kl)))
    cost = [x[5] for x in p.q_items.tolist()]
    assert cost == sorted(cost, reverse=True)
    qt = [-(-x // 64) for x in cost]
    kt = [-(-x[4] // 64) - x[5] // 64 if x[5] < x[4] else 0 for x in p.k_items.tolist()]
    assert p.info == (sum(ql), sum(kl), sum(qt), max(qt, default=0), sum(kt), max(kt, default=0))


def test_plan_refusals():
    with pytest.raises(ValueError, match="negative"):
        lbw().packed_plan([3, -1], device="cpu")
    with pytest.raises(ValueError, match="lengths"):
        lbw().packed_plan([3], [3, 4], device="cpu")
    with pytest.raises(ValueError, match="2\\^31"):
        lbw().packed_plan([2 ** 30, 2 ** 30], device="cpu")
    with pytest.raises(ValueError, match="2\\^31"):
        lbw().packed_plan([1], [2 ** 31 - 255], device="cpu")
    from lbw_amd import _lib
    lib = _lib.load()
    n = ctypes.byref(_lib.PackedPlanInfo())
    lens = (ctypes.c_int32 * 1)(300)
    items = (ctypes.c_int32 * 8)()
    assert lib.lbw_attention_packed_plan(1, lens, lens, 1, items, 1, items, 1, n) == 1
    assert b"room for 3" in lib.lbw_last_error()
    assert lib.lbw_attention_packed_plan(1, None, lens, 1, None, 0, None, 0, n) == 1
    assert lib.lbw_attention_packed_plan(1, lens, lens, 1, None, 0, None, 0, None) == 1
    long = (ctypes.c_int32 * 1)(2 ** 31 - 255)
    assert lib.lbw_attention_packed_plan(1, lens, long, 1, None, 0, None, 0, n) != 0
    assert b"2^31 - 256" in lib.lbw_last_error()


@pytest.mark.parametrize("cname,pyname", [("lbw_head_norm_rope_params", "HeadNormRopeParams"),
                                          ("lbw_head_norm_rope_grads", "HeadNormRopeGrads"),
                                          ("lbw_packed_params", "PackedParams"),
                                          ("lbw_packed_grads", "PackedGrads"),
                                          ("lbw_packed_plan_info", "PackedPlanInfo"),
                                          ("lbw_decode_params", "DecodeParams")])
def test_struct_layouts_match_the_header(cname, pyname):
    from lbw_amd import _lib
    py = getattr(_lib, pyname)
    assert [f[0] for f in py._fields_] == _header_struct_fields(cname)
    text = open(HEADER).read()
    assert "#define LBW_MAX_AXES 4" in text
    assert _layout(py) == _layout(_header_struct(cname, {}))


# ---- the oracle

def _differences(f, xs, grads, seed, steps=3):
    """Directional differences of scalar f against the gradients, in 64 bits."""
    gen = torch.Generator().manual_seed(seed)
    for _ in range(steps):
        ds = [torch.randn(x.shape, generator=gen, dtype=torch.float64) for x in xs]
        h = 1e-5
        num = (f([x + h * d for x, d in zip(xs, ds)]) - f([x - h * d for x, d in zip(xs, ds)])) / (2 * h)
        ana = sum((g * d).sum() for g, d in zip(grads, ds))
        # the third derivative's h^2 and the differences' rounding 1e-16 / h, both near 1e-10 of sums of
        # order 1 to 100
        assert abs(num - ana) <= 1e-6 * (1 + abs(ana)), (num, ana)


@pytest.mark.parametrize("ql,kl,causal", [([5, 0, 9], [5, 3, 4], True), ([4, 6], [9, 6], True),
                                          ([3, 8], [8, 2], False)])
def test_oracle_attention_gradient_against_differences(ql, kl, causal):
    gen = torch.Generator().manual_seed(1)
    rnd = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)  # noqa: E731
    q, k, v, do = rnd(sum(ql), 4, 16), rnd(sum(kl), 2, 16), rnd(sum(kl), 2, 16), rnd(sum(ql), 4, 16)
    r = R.attention(q, k, v, ql, kl, causal, 0.3, do)
    f = lambda xs: (R.attention(*xs, ql, kl, causal, 0.3)["out"] * do).sum()  # noqa: E731
    _differences(f, [q, k, v], [r["dq"], r["dk"], r["dv"]], 2)


@pytest.mark.parametrize("inter", [True, False])
def test_oracle_norm_is_a_rotation_of_the_normed_head(inter):
    gen = torch.Generator().manual_seed(3)
    x = torch.randn(7, 3, 32, generator=gen, dtype=torch.float64)
    ang = torch.rand(7, 8, generator=gen, dtype=torch.float64) * 6
    y = R.head_norm(x, None, ang, inter, 0.0, 1.0)
    assert torch.allclose(y.square().mean(-1), torch.ones(7, 3, dtype=torch.float64))
    back = R.rotate(y, ang.cos(), -ang.sin(), inter)
    assert torch.allclose(back, x / x.square().mean(-1, keepdim=True).sqrt())


# ---- refusals (no kernel runs: the wrappers' ValueError, or the C entry's status)

def _rope(pairs=64, **kw):
    return lbw().axis_rope(torch.zeros(10, pairs), **kw)


def test_axis_rope_refusals():
    with pytest.raises(ValueError, match="add up"):
        _rope(axes=(10, 20))
    with pytest.raises(ValueError, match="1 to 4"):
        _rope(axes=(60, 1, 1, 1, 1))
    with pytest.raises(ValueError, match="multiple of 8"):
        _rope(12, interleaved=False)
    with pytest.raises(ValueError, match="floating"):
        lbw().axis_rope(torch.zeros(10, dtype=torch.int64))


BF = torch.bfloat16


def _qk(T=5, hq=4, hk=2, d=128):
    return torch.zeros(T, hq, d, dtype=BF), torch.zeros(T, hk, d, dtype=BF)


@pytest.mark.parametrize("change,match", [
    (dict(q=torch.zeros(5, 4, 128)), "bf16"),
    (dict(q=torch.zeros(5, 128, 4, dtype=BF).transpose(1, 2)), "contiguous head dim"),
    (dict(k=torch.zeros(4, 2, 128, dtype=BF)), "does not fit"),
    (dict(k=torch.zeros(5, 3, 128, dtype=BF)), "divides"),
    (dict(pos=torch.zeros(5, dtype=torch.int64)), "int32"),
    (dict(pos=torch.zeros(5, 2, dtype=torch.int32)), "pos must"),
    (dict(wk=None), "both or neither"),
    (dict(q=torch.zeros(5, 4, 64, dtype=BF), k=torch.zeros(5, 2, 64, dtype=BF)), "pairs do not fit"),
])
def test_head_norm_refusals(change, match):
    q, k = _qk()
    a = dict(q=q, k=k, wq=torch.ones(128, dtype=BF), wk=torch.ones(128, dtype=BF), rope=_rope(),
             pos=torch.zeros(5, dtype=torch.int32))
    a.update(change)
    with pytest.raises(ValueError, match=match):
        lbw().qk_head_norm_rope(a["q"], a["k"], a["wq"], a["wk"], a["rope"], a["pos"])


def test_head_norm_write_form_refusals():
    q, k = _qk()
    call = lambda **kw: lbw().qk_head_norm_rope_(  # noqa: E731
        q, k, None, None, _rope(), torch.zeros(5, dtype=torch.int32),
        **{"q_out": q.clone(), "k_out": k.clone(), **kw})
    with pytest.raises(ValueError, match="q_out"):
        call(q_out=k)
    with pytest.raises(ValueError, match="v and v_out"):
        call(v=k)
    with pytest.raises(ValueError, match="cache"):
        call(rows=torch.zeros(5, dtype=torch.int32))
    with pytest.raises(ValueError, match="cache"):
        call(rows=torch.zeros(5, dtype=torch.int32), k_out=torch.zeros(4, 8, 2, 128, dtype=BF))
    with pytest.raises(ValueError, match="rows must"):
        call(rows=torch.zeros(5, dtype=torch.int64), k_out=torch.zeros(5, 8, 2, 128, dtype=BF))


def test_packed_refusals():
    plan = lbw().packed_plan([5, 3], device="cpu")
    z = lambda *s: torch.zeros(*s, dtype=BF)  # noqa: E731
    call = lambda q, k, v, **kw: lbw().attention_packed(q, k, v, plan, **kw)  # noqa: E731
    with pytest.raises(ValueError, match="the plan 8"):
        call(z(9, 4, 128), z(8, 2, 128), z(8, 2, 128))
    with pytest.raises(ValueError, match="bf16"):
        call(z(8, 4, 64), z(8, 2, 64), z(8, 2, 64))
    with pytest.raises(ValueError, match="bf16"):
        call(z(8, 4, 128).half(), z(8, 2, 128), z(8, 2, 128))
    with pytest.raises(ValueError, match="divides"):
        call(z(8, 4, 128), z(8, 3, 128), z(8, 3, 128))
    for bad in (-1.0, 0.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="softmax_scale"):
            call(z(8, 4, 128), z(8, 2, 128), z(8, 2, 128), softmax_scale=bad)
    with pytest.raises(ValueError, match="lse"):
        lbw().attention_packed_backward(z(8, 4, 128), z(8, 4, 128), z(8, 2, 128), z(8, 2, 128),
                                        z(8, 4, 128), torch.zeros(8, 4), plan)


def test_decode_refusals():
    z = lambda *s: torch.zeros(*s, dtype=BF)  # noqa: E731
    lens = torch.zeros(2, dtype=torch.int32)
    call = lbw().attention_decode
    with pytest.raises(ValueError, match="q must"):
        call(z(2, 4, 64), z(2, 8, 2, 64), z(2, 8, 2, 64), lens)
    with pytest.raises(ValueError, match="k_cache"):
        call(z(2, 4, 128), z(3, 8, 2, 128), z(3, 8, 2, 128), lens)
    with pytest.raises(ValueError, match="v_cache"):
        call(z(2, 4, 128), z(2, 8, 2, 128), z(2, 9, 2, 128), lens)
    with pytest.raises(ValueError, match="divide"):
        call(z(2, 4, 128), z(2, 8, 3, 128), z(2, 8, 3, 128), lens)
    with pytest.raises(ValueError, match="lens"):
        call(z(2, 4, 128), z(2, 8, 2, 128), z(2, 8, 2, 128), lens.long())
    with pytest.raises(ValueError, match="num_splits"):
        call(z(2, 4, 128), z(2, 8, 2, 128), z(2, 8, 2, 128), lens, num_splits=129)
    with pytest.raises(ValueError, match="out must"):
        call(z(2, 4, 128), z(2, 8, 2, 128), z(2, 8, 2, 128), lens, out=z(2, 5, 128))


def test_c_entries_refuse_before_any_gpu_call():
    from lbw_amd import _lib
    lib = _lib.load()
    d = _lib.DecodeParams(batch=1, q_heads=4, k_heads=2, head_dim=64, capacity=8)
    assert lib.lbw_attention_decode(ctypes.byref(d), None, 0, None) == 2
    p = _lib.PackedParams(q_heads=4, k_heads=3, head_dim=128, q_tokens=1, k_tokens=1)
    assert lib.lbw_attention_packed_fwd(ctypes.byref(p), None, 0, None) == 1
    p = _lib.PackedParams(q_heads=4, k_heads=2, head_dim=128, q_tokens=1, k_tokens=1, q=8)
    assert lib.lbw_attention_packed_fwd(ctypes.byref(p), None, 0, None) == 1
    assert b"16-byte" in lib.lbw_last_error()
    p = _lib.PackedParams(q_heads=4, k_heads=2, head_dim=128, q_tokens=1, k_tokens=1, q=16, k=16, v=16,
                          out=16, q_stride_l=12)
    assert lib.lbw_attention_packed_fwd(ctypes.byref(p), None, 0, None) == 1
    assert b"multiples of 8" in lib.lbw_last_error()
    p.q_stride_l = 1 << 26
    assert lib.lbw_attention_packed_fwd(ctypes.byref(p), None, 0, None) == 2
    p.q_stride_l = 512
    p.softmax_scale = -1.0
    assert lib.lbw_attention_packed_fwd(ctypes.byref(p), None, 0, None) == 1
    n = _lib.HeadNormRopeParams(tokens=1, q_heads=4, k_heads=2, head_dim=48)
    assert lib.lbw_head_norm_rope(ctypes.byref(n), None) == 2
    n = _lib.HeadNormRopeParams(tokens=1, q_heads=4, k_heads=2, head_dim=128, n_axes=2, rope_pairs=64)
    n.axis_pairs[0] = 60
    assert lib.lbw_head_norm_rope(ctypes.byref(n), None) == 1
    assert b"add up" in lib.lbw_last_error()
    assert lib.lbw_attention_packed_fwd(None, None, 0, None) == 1
    assert lib.lbw_head_norm_rope(None, None) == 1


def test_token_limits_of_the_head_norm():
    """Forward: the grid of the tokens, four waves a workgroup, below 2^32 threads; gradient: none."""
    from lbw_amd import _lib
    lib = _lib.load()
    most = 4 * ((1 << 24) - 1)

    def params(tokens):
        p = _lib.HeadNormRopeParams(tokens=tokens, q_heads=1, k_heads=1, head_dim=32, n_axes=1, pos=4)
        for x in ("q", "k"):
            setattr(p, x, 16)
            setattr(p, x + "_stride_l", 32)
        return ctypes.byref(p)
    # (the next check after the tokens': an output's alignment)
    for tokens in (1 << 21, (1 << 21) + 1, most):
        assert lib.lbw_head_norm_rope(params(tokens), None) == 1
        assert b"q_out must be" in lib.lbw_last_error()
    assert lib.lbw_head_norm_rope(params(most + 1), None) == 2
    assert str(most).encode() in lib.lbw_last_error()
    for tokens in (1 << 21, most + 1, (1 << 31) - 1):
        assert lib.lbw_head_norm_rope_bwd(params(tokens), ctypes.byref(_lib.HeadNormRopeGrads()), None, 0, None) == 1
        assert b"dq_out must be" in lib.lbw_last_error()


# ---- autograd's view of the operators: tensors without memory take the same entries

def _meta(*s):
    return torch.zeros(*s, dtype=BF, device="meta")


def _meta_calls():
    """name -> (call, its differentiable inputs)."""
    plan = lbw().packed_plan([3, 2], device="cpu")
    qi, ki = plan.q_items.to("meta"), plan.k_items.to("meta")
    rope = lbw().axis_rope(torch.zeros(8, 64), device="meta")
    pos = torch.zeros(5, dtype=torch.int32, device="meta")
    w = lambda: torch.ones(128, dtype=BF, device="meta")  # noqa: E731
    qkv = lambda: [_meta(5, 4, 128), _meta(5, 2, 128), _meta(5, 2, 128)]  # noqa: E731
    norm = lambda q, k, wq, wk: lbw().qk_head_norm_rope(q, k, wq, wk, rope, pos)[0]  # noqa: E731
    packed = lambda q, k, v: torch.ops.lbw.attention_packed(q, k, v, qi, ki, plan.info)[0]  # noqa: E731
    return {"norm": (norm, qkv()[:2] + [w(), w()]), "packed": (packed, qkv())}


@pytest.mark.parametrize("name,at", [("norm", i) for i in range(4)] + [("packed", i) for i in range(3)])
def test_forward_mode_derivatives_are_refused(name, at):
    import torch.autograd.forward_ad as fw
    call, xs = _meta_calls()[name]
    with fw.dual_level():
        ds = [fw.make_dual(x, torch.ones_like(x)) if i == at else x for i, x in enumerate(xs)]
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(*ds)
        assert call(*xs).shape == xs[0].shape  # (no tangent: as ever)
    f = lambda x: call(*xs[:at], x, *xs[at + 1:])  # noqa: E731
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(f, (xs[at],), (torch.ones_like(xs[at]),))


def _write_calls():
    """name -> (call, inputs by name, written tensors by name)."""
    rope = lbw().axis_rope(torch.zeros(8, 64), device="meta")
    pos = torch.zeros(5, dtype=torch.int32, device="meta")
    w = lambda: torch.ones(128, dtype=BF, device="meta")  # noqa: E731

    def append(q, k, wq, wk, v, q_out, k_out, v_out):
        lbw().qk_head_norm_rope_(q, k, wq, wk, rope, pos, q_out=q_out, k_out=k_out, v=v, v_out=v_out, rows=pos)

    def decode(q, k_cache, v_cache, out):
        lbw().attention_decode(q, k_cache, v_cache, pos, out=out)
    return {"append": (append, dict(q=_meta(5, 4, 128), k=_meta(5, 2, 128), wq=w(), wk=w(), v=_meta(5, 2, 128)),
                       dict(q_out=_meta(5, 4, 128), k_out=_meta(5, 9, 2, 128), v_out=_meta(5, 9, 2, 128))),
            "decode": (decode, dict(q=_meta(5, 4, 128), k_cache=_meta(5, 9, 2, 128), v_cache=_meta(5, 9, 2, 128)),
                       dict(out=_meta(5, 4, 128)))}


@pytest.mark.parametrize("name,arg", [("append", a) for a in ("q", "k", "wq", "wk", "v", "q_out", "k_out", "v_out")] +
                         [("decode", a) for a in ("q", "k_cache", "v_cache", "out")])
def test_write_forms_refuse_tensors_that_require_a_gradient(name, arg):
    import torch.autograd.forward_ad as fw
    call, ins, outs = _write_calls()[name]
    args = {**ins, **outs}
    args[arg].requires_grad_()
    with pytest.raises(NotImplementedError, match="not differentiable"):
        call(**args)
    with torch.no_grad():
        call(**args)
    args[arg] = args[arg] * 1                     # (of a graph, and not a leaf)
    with pytest.raises(NotImplementedError, match="not differentiable"):
        call(**args)
    args[arg] = args[arg].detach()
    call(**args)
    with fw.dual_level():
        args[arg] = fw.make_dual(args[arg], torch.ones_like(args[arg]))
        with pytest.raises(NotImplementedError, match="not differentiable"):
            call(**args)


def test_in_place_in_a_graph_is_refused():
    """q of a projection that is trained, overwritten: its gradient would miss the norm and the rotation."""
    call, ins, outs = _write_calls()["append"]
    q = _meta(5, 4, 128).requires_grad_() * 2
    with pytest.raises(NotImplementedError, match="not differentiable"):
        call(**{**ins, **outs, "q": q, "q_out": q})


@pytest.mark.parametrize("name", ["append", "decode"])
@pytest.mark.parametrize("mode", [torch.enable_grad, torch.no_grad, torch.inference_mode])
def test_writes_are_counted(name, mode):
    call, ins, outs = _write_calls()[name]
    before = {n: t._version for n, t in {**ins, **outs}.items()}
    with mode():
        call(**ins, **outs)
    assert all(t._version == before[n] for n, t in ins.items())
    assert all(t._version == before[n] + 1 for n, t in outs.items())
    with torch.inference_mode():
        outs = {n: torch.zeros_like(t) for n, t in outs.items()}
        call(**ins, **outs)                       # inference tensors, which have no count
    with torch.no_grad():
        call(**ins, **outs)


@pytest.mark.parametrize("name,out", [("append", "q_out"), ("append", "k_out"), ("append", "v_out"), ("decode", "out")])
def test_backward_over_an_overwritten_tensor_raises(name, out):
    call, ins, outs = _write_calls()[name]
    h = torch.zeros_like(outs[out]).requires_grad_() * 1
    y = (h * h).sum()
    outs[out] = h.detach()
    call(**ins, **outs)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


@pytest.mark.parametrize("scale,status", [(1e-31, 2), (2e6, 2), (1e8, 2), (3e38, 2), (float("inf"), 1), (-1.0, 1)])
def test_scales_that_leave_fp32_are_refused(scale, status):
    """At 1e8 rows of ordinary scores gave 0 or NaN, from 3e8 on rows that see no key gave NaN."""
    from lbw_amd import _lib
    lib = _lib.load()
    p = _lib.PackedParams(q_heads=4, k_heads=2, head_dim=128, softmax_scale=scale)
    assert lib.lbw_attention_packed_fwd(ctypes.byref(p), None, 0, None) == status
    assert b"softmax_scale" in lib.lbw_last_error()
    assert lib.lbw_attention_packed_bwd(ctypes.byref(p), ctypes.byref(_lib.PackedGrads()), None, 0, None) == status
    d = _lib.DecodeParams(batch=0, q_heads=4, k_heads=2, head_dim=128, softmax_scale=scale)
    assert lib.lbw_attention_decode(ctypes.byref(d), None, 0, None) == status
    for ok in (1e-30, 0.0, 1e6):
        p.softmax_scale = d.softmax_scale = ok
        assert lib.lbw_attention_packed_fwd(ctypes.byref(p), None, 0, None) == 0
        assert lib.lbw_attention_decode(ctypes.byref(d), None, 0, None) == 0
