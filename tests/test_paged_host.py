"""Operators over a paged cache on the CPU: refusals of the C entry points (all before any launch), the structs, shapes
for tracing, the wrappers' errors."""
import ctypes
import os

import pytest
import torch

from test_capi import _header_struct, _header_struct_fields, _layout

BF = torch.bfloat16
NAMES = [("lbw_paged_kv", "PagedKv"), ("lbw_paged_append_params", "PagedAppendParams"),
         ("lbw_attention_paged_params", "AttentionPagedParams"), ("lbw_paged_select_params", "PagedSelectParams")]
ADDR = 0x7f0000000000  # an aligned address that nothing follows: every call below is refused before a launch


@pytest.mark.parametrize("cname,pyname", NAMES)
def test_structs_match_the_header(cname, pyname):
    from lbw_amd import _lib
    py = getattr(_lib, pyname)
    assert [f[0] for f in py._fields_] == _header_struct_fields(cname)
    kv = _header_struct("lbw_paged_kv", {})
    assert _layout(py) == _layout(_header_struct(cname, {"lbw_paged_kv": kv}))


def _cache(p, heads, dim, page=64, pages=4, width=3):
    c = p.cache
    c.k = c.v = c.bounds = c.table = ADDR
    c.k_stride_p = c.v_stride_p = heads * page * dim
    c.k_stride_l = c.v_stride_l = dim
    c.k_stride_h = c.v_stride_h = page * dim
    c.pages, c.page_size, c.table_stride, c.table_width = pages, page, width, width
    return p


def _append(**kw):
    from lbw_amd import _lib
    p = _cache(_lib.PagedAppendParams(), 2, 128)
    p.tokens, p.batch, p.q_heads, p.k_heads, p.head_dim = 3, 3, 4, 2, 128
    for n, h in (("q", 4), ("k", 2), ("v", 2), ("q_out", 4)):
        setattr(p, n, ADDR)
        setattr(p, n + "_stride_l", h * 128)
        setattr(p, n + "_stride_h", 128)
    p.rope, p.rope_rows, p.rope_pairs, p.n_axes = ADDR, 10, 64, 1
    p.axis_pairs[0] = 64
    p.pos, p.pos_stride, p.lens = ADDR, 1, ADDR
    p.q_out_scale = p.k_out_scale = 1.0
    return _set(p, kw)


def _attention(**kw):
    from lbw_amd import _lib
    p = _cache(_lib.AttentionPagedParams(), 2, 128)
    _queries(p)
    p.out, p.out_stride_b, p.out_stride_h = ADDR, 512, 128
    return _set(p, kw)


def _select(**kw):
    from lbw_amd import _lib
    p = _cache(_lib.PagedSelectParams(), 2, 128)
    _queries(p)
    p.count, p.first, p.last, p.selected = 2, 1, 1, ADDR
    return _set(p, kw)


def _queries(p):
    p.batch, p.q_heads, p.k_heads, p.head_dim = 3, 4, 2, 128
    p.q, p.q_stride_b, p.q_stride_h, p.lens = ADDR, 512, 128, ADDR


def _set(p, kw):
    for n, x in kw.items():
        at = p
        *path, last = n.split(".")
        for s in path:
            at = getattr(at, s)
        if last == "axis0":
            at.axis_pairs[0] = x
        else:
            setattr(at, last, x)
    return p


CACHE = [({"cache.page_size": 48}, "page_size"), ({"cache.page_size": 8}, "page_size"),
         ({"cache.page_size": 2048}, "page_size"), ({"cache.page_size": 0}, "page_size"),
         ({"cache.page_size": -64}, "page_size"), ({"cache.pages": 0}, "pages"), ({"cache.pages": -5}, "pages"),
         ({"cache.table_width": -1}, "table_width"), ({"cache.table_stride": -3}, "table_stride"),
         ({"cache.table": None}, "table missing"), ({"lens": None}, "lens missing"),
         ({"q_heads": 3}, "must divide"), ({"k_heads": 0}, "must divide"), ({"q": ADDR + 8}, "q must be"),
         ({"q": None}, "q must be")]
KV = [({"cache.k": None}, "cache's k"), ({"cache.v": ADDR + 2}, "cache's v"), ({"cache.k_stride_l": 100}, "multiples of 8"),
      ({"cache.v_stride_h": -128}, "negative"), ({"cache.k_stride_p": 12}, "page stride"),
      ({"cache.v_stride_p": -8}, "page stride"), ({"cache.k_stride_l": 1 << 24}, "token stride")]


@pytest.mark.parametrize("kw,message", CACHE + KV + [
    ({"tokens": -1}, "tokens"), ({"batch": -1}, "batch"), ({"batch": 2}, "need starts"), ({"head_dim": 96}, "head_dim"),
    ({"n_axes": 0}, "n_axes"), ({"axis0": 60}, "add up"), ({"rope": ADDR + 4}, "rotation table"),
    ({"eps": -1.0, "norm": 1}, "eps"), ({"wq": ADDR, "wk": ADDR}, "without the norm"),
    ({"wq": ADDR + 4, "norm": 1}, "weights"), ({"pos": None, "n_axes": 2}, "pos missing"),
    ({"v": None}, "v must be"), ({"q_out": ADDR + 4}, "q_out must be"), ({"q_out_stride_h": 1 << 26}, "head stride"),
    ({"cache.k_stride_h": 1 << 26}, "head stride"), ({"cache.bounds": ADDR + 8}, "bounds"),
    ({"tokens": 33554431, "batch": 33554431}, "above")])
def test_append_refusals(kw, message):
    from lbw_amd import _lib
    lib = _lib.load()
    assert lib.lbw_paged_append(ctypes.byref(_append(**kw)), None) != 0
    assert message in lib.lbw_last_error().decode()


@pytest.mark.parametrize("kw,message", CACHE + KV + [
    ({"batch": -2}, "batch"), ({"head_dim": 64}, "only 128"), ({"out": None}, "out must be"),
    ({"out_stride_h": 4}, "multiples"), ({"num_splits": 129}, "num_splits"), ({"num_splits": -1}, "num_splits"),
    ({"softmax_scale": -1.0}, "softmax_scale"), ({"softmax_scale": 1e8}, "softmax_scale"),
    ({"softmax_scale": float("nan")}, "softmax_scale"), ({"softmax_scale": float("inf")}, "softmax_scale"),
    ({"selected": ADDR, "n_selected": -1}, "n_selected"), ({"selected": ADDR, "n_selected": 1 << 25}, "n_selected"),
    ({"prefix_keys": 5}, "prefix"), ({"prefix_keys": -1}, "prefix"),
    ({"prefix_keys": 129, "prefix_width": 2, "prefix_table": ADDR}, "prefix"),
    ({"prefix_keys": 128, "prefix_width": 2}, "prefix_table missing"),
    ({"batch": 1 << 20, "q_heads": 64}, "batch")])
def test_attention_refusals(kw, message):
    from lbw_amd import _lib
    lib = _lib.load()
    p = _attention(**kw)
    assert lib.lbw_attention_paged_workspace_size(ctypes.byref(p)) == 0
    assert lib.lbw_attention_paged(ctypes.byref(p), None, 0, None) != 0
    assert message in lib.lbw_last_error().decode()


@pytest.mark.parametrize("kw,message", CACHE + [
    ({"count": 0}, "count"), ({"first": -1}, "count"), ({"last": 2}, "count"),
    ({"first": 2147483647, "last": 2147483647, "count": 2147483647}, "count"), ({"cache.bounds": None}, "bounds"),
    ({"cache.bounds": ADDR + 8}, "bounds"), ({"selected": None}, "selected"), ({"head_dim": 256}, "only 128"),
    ({"batch": 1 << 23}, "batch")])
def test_select_refusals(kw, message):
    from lbw_amd import _lib
    lib = _lib.load()
    p = _select(**kw)
    assert lib.lbw_paged_select_workspace_size(ctypes.byref(p)) == 0
    assert lib.lbw_paged_select(ctypes.byref(p), None, 0, None) != 0
    assert message in lib.lbw_last_error().decode()


def test_prefixes_of_more_pieces_than_a_launch_has():
    """A piece lists 4095 pages at most, so 2^27 pages of 16 tokens make 32801 pieces, here for 16000 query rows."""
    from lbw_amd import _lib
    lib = _lib.load()
    long = {"prefix_table": ADDR, "prefix_width": 1 << 27, "prefix_keys": 0x7fffff00, "cache.page_size": 16,
            "q_heads": 8, "k_heads": 8}
    p = _attention(batch=16000, **long)
    assert lib.lbw_attention_paged_workspace_size(ctypes.byref(p)) == 0
    assert lib.lbw_attention_paged(ctypes.byref(p), None, 0, None) == 2
    assert "prefix of 2147483392 keys in pages of 16" in lib.lbw_last_error().decode()
    assert lib.lbw_attention_paged_workspace_size(ctypes.byref(_attention(batch=100, **long))) > 100 * 8 * 32800 * 520
    # as many as a launch has, and more
    big = {"q_heads": 40, "k_heads": 8, "batch": 400000}
    assert lib.lbw_attention_paged_workspace_size(ctypes.byref(_attention(num_splits=1, **big))) == 0
    assert lib.lbw_attention_paged(ctypes.byref(_attention(num_splits=128, selected=ADDR, n_selected=1, **big)), None, 0,
                                   None) == 2
    assert "num_splits 128" in lib.lbw_last_error().decode()


def test_null_params_and_empty_calls():
    from lbw_amd import _lib
    lib = _lib.load()
    assert lib.lbw_paged_append(None, None) != 0
    assert lib.lbw_attention_paged(None, None, 0, None) != 0
    assert lib.lbw_paged_select(None, None, 0, None) != 0
    # nothing to do: no launch, no pointers wanted
    assert lib.lbw_paged_append(ctypes.byref(_append(tokens=0, batch=0, q=None, k=None, v=None, q_out=None, lens=None,
                                                     **{"cache.table": None})), None) == 0
    assert lib.lbw_attention_paged(ctypes.byref(_attention(batch=0, q=None, out=None, lens=None)), None, 0, None) == 0
    assert lib.lbw_paged_select(ctypes.byref(_select(batch=0, q=None, selected=None, lens=None)), None, 0, None) == 0


def test_workspaces():
    from lbw_amd import _lib
    lib = _lib.load()
    # scores only where a table is wider than the choice and not short: 8 bytes a page
    wide = {"cache.table_width": 1000, "cache.table_stride": 1000}
    assert lib.lbw_paged_select_workspace_size(ctypes.byref(_select(count=1000, **wide))) == 0
    assert lib.lbw_paged_select_workspace_size(ctypes.byref(_select())) == 0
    p = _select(**wide)
    assert lib.lbw_paged_select_workspace_size(ctypes.byref(p)) == 3 * 2 * 1000 * 8
    assert lib.lbw_paged_select(ctypes.byref(p), None, 0, None) == 4
    assert lib.lbw_paged_select(ctypes.byref(p), ctypes.c_void_p(ADDR + 8), 1 << 20, None) == 4
    # partial results of 130 floats a row: (pieces + batch) or batch * splits rows a head
    p = _attention(num_splits=3)
    assert lib.lbw_attention_paged_workspace_size(ctypes.byref(p)) == 4 * (3 * 3 + 3) * 130 * 4
    p = _attention(num_splits=3, selected=ADDR, n_selected=2)
    assert lib.lbw_attention_paged_workspace_size(ctypes.byref(p)) == 4 * (3 * 3) * 130 * 4
    p = _attention(num_splits=1, prefix_table=ADDR, prefix_width=2, prefix_keys=100)
    assert lib.lbw_attention_paged_workspace_size(ctypes.byref(p)) == 4 * (3 + 3) * 130 * 4
    assert lib.lbw_attention_paged(ctypes.byref(p), None, 0, None) == 4
    assert lib.lbw_attention_paged(ctypes.byref(p), ctypes.c_void_p(ADDR), 100, None) == 4
    assert lib.lbw_attention_paged_workspace_size(ctypes.byref(_attention(num_splits=1))) == 0


def _meta(*shape, dtype=BF):
    return torch.empty(*shape, dtype=dtype, device="meta")


def test_shapes_for_tracing():
    from lbw_amd import _lib
    ops = _lib.ops()
    q, pool = _meta(3, 4, 128), _meta(9, 16, 2, 128)
    table, lens = _meta(3, 5, dtype=torch.int32), _meta(3, dtype=torch.int32)
    out = ops.attention_paged(q, pool, pool, table, lens)
    assert out.shape == q.shape and out.dtype == BF
    sel = ops.paged_select(q, _meta(9, 2, 2, 128), table, lens, 16, 7, 1, 1)
    assert sel.shape == (3, 2, 7) and sel.dtype == torch.int32
    ops.attention_paged_out(q, pool, pool, table, lens, sel, None, None, -1, 0.0, 0, _meta(3, 4, 128))
    ops.paged_append_(q, _meta(3, 2, 128), _meta(3, 2, 128), None, None, _meta(8, 64, 2, dtype=torch.float32), [64],
                      True, None, False, 0.0, 1.0, 1.0, table, lens, None, q, pool, pool, None)


def test_no_gradients_and_no_tangents():
    import torch.autograd.forward_ad as fwd
    from lbw_amd import _lib
    ops = _lib.ops()
    q, pool, edge = _meta(3, 4, 128), _meta(9, 16, 2, 128), _meta(9, 2, 2, 128)
    table, lens = _meta(3, 5, dtype=torch.int32), _meta(3, dtype=torch.int32)

    def calls(q):
        return [lambda: ops.attention_paged(q, pool, pool, table, lens),
                lambda: ops.paged_select(q, edge, table, lens, 16, 7, 1, 1),
                lambda: ops.attention_paged_out(q, pool, pool, table, lens, None, None, None, -1, 0.0, 0, _meta(3, 4, 128)),
                lambda: ops.paged_append_(q, _meta(3, 2, 128), _meta(3, 2, 128), None, None,
                                          _meta(8, 64, 2, dtype=torch.float32), [64], True, None, False, 0.0, 1.0, 1.0,
                                          table, lens, None, _meta(3, 4, 128), pool, pool, None)]

    wanted = calls(_meta(3, 4, 128).requires_grad_())
    out = wanted[0]()
    with pytest.raises(RuntimeError, match="not implemented"):
        out.backward(torch.empty_like(out))
    assert not wanted[1]().requires_grad
    for call in wanted[2:]:
        with pytest.raises(NotImplementedError, match="not differentiable"):
            call()
        with torch.no_grad():
            call()
    with fwd.dual_level():
        for call in calls(fwd.make_dual(q, _meta(3, 4, 128))):
            with pytest.raises(NotImplementedError):
                call()


def test_wrapper_errors():
    """Wrong arguments are named, whatever device they are on."""
    import lbw_amd as L
    q, k = torch.zeros(3, 4, 128, dtype=BF), torch.zeros(3, 2, 128, dtype=BF)
    c = L.paged_kv(5, 16, 2, bounds=True, device="cpu")
    assert c.k.shape == c.v.shape == (5, 16, 2, 128) and c.bounds.shape == (5, 2, 2, 128)
    assert c.k.stride() == (2 * 16 * 128, 128, 16 * 128, 1)
    table, lens = torch.zeros(3, 4, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    rope = L.axis_rope(torch.zeros(8, 64), device="cpu")
    rope3 = L.axis_rope(torch.zeros(8, 64), (22, 21, 21), device="cpu")
    for bad in ((0, 16, 2), (4, 48, 2), (4, 8, 2), (4, 2048, 2), (4, 16, 0)):
        with pytest.raises(ValueError):
            L.paged_kv(*bad, device="cpu")

    def append(match, cache=c, q=q, k=k, v=k, table=table, lens=lens, rope=rope, pos=None, **kw):
        with pytest.raises(ValueError, match=match):
            L.paged_append_(cache, q, k, v, table, lens, rope, pos, **kw)

    append("k .* do not fit", k=k[:2])
    append("do not fit", v=k[:, :1])
    append("q must be", q=q.float())
    append("q_out", q_out=torch.zeros(3, 5, 128, dtype=BF))
    append("belong to the norm", wq=torch.ones(128), wk=torch.ones(128))
    append("both or neither", wq=torch.ones(128), eps=1e-6)
    append("needs pos", rope=rope3)
    append("pos must be", pos=torch.zeros(3, 2, dtype=torch.int32))
    append("pos must be", pos=torch.zeros(3))
    append("lens must be", lens=lens.long())
    append("lens must be", lens=lens[:2])
    append("table must be", table=table[0])
    append("starts must be", starts=lens)
    append("cache.k must be", cache=L.PagedKV(c.k[:, :, :1], c.v))
    append("cache.bounds", cache=L.PagedKV(c.k, c.v, c.bounds[:3]))
    append("page_size 5", cache=L.PagedKV(c.k[:, :5], c.v[:, :5]))

    def attend(match, q=q, cache=c, table=table, lens=lens, **kw):
        with pytest.raises(ValueError, match=match):
            L.attention_paged(q, cache, table, lens, **kw)

    attend("q must be", q=q[..., :64])
    attend("do not divide", q=q[:, :3])
    attend("cache.v must be", cache=L.PagedKV(c.k, c.v[:2]))
    attend("lens must be", lens=lens.float())
    attend("num_splits", num_splits=200)
    attend("selected must be", selected=torch.zeros(3, 4, 2, dtype=torch.int32))
    attend("without prefix_table", prefix_len=3)
    attend("without prefix_table", prefix_len=lens[:1])
    attend("is negative", prefix_table=table[0], prefix_len=-1)
    attend("prefix_table must be", prefix_table=table)
    attend("prefix_len 65", prefix_table=table[0], prefix_len=65)
    attend("prefix_len must be", prefix_table=table[0], prefix_len=lens)
    attend("out must be", out=q.float())
    attend("softmax_scale", softmax_scale=-2.0)

    def select(match, q=q, cache=c, table=table, lens=lens, count=2, **kw):
        with pytest.raises(ValueError, match=match):
            L.paged_select(q, cache, table, lens, count, **kw)

    select("no bounds", cache=L.PagedKV(c.k, c.v))
    select("q must be", q=q[0])
    select("count 0", count=0)
    select("count 2", first=2, last=1)
    select("table must be", table=table.long())


def test_calls_on_the_cpu_raise():
    """Right arguments on the CPU: there is no fallback."""
    import lbw_amd as L
    c = L.paged_kv(5, 16, 2, bounds=True, device="cpu")
    q, table, lens = torch.zeros(3, 4, 128, dtype=BF), torch.zeros(3, 4, dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    with pytest.raises((RuntimeError, NotImplementedError)):
        L.attention_paged(q, c, table, lens)
    with pytest.raises((RuntimeError, NotImplementedError)):
        L.paged_select(q, c, table, lens, 2)
    with pytest.raises((RuntimeError, NotImplementedError)):
        L.paged_append_(c, q, q[:, :2], q[:, :2], table, lens, L.axis_rope(torch.zeros(8, 64), device="cpu"))


def test_exported_from_the_package():
    import lbw_amd
    for n in ("PagedKV", "paged_kv", "paged_append_", "attention_paged", "paged_select"):
        assert n in lbw_amd.__all__ and hasattr(lbw_amd, n)
    assert os.path.exists(lbw_amd._lib.OPS_PATH)
