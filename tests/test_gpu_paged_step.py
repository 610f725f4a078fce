"""The operators over a paged cache together, as a serving loop uses them: prompts into pages, tokens one by one, branches off
one history, windows of which only some pages are looked at; captured into graphs, compiled, on other streams and from
several threads."""
import math
import threading

import pytest
import torch

import packed_ref as R
import paged_ref as P

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
HQ, HK, D, PAGE = 6, 2, 128, 16
SCALE = 1 / math.sqrt(D)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Model:
    """One attention layer's state: norm weights, a rotation of three axes, a pool of pages that are handed out in turn."""

    def __init__(self, batch, width, pages, seed=0):
        import lbw_amd
        g = torch.Generator().manual_seed(seed)
        self.g = g
        self.w = [(1 + 0.1 * torch.randn(D, generator=g)).to(BF).cuda() for _ in range(2)]
        self.angles = lbw_amd.wan_rope_freqs(D, 512).cuda()
        self.rope = lbw_amd.axis_rope(self.angles, (22, 21, 21))
        self.cache = lbw_amd.paged_kv(pages, PAGE, HK, bounds=True)
        for x in (self.cache.k, self.cache.v, self.cache.bounds):
            x.fill_(float("nan"))            # nothing that was not written may matter
        self.free = torch.randperm(pages, generator=g).int().tolist()
        self.table = torch.full((batch, width), -1, dtype=torch.int32, device="cuda")
        self.lens = torch.zeros(batch, dtype=torch.int32, device="cuda")
        self.host = [0] * batch
        self.seen = [[] for _ in range(batch)]   # (q, k, v, pos) of every token so far

    def grow(self, b, n):
        have, need = P.pages_of(self.host[b], PAGE), P.pages_of(self.host[b] + n, PAGE)
        for j in range(have, need):
            self.table[b, j] = self.free.pop()
        self.host[b] += n

    def tokens(self, n):
        qkv = torch.randn(n, HQ + 2 * HK, D, generator=self.g).to(BF).cuda()
        pos = torch.randint(0, 60, (n, 3), generator=self.g, dtype=torch.int32).cuda()
        return qkv, pos

    def append(self, new, starts=True):
        """new[b] tokens for every sequence -> their turned q."""
        import lbw_amd
        qkv, pos = self.tokens(sum(new))
        q, k, v = qkv.split([HQ, HK, HK], 1)
        for b, n in enumerate(new):
            self.grow(b, n)
        st = _i32([sum(new[:b]) for b in range(len(new) + 1)]) if starts else None
        out = lbw_amd.paged_append_(self.cache, q, k, v, self.table, self.lens, self.rope, pos, starts=st,
                                    wq=self.w[0], wk=self.w[1], eps=1e-6)
        self.lens += _i32(new)
        at = 0
        for b, n in enumerate(new):
            s = slice(at, at + n)
            self.seen[b].append((k[s], v[s], pos[s]))
            at += n
        return out, q, pos

    def keys(self, b):
        """k' and v of sequence b as the cache has them, checked against the definition."""
        n = self.host[b]
        k, v = (P.rows(x, self.table[b, :P.pages_of(n, PAGE)], n) for x in (self.cache.k, self.cache.v))
        if n:
            raw_k, raw_v, pos = (torch.cat(x) for x in zip(*self.seen[b]))
            want = P.turned(raw_k, self.w[1], R.token_angles(self.angles, (22, 21, 21), pos), True, 1e-6, 1.0)
            R.assert_within(f"keys of sequence {b}", k, want, R.head_norm_allow(want))
            assert torch.equal(v, raw_v)
            for j in range(P.pages_of(n, PAGE)):
                rows = k[j * PAGE:(j + 1) * PAGE]
                assert torch.equal(self.cache.bounds[self.table[b, j].long()],
                                   torch.stack((rows.amin(0), rows.amax(0)), 1))
        return k, v

    def check(self, out, q, pos, prefix=None, prefix_len=0, selected=None):
        wq = P.turned(q, self.w[0], R.token_angles(self.angles, (22, 21, 21), pos), True, 1e-6, 1.0)
        R.assert_within("q", self.q, wq, R.head_norm_allow(wq))
        for b in range(len(self.host)):
            self.keys(b)
        want, allow = P.attention(self.q, self.cache.k, self.cache.v, self.table, self.host, SCALE, prefix, prefix_len,
                                  selected)
        R.assert_within("out", out, want, allow)


def test_prompts_then_tokens():
    import lbw_amd
    m = Model(3, 12, 40)
    m.append([40, 0, 17])
    m.append([3, 70, 15])                    # prompts that go on inside begun pages
    for step in range(20):
        m.q, q, pos = m.append([1, 1, 1], starts=step % 2 == 0)
        out = lbw_amd.attention_paged(m.q, m.cache, m.table, m.lens)
        if step % 4 == 3:
            m.check(out, q, pos)


def test_branches_off_one_history():
    """A prompt whose pages become the prefix of five branches; each goes on in pages of its own."""
    import lbw_amd
    one = Model(1, 12, 12, seed=1)
    one.append([150])
    prefix = one.table[0, :10].contiguous()
    m = Model(5, 6, 40, seed=1)
    m.cache = one.cache
    used = set(one.table[0].tolist())
    big = lbw_amd.paged_kv(60, PAGE, HK, bounds=True)
    for a, b in zip((big.k, big.v, big.bounds), (one.cache.k, one.cache.v, one.cache.bounds)):
        a.fill_(float("nan"))
        a[:12] = b
    m.cache = big
    m.free = [p for p in range(60) if p not in used]
    m.append([20, 0, 1, 33, 16])
    for step in range(6):
        m.q, q, pos = m.append([1] * 5, starts=False)
        out = lbw_amd.attention_paged(m.q, m.cache, m.table, m.lens, prefix_table=prefix, prefix_len=150)
        m.check(out, q, pos, prefix, 150)
    alone = lbw_amd.attention_paged(m.q, m.cache, m.table, m.lens)
    m.check(alone, q, pos)


def test_looking_at_some_pages():
    import lbw_amd
    m = Model(2, 40, 90, seed=2)
    m.append([400, 333])
    for step in range(8):
        m.q, q, pos = m.append([1, 1], starts=False)
        sel = lbw_amd.paged_select(m.q, m.cache, m.table, m.lens, 7, first=1, last=2)
        assert torch.equal(sel.cpu(), P.select(m.q, m.cache.bounds, m.table, m.host, PAGE, 7, 1, 2))
        m.check(lbw_amd.attention_paged(m.q, m.cache, m.table, m.lens, selected=sel), q, pos, selected=sel)
    # as many as there are: the whole sequence
    sel = lbw_amd.paged_select(m.q, m.cache, m.table, m.lens, 40)
    m.check(lbw_amd.attention_paged(m.q, m.cache, m.table, m.lens, selected=sel), q, pos)


def _step_state(seed, batch=3, width=70, prefix=100):
    import lbw_amd
    g = torch.Generator().manual_seed(seed)
    pages = batch * width + 10
    pool = P.make_pool(pages, PAGE, HK, D, g)
    cache = lbw_amd.PagedKV(*pool, torch.stack((pool[0].amin(1), pool[0].amax(1)), 2).contiguous())
    order = torch.randperm(pages, generator=g).int()
    table = order[:batch * width].view(batch, width).cuda()
    rope = lbw_amd.axis_rope(lbw_amd.wan_rope_freqs(D, 2048).cuda(), interleaved=False)
    lens = torch.randint(0, width * PAGE, (batch,), generator=g, dtype=torch.int32).cuda()
    qkv = torch.randn(batch, HQ + 2 * HK, D, generator=g).to(BF).cuda()
    return {"cache": cache, "table": table, "rope": rope, "lens": lens, "qkv": qkv,
            "prefix": order[batch * width:batch * width + 7].cuda(), "prefix_len": _i32([prefix])}


def _step(s, count=9):
    """One decode step: the token appended, then attention over all keys behind the prefix, and over selected pages."""
    import lbw_amd
    q, k, v = s["qkv"].split([HQ, HK, HK], 1)
    q2 = lbw_amd.paged_append_(s["cache"], q, k, v, s["table"], s["lens"], s["rope"], eps=1e-6)
    now = s["lens"] + 1
    out = lbw_amd.attention_paged(q2, s["cache"], s["table"], now, prefix_table=s["prefix"],
                                  prefix_len=s["prefix_len"])
    own = lbw_amd.attention_paged(q2, s["cache"], s["table"], now)
    sel = lbw_amd.paged_select(q2, s["cache"], s["table"], now, count, first=1, last=2)
    return q2, out, own, sel, lbw_amd.attention_paged(q2, s["cache"], s["table"], now, selected=sel)


def _copy(s):
    import lbw_amd
    c = s["cache"]
    return {**s, "cache": lbw_amd.PagedKV(c.k.clone(), c.v.clone(), c.bounds.clone())}


def _same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def _same_cache(a, b):
    return _same((a["cache"].k, a["cache"].v, a["cache"].bounds), (b["cache"].k, b["cache"].v, b["cache"].bounds))


def test_captured_steps_follow_the_device():
    """Two graphs of the step, replayed in turn with new lengths, tables, tokens and prefix lengths, eager work between."""
    s = _step_state(1)
    _step(_copy(s))
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = _step(s)
        graphs.append((g, got))
    for seed in (2, 3, 4, 5):
        new = _step_state(seed, prefix=(0, 33, 112, 5000)[seed - 2])
        for n in ("lens", "qkv", "table", "prefix", "prefix_len"):
            s[n].copy_(new[n])
        if seed == 3:
            s["lens"][1] = 0
        for g, got in graphs:
            for x, y in zip((s["cache"].k, s["cache"].v, s["cache"].bounds),
                            (new["cache"].k, new["cache"].v, new["cache"].bounds)):
                x.copy_(y)
            eager = _copy(s)
            g.replay()
            want = _step(eager)              # (eager work while the graph may still run)
            torch.cuda.synchronize()
            assert _same(got, want) and _same_cache(s, eager)


def test_captured_prompt():
    import lbw_amd
    s = _step_state(6)
    T = 90
    g0 = torch.Generator().manual_seed(7)
    qkv = torch.randn(T, HQ + 2 * HK, D, generator=g0).to(BF).cuda()
    starts, q_out = _i32([0, 30, 30, 90]), torch.zeros(T, HQ, D, dtype=BF, device="cuda")
    s["lens"].copy_(_i32([3, 40, 100]))
    q, k, v = qkv.split([HQ, HK, HK], 1)

    def run(cache, out):
        return lbw_amd.paged_append_(cache, q, k, v, s["table"], s["lens"], s["rope"], starts=starts, q_out=out)

    run(_copy(s)["cache"], q_out.clone())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        run(s["cache"], q_out)
    for new in ([0, 30, 30, 90], [0, 0, 90, 90], [5, 6, 40, 41], [0, 90, 90, 90]):
        starts.copy_(_i32(new))
        qkv.normal_()
        q_out.fill_(3.0)
        eager, want = _copy(s), q_out.clone()
        g.replay()
        run(eager["cache"], want)
        torch.cuda.synchronize()
        assert torch.equal(q_out, want) and _same_cache(s, eager)


def test_other_streams_and_threads_at_once():
    jobs = []
    for i in range(4):
        s = _step_state(20 + i, batch=2 + i)
        jobs.append((s, _step(_copy(s))))
    torch.cuda.synchronize()
    bad = []

    def work(s, want):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(5):
                    got = _step(s)           # (the same rows again: the same cache)
                    stream.synchronize()
                    if not _same(got, want):
                        bad.append("differs")
        except Exception as e:  # noqa: BLE001
            bad.append(repr(e))
    threads = [threading.Thread(target=work, args=j) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad, bad


def test_tensors_made_on_another_stream():
    s = _step_state(30)
    want = _step(_copy(s))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        mine = _copy(s)
        mine["qkv"] = s["qkv"].clone()
        got = _step(mine)
    torch.cuda.current_stream().wait_stream(side)
    assert _same(got, want)


@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_compiled_step_gives_the_same_bits(backend):
    """One graph, no break: append, attention, selection, attention over it."""
    s = _step_state(40)
    want_state, got_state = _copy(s), _copy(s)
    want = _step(want_state)
    torch._dynamo.reset()

    def step(k, v, bounds, table, lens, qkv, prefix, prefix_len):
        import lbw_amd
        return _step({"cache": lbw_amd.PagedKV(k, v, bounds), "table": table, "rope": s["rope"], "lens": lens,
                      "qkv": qkv, "prefix": prefix, "prefix_len": prefix_len})

    c = got_state["cache"]
    got = torch.compile(step, backend=backend, fullgraph=True)(
        c.k, c.v, c.bounds, s["table"], s["lens"], s["qkv"], s["prefix"], s["prefix_len"])
    assert _same(got, want) and _same_cache(got_state, want_state)


def test_under_inference_mode_and_fake_tensors():
    import lbw_amd
    from torch._subclasses.fake_tensor import FakeTensorMode
    s = _step_state(50)
    want = _step(_copy(s))
    with torch.inference_mode():
        mine = _copy(s)
        assert _same(_step(mine), want)
    with FakeTensorMode(allow_non_fake_inputs=True):
        q = torch.empty(16, HQ, D, dtype=BF, device="cuda")
        pool = torch.empty(9, PAGE, HK, D, dtype=BF, device="cuda")
        table, lens = (torch.empty(*x, dtype=torch.int32, device="cuda") for x in ((16, 5), (16,)))
        cache = lbw_amd.PagedKV(pool, pool, torch.empty(9, HK, 2, D, dtype=BF, device="cuda"))
        sel = lbw_amd.paged_select(q, cache, table, lens, 4)
        assert sel.shape == (16, HK, 4)
        assert lbw_amd.attention_paged(q, cache, table, lens, selected=sel).shape == q.shape


def test_large_batches():
    """More sequences than a wave has lanes, of very different lengths, in every form."""
    import lbw_amd
    g = torch.Generator().manual_seed(60)
    B = 200
    old = torch.randint(0, 300, (B,), generator=g).tolist()
    new = [int(x) if x > 0 else 0 for x in torch.randint(-2, 6, (B,), generator=g)]
    m = Model(B, 22, 4400, seed=61)
    m.append(old)
    m.append(new)
    m.q, q, pos = m.append([1] * B, starts=False)
    out = lbw_amd.attention_paged(m.q, m.cache, m.table, m.lens)
    for splits in (0, 1, 2):
        again = lbw_amd.attention_paged(m.q, m.cache, m.table, m.lens, num_splits=splits)
        want, allow = P.attention(m.q, m.cache.k, m.cache.v, m.table, m.host, SCALE)
        R.assert_within("out", again, want, allow)
    prefix = m.table[0, :4].contiguous()
    n = min(50, m.host[0])
    out = lbw_amd.attention_paged(m.q, m.cache, m.table, m.lens, prefix_table=prefix, prefix_len=n)
    m.check(out, q, pos, prefix, n)
    sel = lbw_amd.paged_select(m.q, m.cache, m.table, m.lens, 5, first=1, last=1)
    assert torch.equal(sel.cpu(), P.select(m.q, m.cache.bounds, m.table, m.host, PAGE, 5, 1, 1))
    out = lbw_amd.attention_paged(m.q, m.cache, m.table, m.lens, selected=sel)
    want, allow = P.attention(m.q, m.cache.k, m.cache.v, m.table, m.host, SCALE, selected=sel)
    R.assert_within("selected", out, want, allow)


def test_several_tokens_of_one_sequence_are_as_many_rows():
    """A draft is appended at once; each of its tokens looks at what is before it, itself included."""
    import lbw_amd
    m = Model(3, 12, 40, seed=70)
    m.append([40, 0, 90])
    before, new = list(m.host), [5, 3, 0]
    m.q, q, pos = m.append(new)
    row = [b for b, n in enumerate(new) for _ in range(n)]
    lens = [before[b] + 1 + i for b, n in enumerate(new) for i in range(n)]
    table = m.table[row].contiguous()
    out = lbw_amd.attention_paged(m.q, m.cache, table, _i32(lens))
    want, allow = P.attention(m.q, m.cache.k, m.cache.v, table, lens, SCALE)
    R.assert_within("out", out, want, allow)
    sel = lbw_amd.paged_select(m.q, m.cache, table, _i32(lens), 2, first=1, last=1)
    assert torch.equal(sel.cpu(), P.select(m.q, m.cache.bounds, table, lens, PAGE, 2, 1, 1))
    # taken back and written anew: bounds that hold what is there, and may be wider
    m.lens -= _i32(new)
    q2, k2, v2 = torch.randn(8, HQ + 2 * HK, D, generator=m.g).to(BF).cuda().split([HQ, HK, HK], 1)
    lbw_amd.paged_append_(m.cache, q2, k2, v2, m.table, m.lens, m.rope, pos, starts=_i32([0, 5, 8, 8]), wq=m.w[0],
                          wk=m.w[1], eps=1e-6)
    for b in range(3):
        n = before[b] + new[b]
        k = P.rows(m.cache.k, m.table[b, :P.pages_of(n, PAGE)], n)
        for j in range(P.pages_of(n, PAGE)):
            lo, hi = m.cache.bounds[m.table[b, j].long()].unbind(1)
            rows = k[j * PAGE:(j + 1) * PAGE]
            assert (lo <= rows.amin(0)).all() and (hi >= rows.amax(0)).all()


def test_a_prompt_beside_packed_attention():
    """The last token of a prompt over its pages is the last row of attention over the prompt packed."""
    import lbw_amd
    m = Model(2, 12, 40, seed=71)
    qkv, pos = m.tokens(150)
    q, k, v = qkv.split([HQ, HK, HK], 1)
    m.grow(0, 100), m.grow(1, 50)
    starts = _i32([0, 100, 150])
    qt = lbw_amd.paged_append_(m.cache, q, k, v, m.table, m.lens, m.rope, pos, starts=starts, wq=m.w[0], wk=m.w[1],
                               eps=1e-6)
    m.lens += starts.diff()
    qn, kn = lbw_amd.qk_head_norm_rope(q, k, m.w[0], m.w[1], m.rope, pos, eps=1e-6)
    assert torch.equal(qn, qt)
    for b, (s, e) in enumerate(((0, 100), (100, 150))):
        assert torch.equal(P.rows(m.cache.k, m.table[b, :P.pages_of(e - s, PAGE)], e - s), kn[s:e])
    packed = lbw_amd.attention_packed(qn, kn, v, lbw_amd.packed_plan([100, 50]))
    out = lbw_amd.attention_paged(qt[[99, 149]].contiguous(), m.cache, m.table, m.lens)
    want, allow = P.attention(qt[[99, 149]], m.cache.k, m.cache.v, m.table, m.host, SCALE)
    R.assert_within("paged", out, want, allow)
    R.assert_within("packed", packed[[99, 149]], want, allow)


def test_tensors_on_two_devices_are_refused():
    import lbw_amd
    s = _step_state(72)
    c, q = s["cache"], s["qkv"][:, :HQ].contiguous()
    cpu = lbw_amd.PagedKV(c.k.cpu(), c.v.cpu(), c.bounds.cpu())
    for kw in ({"q": q.cpu()}, {"cache": cpu}, {"table": s["table"].cpu()}, {"lens": s["lens"].cpu()}):
        a = {"q": q, "cache": c, "table": s["table"], "lens": s["lens"], **kw}
        with pytest.raises((RuntimeError, ValueError)):
            lbw_amd.attention_paged(**a)
        with pytest.raises((RuntimeError, ValueError)):
            lbw_amd.paged_select(**a, count=3)
        k = s["qkv"][:, HQ:HQ + HK]
        with pytest.raises((RuntimeError, ValueError)):
            lbw_amd.paged_append_(a["cache"], a["q"], k, k, a["table"], a["lens"], s["rope"])
    for kw in ({"prefix_table": s["prefix"].cpu()}, {"prefix_table": s["prefix"], "prefix_len": s["prefix_len"].cpu()},
               {"selected": torch.zeros(3, HK, 2, dtype=torch.int32)}, {"out": q.cpu()}):
        with pytest.raises((RuntimeError, ValueError)):
            lbw_amd.attention_paged(q, c, s["table"], s["lens"], **kw)


def test_thousands_of_sequences_are_as_a_few_of_them():
    import lbw_amd
    B, hq, hk, width = 4500, 40, 8, 3
    g = torch.Generator(device="cuda").manual_seed(80)
    k, v = (torch.randn(700, PAGE, hk, D, generator=g, device="cuda").to(BF) for _ in range(2))
    cache = lbw_amd.PagedKV(k, v, torch.stack((k.amin(1), k.amax(1)), 2).contiguous())
    table = torch.randint(0, 700, (B, width), generator=g, device="cuda", dtype=torch.int32)
    lens = torch.randint(0, width * PAGE + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    q = torch.randn(B, hq, D, generator=g, device="cuda").to(BF)
    prefix = table[0]
    sel = lbw_amd.paged_select(q, cache, table, lens, 2)
    some = torch.randint(0, B, (60,), generator=g, device="cuda").tolist() + [0, B - 1]
    few = (q[some].contiguous(), cache, table[some].contiguous(), lens[some].contiguous())
    assert torch.equal(lbw_amd.paged_select(few[0], cache, few[2], few[3], 2), sel[some])
    for kw, kw_few in (({}, {}), ({"selected": sel}, {"selected": sel[some].contiguous()}),
                       ({"prefix_table": prefix, "prefix_len": 40},) * 2):
        got = lbw_amd.attention_paged(q, cache, table, lens, num_splits=1, **kw)
        want, allow = P.attention(few[0], k, v, few[2], few[3].tolist(), SCALE, kw.get("prefix_table"), kw.get("prefix_len", 0),
                                  kw_few.get("selected"))
        R.assert_within(str(list(kw)), got[some], want, allow)
        again = lbw_amd.attention_paged(q, cache, table, lens, **kw)
        R.assert_within(str(list(kw)), again[some], want, allow)
