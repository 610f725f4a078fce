"""The operators on packed sequences together, as a training step and a serving loop use them: per-head
norm + rotation into packed attention with the gradient back through both, prompt then tokens over the
cache, and captured into graphs, on other streams, from several threads."""
import math
import threading

import pytest
import torch

import packed_ref as R

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
HQ, HK, D = 6, 2, 128


def _setup(n, seed, inter=True):
    import lbw_amd
    g = torch.Generator().manual_seed(seed)
    qkv = (torch.randn(n, HQ + 2 * HK, D, generator=g)).to(BF).cuda()
    w = [(1 + 0.1 * torch.randn(D, generator=g)).to(BF).cuda() for _ in range(2)]
    ang = lbw_amd.wan_rope_freqs(D, 512).cuda()
    rope = lbw_amd.axis_rope(ang, (22, 21, 21), interleaved=inter)
    pos = torch.randint(0, 60, (n, 3), generator=g, dtype=torch.int32).cuda()
    do = torch.randn(n, HQ, D, generator=g).to(BF).cuda()
    return qkv, w, ang, rope, pos, do


def _step(qkv, wq, wk, rope, pos, plan, do):
    """Leaves -> (out, gradients)."""
    import lbw_amd
    q, k, v = qkv.split([HQ, HK, HK], 1)
    q2, k2 = lbw_amd.qk_head_norm_rope(q, k, wq, wk, rope, pos)
    out = lbw_amd.attention_packed(q2, k2, v, plan)
    return (out,) + torch.autograd.grad(out, (qkv, wq, wk), do)


def _leaves(*ts):
    return [t.detach().clone().requires_grad_() for t in ts]


def test_training_step_against_64_bits():
    import lbw_amd
    lens = [100, 1, 0, 77]
    n = sum(lens)
    qkv, w, ang, rope, pos, do = _setup(n, 1)
    leaves = _leaves(qkv, *w)
    out, dqkv, dwq, dwk = _step(*leaves, rope, pos, lbw_amd.packed_plan(lens), do)
    # the same step in 64 bits by autograd over elementary operations
    X, WQ, WK = [t.detach().double().requires_grad_() for t in leaves]
    a = R.token_angles(ang, (22, 21, 21), pos)
    q, k, v = X.split([HQ, HK, HK], 1)
    q2, k2 = R.head_norm(q, WQ, a, True, 1e-6, 1.0), R.head_norm(k, WK, a, True, 1e-6, 1.0)
    rows, at = [], 0
    for L in lens:
        s = slice(at, at + L)
        at += L
        kk, vv = k2[s].repeat_interleave(HQ // HK, 1), v[s].repeat_interleave(HQ // HK, 1)
        S = torch.einsum("ihd,jhd->hij", q2[s], kk) / math.sqrt(D)
        S = S.masked_fill(torch.ones(L, L, dtype=torch.bool, device="cuda").triu(1), -math.inf)
        rows.append(torch.einsum("hij,jhd->ihd", torch.softmax(S, -1), vv))
    O = torch.cat(rows)
    want = (O,) + torch.autograd.grad(O, (X, WQ, WK), do.double())
    # Each tensor between the operators is rounded to bf16 (q', k', dq', dk', out, the gradients) and P
    # and dS inside: a dozen roundings of H each, relative to the sums of the terms; in the 2-norm, where
    # independent roundings add in squares, below 4 H of the result.
    for name, x, y in zip(("out", "dqkv", "dwq", "dwk"), (out, dqkv, dwq, dwk), want):
        rel = ((x.double() - y).norm() / y.norm()).item()
        assert rel < 4 * R.H, (name, rel)


def test_prompt_then_tokens_equals_the_whole_prompt():
    """Prefill a cache, then decode token by token: the same rows as the packed call over everything."""
    import lbw_amd
    B, prompt, new = 3, [40, 1, 65], 5
    total = [p + new for p in prompt]
    qkv, w, ang, rope, pos, _ = _setup(sum(total), 2)
    plan = lbw_amd.packed_plan(total)
    q, k, v = qkv.split([HQ, HK, HK], 1)
    q2, k2 = lbw_amd.qk_head_norm_rope(q, k, *w, rope, pos)
    whole = lbw_amd.attention_packed(q2, k2, v, plan)
    ref = R.attention(q2, k2, v, total, total, True, 1 / math.sqrt(D))
    at = [sum(total[:b]) for b in range(B)]
    kc = torch.full((B, 80, HK, D), float("nan"), dtype=BF, device="cuda")
    vc = kc.clone()
    for b in range(B):  # the prompt's rows
        s = slice(at[b], at[b] + prompt[b])
        kc[b, :prompt[b]], vc[b, :prompt[b]] = k2[s], v[s]
    lens = torch.tensor(prompt, dtype=torch.int32, device="cuda")
    qo = torch.empty(B, HQ, D, dtype=BF, device="cuda")
    for step in range(new):
        idx = torch.tensor([at[b] + prompt[b] + step for b in range(B)], device="cuda")
        tok, p = qkv[idx], pos[idx]
        tq, tk, tv = tok.split([HQ, HK, HK], 1)
        lbw_amd.qk_head_norm_rope_(tq, tk, *w, rope, p, q_out=qo, k_out=kc, v=tv, v_out=vc, rows=lens)
        lens = lens + 1
        out = lbw_amd.attention_decode(qo, kc, vc, lens)
        R.assert_within("decoded", out, ref["out"][idx], ref["out_a"][idx])
        R.assert_within("packed", whole[idx], ref["out"][idx], ref["out_a"][idx])


def test_continued_prompt_reads_a_cache_view():
    """A prompt continued over cached keys: q shorter than k, K and V as strided views."""
    import lbw_amd
    buf = torch.randn(2, 150, HK + 1, D, device="cuda").to(BF)
    k, v = buf[0, :, :HK], buf[1, :, :HK]
    q = torch.randn(20, HQ, D, device="cuda").to(BF)
    out = lbw_amd.attention_packed(q, k, v, lbw_amd.packed_plan([7, 13], [100, 50]))
    r = R.attention(q, k, v, [7, 13], [100, 50], True, 1 / math.sqrt(D))
    R.assert_within("out", out, r["out"], r["out_a"])


def test_captured_training_step_replays():
    import lbw_amd
    lens = [130, 64]
    qkv, w, _, rope, pos, do = _setup(sum(lens), 3)
    plan = lbw_amd.packed_plan(lens)
    leaves = _leaves(qkv, *w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            _step(*leaves, rope, pos, plan, do)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):  # two graphs of the same call, each with its own workspaces
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = _step(*leaves, rope, pos, plan, do)
        graphs.append((g, got))
    for seed in (4, 5, 6):
        fresh, w2, _, _, pos2, do2 = _setup(sum(lens), seed)
        with torch.no_grad():
            for dst, src in zip((*leaves, pos, do), (fresh, *w2, pos2, do2)):
                dst.copy_(src)
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        want = _step(*_leaves(*leaves), rope, pos, plan, do)
        torch.cuda.synchronize()
        for _, got in graphs:
            for x, y in zip(got, want):
                assert torch.equal(x, y)


def test_capture_with_a_live_eager_graph_of_the_leaves_raises():
    import lbw_amd
    lens = [40]
    qkv, w, _, rope, pos, do = _setup(40, 7)
    plan = lbw_amd.packed_plan(lens)
    q, k, v = _leaves(*[t.contiguous() for t in qkv.split([HQ, HK, HK], 1)])
    alive = lbw_amd.attention_packed(q, k, v, plan)  # an eager graph of the leaves, kept
    g = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="eager graph"):
        with torch.cuda.graph(g):
            out = lbw_amd.attention_packed(q, k, v, plan)
            out.backward(do)
    torch.cuda.synchronize()
    grads = torch.autograd.grad(alive, (q, k, v), do)  # and the eager one still works
    assert all(torch.isfinite(x).all() for x in grads)


def test_captured_decode_follows_device_lengths():
    import lbw_amd
    g0 = torch.Generator().manual_seed(8)
    q = torch.randn(3, HQ, D, generator=g0).to(BF).cuda()
    kc, vc = (torch.randn(3, 2000, HK, D, generator=g0).to(BF).cuda() for _ in range(2))
    lens = torch.tensor([5, 100, 1999], dtype=torch.int32, device="cuda")
    lbw_amd.attention_decode(q, kc, vc, lens)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = lbw_amd.attention_decode(q, kc, vc, lens)
        graphs.append((g, out))
    for new in ([6, 0, 2000], [700, 1, 33], [2000, 2000, 2000]):
        lens.copy_(torch.tensor(new, dtype=torch.int32))
        for g, _ in graphs:
            g.replay()
        want = lbw_amd.attention_decode(q, kc, vc, lens)
        torch.cuda.synchronize()
        for _, out in graphs:
            assert torch.equal(out, want)


def test_other_streams_and_threads_at_once():
    import lbw_amd
    jobs = []
    for i in range(4):
        lens = [50 + 40 * i, 129]
        qkv, w, _, rope, pos, do = _setup(sum(lens), 20 + i)
        plan = lbw_amd.packed_plan(lens)
        jobs.append((qkv, w, rope, pos, plan, do, _step(*_leaves(qkv, *w), rope, pos, plan, do)))
    torch.cuda.synchronize()
    bad = []

    def work(job):
        qkv, w, rope, pos, plan, do, want = job
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for _ in range(5):
                    got = _step(*_leaves(qkv, *w), rope, pos, plan, do)
                    s.synchronize()
                    if not all(torch.equal(x, y) for x, y in zip(got, want)):
                        bad.append("differs")
        except Exception as e:  # noqa: BLE001
            bad.append(repr(e))
    threads = [threading.Thread(target=work, args=(j,)) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad, bad


def test_traces_under_fake_tensors():
    import lbw_amd
    from torch._subclasses.fake_tensor import FakeTensorMode
    plan = lbw_amd.packed_plan([9, 7])
    with FakeTensorMode(allow_non_fake_inputs=True):
        q = torch.empty(16, HQ, D, dtype=BF, device="cuda")
        k = torch.empty(16, HK, D, dtype=BF, device="cuda")
        out, lse = torch.ops.lbw.attention_packed(q, k, k, plan.q_items, plan.k_items, plan.info,
                                                  0.0, True)
        assert out.shape == q.shape and lse.shape == (HQ, 16)
        kc = torch.empty(16, 30, HK, D, dtype=BF, device="cuda")
        lens = torch.empty(16, dtype=torch.int32, device="cuda")
        assert torch.ops.lbw.attention_decode(q, kc, kc, lens).shape == q.shape


@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_compiled_step_gives_the_same_bits(backend):
    """One graph, no break: the training step with its gradients, and a decode step that writes the cache."""
    import lbw_amd
    lens = [70, 1, 33]
    qkv, w, _, rope, pos, do = _setup(sum(lens), 9)
    plan = lbw_amd.packed_plan(lens)

    def forward(qkv, wq, wk):
        q, k, v = qkv.split([HQ, HK, HK], 1)
        q2, k2 = lbw_amd.qk_head_norm_rope(q, k, wq, wk, rope, pos)
        return lbw_amd.attention_packed(q2, k2, v, plan)

    def step(f):
        x = _leaves(qkv, *w)
        out = f(*x)
        return (out,) + torch.autograd.grad(out, x, do)

    def decode(q, k, v, kc, vc, rows):
        lbw_amd.qk_head_norm_rope_(q, k, w[0], w[1], rope, pos[:3], q_out=q, k_out=kc, v=v, v_out=vc, rows=rows)
        return lbw_amd.attention_decode(q, kc, vc, rows + 1)

    def serve(f):
        q, k, v = (t[:3].clone() for t in qkv.split([HQ, HK, HK], 1))
        kc, vc = (torch.full((3, 20, HK, D), x, dtype=BF, device="cuda") for x in (0.5, 2.0))
        rows = torch.tensor([0, 19, 7], dtype=torch.int32, device="cuda")
        return f(q, k, v, kc, vc, rows), q, kc, vc

    torch._dynamo.reset()
    compiled = lambda f: torch.compile(f, backend=backend, fullgraph=True)  # noqa: E731
    for run, f in ((step, forward), (serve, decode)):
        for got, want in zip(run(compiled(f)), run(f)):
            assert torch.equal(got, want)


def test_a_tangent_of_the_outputs_gradient_is_refused():
    """Forward mode over a backward pass: raised, as in the forward calls, not a derivative without it."""
    import lbw_amd
    import torch.autograd.forward_ad as fw
    qkv, w, _, rope, pos, do = _setup(40, 10)
    plan = lbw_amd.packed_plan([40])
    q, k, v = _leaves(*[t.contiguous() for t in qkv.split([HQ, HK, HK], 1)])
    outs = [lbw_amd.attention_packed(q, k, v, plan), lbw_amd.qk_head_norm_rope(q, k, *w, rope, pos)[0]]
    for out in outs:
        want = torch.autograd.grad(out, q, do, retain_graph=True)[0]
        with fw.dual_level():
            with pytest.raises(NotImplementedError):
                torch.autograd.grad(out, q, fw.make_dual(do, torch.ones_like(do)), retain_graph=True)
        assert torch.equal(torch.autograd.grad(out, q, do)[0], want)
