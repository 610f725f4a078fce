"""Cases of the operators for training and serving on packed sequences, for timing and comparing.

Three operators and their gradients:

- ``qk_head_norm_rope``: RMSNorm of every query and key head and the rotation of its pairs by the
  token's position on one or several axes, in one pass; with its gradient (kind "norm_train"), and
  in the form that writes a decoded token's K and V into its cache row (kind "append");
- ``attention_packed``: attention over sequences packed one after another, causal or full, grouped
  heads, keys longer than the queries where a prompt continues; with its gradient ("packed_train");
- ``attention_decode``: one query token per sequence over its cache ("decode").

Head counts are those of the 1.3B (12 heads x 128) and 14B (40 heads x 128) models, as they are
and with grouped key/value heads; lengths are those of their frames (1560 tokens at 480p, 3600 at
720p), chunks (4680) and windows (46800), of the text context (512), and odd and ragged ones.

With ``own`` false, run() computes the operators from elementary torch operations in 32 bits on
padded batches; with ``own`` true it makes the library's calls.
"""
import math
import os
import sys

import torch

own = False

D = 128
EPS = 1e-6
BF16 = torch.bfloat16


def _lbw():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                       "lingbot-world-v2_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import lbw_amd
    return lbw_amd


def listed():
    return [
        # one decoded token: its q and k normalised and rotated, its K and V committed to the
        # cache; nothing but latency
        {"name": "append_1", "kind": "append", "batch": 1, "heads": 40, "kv_heads": 8, "dim": 128,
         "rot": 128, "axes": 1, "inter": False, "capacity": 1024},
        # a batch of 64 sequences, one token each
        {"name": "append_64", "kind": "append", "batch": 64, "heads": 40, "kv_heads": 8,
         "dim": 128, "rot": 128, "axes": 3, "inter": True, "capacity": 257},
        # a chunk of three 480p frames of the 14B model, video positions (time, height, width)
        {"name": "norm_train_14b_480p", "kind": "norm_train", "tokens": 4680, "heads": 40,
         "kv_heads": 8, "dim": 128, "rot": 128, "axes": 3, "inter": True},
        # a training batch of the 1.3B model, ragged token count, equal heads
        {"name": "norm_train_13b_32759", "kind": "norm_train", "tokens": 32759, "heads": 12,
         "kv_heads": 12, "dim": 128, "rot": 128, "axes": 3, "inter": True},
        # a handful of short prompts, one of them empty and one a single token
        {"name": "packed_short", "kind": "packed", "heads": 12, "kv_heads": 4, "causal": True,
         "q_lens": "17,1,60,0,33", "k_lens": "17,1,60,0,33"},
        # prompts that continue: 256 new tokens over caches of several lengths
        {"name": "packed_continued", "kind": "packed", "heads": 40, "kv_heads": 8, "causal": True,
         "q_lens": "256,256,256", "k_lens": "4680,1816,3111"},
        # whole prompts of a chunk's size, causal, grouped heads
        {"name": "packed_14b_prompts", "kind": "packed", "heads": 40, "kv_heads": 8,
         "causal": True, "q_lens": "4680,3600,1561", "k_lens": "4680,3600,1561"},
        # a training step on short clips
        {"name": "packed_train_short", "kind": "packed_train", "heads": 12, "kv_heads": 4,
         "causal": True, "q_lens": "311,97,512,5", "k_lens": "311,97,512,5"},
        # a training step on whole chunks, causal, grouped heads
        {"name": "packed_train_14b", "kind": "packed_train", "heads": 40, "kv_heads": 8,
         "causal": True, "q_lens": "4680,3599,2340", "k_lens": "4680,3599,2340"},
        # a training step with full attention over single 480p frames, equal heads (1.3B)
        {"name": "packed_train_full_13b", "kind": "packed_train", "heads": 12, "kv_heads": 12,
         "causal": False, "q_lens": "1560,1560,1560,1203", "k_lens": "1560,1560,1560,1203"},
        # one sequence of a few hundred tokens: a decode step's latency
        {"name": "decode_1", "kind": "decode", "heads": 40, "kv_heads": 8, "capacity": 1024,
         "lens": "500"},
        # long windows: eight sequences, one as long as the 14B 720p window
        {"name": "decode_8_long", "kind": "decode", "heads": 40, "kv_heads": 8,
         "capacity": 46800, "lens": "46800,39601,21777,46799,10921,30420,15600,28081"},
    ]


def _log(rng, a, b):
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


_HEADS = [(40, 8), (40, 40), (12, 12), (12, 4), (5, 1), (16, 2), (6, 3), (3, 3)]


def _text(lens):
    return ",".join(str(x) for x in lens)


def _lens(text):
    return [int(x) for x in text.split(",")]


def draw(rng):
    top = {}
    for c in listed():
        w = work(c)
        for m in ("bytes", "flops"):
            top[m] = max(top.get(m, 0), w[m])
    while True:
        c = _draw(rng)
        w = work(c)
        if w["bytes"] <= top["bytes"] and w["flops"] <= top["flops"]:
            return c


def _draw(rng):
    kind = rng.choice(["append", "norm_train", "packed", "packed", "packed_train", "packed_train",
                       "decode", "decode"])
    heads, kv = rng.choice(_HEADS)
    if kind in ("append", "norm_train"):
        dim = rng.choice([64, 128, 128, 256])
        axes = rng.choice([1, 2, 3, 3])
        rot = dim if rng.random() < 0.7 else dim // 2
        c = {"kind": kind, "heads": heads, "kv_heads": kv, "dim": dim, "rot": rot, "axes": axes,
             "inter": rng.random() < 0.5}
        if kind == "append":
            return {**c, "batch": _log(rng, 1, 256), "capacity": _log(rng, 2, 600)}
        return {**c, "tokens": _log(rng, 33, 32760)}
    if kind == "decode":
        n = _log(rng, 1, 48)
        cap = _log(rng, 40, 46800)
        lens = [cap if rng.random() < 0.2 else rng.randint(max(0, cap // 3), cap)
                for _ in range(n)]
        if n > 2 and rng.random() < 0.5:
            lens[rng.randrange(n)] = rng.choice([0, 1])
        return {"kind": kind, "heads": heads, "kv_heads": kv, "capacity": cap,
                "lens": _text(lens)}
    while True:
        n = rng.randint(1, 8)
        most = _log(rng, 16, 4680)
        ql = [most if i == 0 else rng.randint(max(1, most // 3), most) for i in range(n)]
        if n > 2 and rng.random() < 0.4:
            ql[rng.randrange(1, n)] = rng.choice([0, 1])
        more = rng.random() < 0.4 and kind == "packed"
        kl = [x + rng.randint(0, 2000) if more else x for x in ql]
        # (the padded plain form's scores: at most about 10 GB in 32 bits)
        if n * heads * max(ql) * max(kl) <= 2.7e9:
            return {"kind": kind, "heads": heads, "kv_heads": kv, "causal": rng.random() < 0.75,
                    "q_lens": _text(ql), "k_lens": _text(kl)}


def _pairs(c):
    """(query, key) pairs that are not masked, per query head."""
    n = 0
    for lq, lk in zip(_lens(c["q_lens"]), _lens(c["k_lens"])):
        if not c["causal"]:
            n += lq * lk
        else:
            # row i sees keys 0 .. i + lk - lq
            first = max(0, lq - lk)  # rows before it see none
            rows = lq - first
            n += rows * (lk + (first + lk - lq + 1)) // 2 if rows > 0 else 0
    return n


def work(c):
    hq, hk = c["heads"], c["kv_heads"]
    if c["kind"] == "append":
        n = c["batch"] * c["dim"]
        return {"bytes": 2 * n * (2 * hq + 4 * hk), "flops": 8 * n * (hq + hk)}
    if c["kind"] == "norm_train":
        # forward: q, k in, q', k' out; backward: the gradients and q, k in, dq, dk out
        n = c["tokens"] * c["dim"] * (hq + hk)
        return {"bytes": 2 * 5 * n + 4 * c["axes"] * c["tokens"], "flops": 24 * n}
    if c["kind"] == "decode":
        keys, b = sum(_lens(c["lens"])), len(_lens(c["lens"]))
        return {"bytes": 2 * D * (2 * hk * keys + 2 * hq * b), "flops": 4 * D * hq * keys}
    tq, tk = sum(_lens(c["q_lens"])), sum(_lens(c["k_lens"]))
    fwd, flops = 2 * D * (2 * hq * tq + 2 * hk * tk), 4 * D * hq * _pairs(c)
    if c["kind"] == "packed":
        return {"bytes": fwd, "flops": flops}
    # the step's inputs (q, k, v, dout) and outputs (out, dq, dk, dv)
    return {"bytes": fwd + 2 * D * (2 * hq * tq + 2 * hk * tk), "flops": flops * 7 // 2}


# ---- inputs

def _axes_split(pairs, axes):
    """Pairs per axis: the time axis takes what the others leave, as the video models split."""
    if axes == 1:
        return [pairs]
    if axes == 2:
        return [pairs - pairs // 2, pairs // 2]
    return [pairs - 2 * (pairs // 3), pairs // 3, pairs // 3]


def _angles(c, rows, device):
    """[rows, rot / 2]: the angle of every pair at every position of its axis, in 32 bits."""
    cols = []
    for n in _axes_split(c["rot"] // 2, c["axes"]):
        freq = 10000.0 ** (-torch.arange(n, dtype=torch.float64, device=device) / max(1, n))
        cols.append(torch.outer(torch.arange(rows, dtype=torch.float64, device=device), freq))
    return torch.cat(cols, 1).float()


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)

    def rnd(*shape, dtype=BF16, gain=1.0):
        return (torch.randn(*shape, generator=g, device=dev) * gain).to(dtype)

    c = case
    hq, hk = c["heads"], c["kv_heads"]
    s = {"case": c}
    if c["kind"] in ("append", "norm_train"):
        d = c["dim"]
        t = c["batch"] if c["kind"] == "append" else c["tokens"]
        rows = max(64, c.get("capacity", 0)) if c["axes"] == 1 else 64
        if c["kind"] == "norm_train" and c["axes"] == 1:
            rows = t
        s["angles"] = _angles(c, rows, dev)
        s["cos"] = s["angles"].double().cos().float()
        s["sin"] = s["angles"].double().sin().float()
        s["axes"] = _axes_split(c["rot"] // 2, c["axes"])
        # the axis whose position turns a pair
        s["axis_of"] = torch.repeat_interleave(torch.arange(c["axes"], device=dev),
                                               torch.tensor(s["axes"], device=dev))
        # the fused projection's output: q, k and v as its column blocks
        qkv = rnd(t, (hq + 2 * hk) * d, gain=1.7)
        s["q"] = qkv[:, :hq * d].unflatten(1, (hq, d))
        s["k"] = qkv[:, hq * d:(hq + hk) * d].unflatten(1, (hk, d))
        s["v"] = qkv[:, (hq + hk) * d:].unflatten(1, (hk, d))
        s["wq"] = 1 + rnd(d, gain=0.1)
        s["wk"] = 1 + rnd(d, gain=0.1)
        if c["kind"] == "append":
            # the sequences' lengths so far; the token goes to that row of its cache
            s["lens"] = torch.randint(0, c["capacity"], (t,), generator=g, device=dev,
                                      dtype=torch.int32)
            pos = torch.randint(0, 64, (t, c["axes"]), generator=g, device=dev, dtype=torch.int32)
            s["pos"] = s["lens"][:, None].clone() if c["axes"] == 1 else pos
            s["k_cache"] = rnd(t, c["capacity"], hk, d)
            s["v_cache"] = rnd(t, c["capacity"], hk, d)
            s["q_out"] = torch.empty(t, hq, d, dtype=BF16, device=dev)
        else:
            if c["axes"] == 1:
                s["pos"] = torch.arange(t, device=dev, dtype=torch.int32)[:, None]
            else:
                s["pos"] = torch.randint(0, 64, (t, c["axes"]), generator=g, device=dev,
                                         dtype=torch.int32)
            s["dq"], s["dk"] = rnd(t, hq, d), rnd(t, hk, d)
            for name in ("q", "k", "wq", "wk"):
                s[name] = s[name].detach().requires_grad_(own)
        if own:
            s["rope"] = _lbw().axis_rope(s["angles"], s["axes"], interleaved=c["inter"])
        return s
    # heads of different temperature: some of them attend to a few keys, others to all
    heat = 0.5 + 1.5 * torch.rand(hq, 1, generator=g, device=dev)
    if c["kind"] == "decode":
        lens = _lens(c["lens"])
        s["q"] = (rnd(len(lens), hq, D).float() * heat).to(BF16)
        s["k_cache"] = rnd(len(lens), c["capacity"], hk, D)
        s["v_cache"] = rnd(len(lens), c["capacity"], hk, D)
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
        return s
    ql, kl = _lens(c["q_lens"]), _lens(c["k_lens"])
    s["q"] = (rnd(sum(ql), hq, D).float() * heat).to(BF16)
    s["k"], s["v"] = rnd(sum(kl), hk, D), rnd(sum(kl), hk, D)
    s["q_lens"] = torch.tensor(ql, device=dev)
    s["k_lens"] = torch.tensor(kl, device=dev)
    s["most_q"], s["most_k"] = max(ql), max(kl)
    if c["kind"] == "packed_train":
        s["dout"] = rnd(sum(ql), hq, D)
        for name in ("q", "k", "v"):
            s[name].requires_grad_(own)
    if own:
        # made once for a batch's lengths, used by every layer's call
        s["plan"] = _lbw().packed_plan(ql, kl, causal=c["causal"], device=dev)
    return s


# ---- the library's calls

def _run_own(s):
    lbw, c = _lbw(), s["case"]
    if c["kind"] == "append":
        lbw.qk_head_norm_rope_(s["q"], s["k"], s["wq"], s["wk"], s["rope"], s["pos"], EPS,
                               q_out=s["q_out"], k_out=s["k_cache"], v=s["v"], v_out=s["v_cache"],
                               rows=s["lens"])
        return s["q_out"], s["k_cache"], s["v_cache"]
    if c["kind"] == "norm_train":
        q2, k2 = lbw.qk_head_norm_rope(s["q"], s["k"], s["wq"], s["wk"], s["rope"], s["pos"], EPS)
        grads = torch.autograd.grad((q2, k2), (s["q"], s["k"], s["wq"], s["wk"]),
                                    (s["dq"], s["dk"]))
        return (q2, k2) + grads
    if c["kind"] == "decode":
        return lbw.attention_decode(s["q"], s["k_cache"], s["v_cache"], s["lens"])
    out = lbw.attention_packed(s["q"], s["k"], s["v"], s["plan"])
    if c["kind"] == "packed":
        return out
    return (out,) + torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["dout"])


# ---- the plain forms

def _turn(x, cos, sin, rot, inter, back=False):
    """The first `rot` values of each head turned by their pairs' angles (back: the other way)."""
    h = rot // 2
    y = x[..., :rot]
    a, b = (y[..., 0::2], y[..., 1::2]) if inter else (y[..., :h], y[..., h:])
    sin = -sin if back else sin
    u, w = a * cos - b * sin, a * sin + b * cos
    y = torch.stack((u, w), -1).flatten(-2) if inter else torch.cat((u, w), -1)
    return torch.cat((y, x[..., rot:]), -1)


def _plain_norm(s, x, w, cos, sin):
    c = s["case"]
    x, w = x.float(), w.float()
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    return _turn(x * r * w, cos, sin, c["rot"], c["inter"])


def _plain_norm_grad(s, x, w, dy, cos, sin):
    c = s["case"]
    x, w, dy = x.float(), w.float(), dy.float()
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    g = _turn(dy, cos, sin, c["rot"], c["inter"], back=True)
    xn = x * r
    dw = (g * xn).sum((0, 1))
    g = g * w
    return (r * (g - xn * (g * xn).mean(-1, keepdim=True))).to(BF16), dw.to(BF16)


def _padded(x, lens, most):
    """[tokens, heads, D] -> [sequences, heads, most, D] in 32 bits, zeros past each length."""
    at = torch.arange(most, device=x.device)
    there = at < lens[:, None]
    idx = (torch.cumsum(lens, 0) - lens)[:, None] + at
    y = x.float()[torch.where(there, idx, 0)] * there[:, :, None, None]
    return y.transpose(1, 2).contiguous()


def _packed(y, lens):
    """The inverse of _padded, rounded to bf16."""
    most = y.shape[2]
    there = torch.arange(most, device=y.device) < lens[:, None]
    return y.transpose(1, 2)[there].to(BF16)


def _plain_attention(s):
    c = s["case"]
    hq, hk = c["heads"], c["kv_heads"]
    grp, lq, lk = hq // hk, s["most_q"], s["most_k"]
    n = len(s["q_lens"])
    # a group's query heads stand one after another, as rows of one product
    q = _padded(s["q"], s["q_lens"], lq).view(n * hk, grp * lq, D)
    k = _padded(s["k"], s["k_lens"], lk).view(n * hk, lk, D)
    v = _padded(s["v"], s["k_lens"], lk).view(n * hk, lk, D)
    scale = 1.0 / math.sqrt(D)
    p = torch.bmm(q, k.transpose(1, 2)).mul_(scale).view(n, hk, grp, lq, lk)
    i = torch.arange(lq, device=q.device)[:, None]
    j = torch.arange(lk, device=q.device)[None, :]
    ql, kl = s["q_lens"][:, None, None], s["k_lens"][:, None, None]
    seen = (j < kl) & (i < ql)
    if c["causal"]:
        seen = seen & (j <= i + kl - ql)
    p.masked_fill_(~seen[:, None, None], -math.inf)
    m = p.amax(-1, keepdim=True) if lk else p.sum(-1, keepdim=True)
    p.sub_(torch.where(m == -math.inf, 0.0, m)).exp_()
    p.div_(p.sum(-1, keepdim=True).clamp_min_(1e-37))
    p = p.view(n * hk, grp * lq, lk)
    out = _packed(torch.bmm(p, v).view(n, hq, lq, D), s["q_lens"])
    if c["kind"] == "packed":
        return out
    do = _padded(s["dout"], s["q_lens"], lq).view(n * hk, grp * lq, D)
    dv = torch.bmm(p.transpose(1, 2), do)
    ds = torch.bmm(do, v.transpose(1, 2))
    ds.sub_((ds * p).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq, dk = torch.bmm(ds, k), torch.bmm(ds.transpose(1, 2), q)
    return (out, _packed(dq.view(n, hq, lq, D), s["q_lens"]),
            _packed(dk.view(n, hk, lk, D), s["k_lens"]),
            _packed(dv.view(n, hk, lk, D), s["k_lens"]))


def _plain_decode(s):
    c = s["case"]
    n, hk = s["q"].shape[0], c["kv_heads"]
    q = s["q"].float().view(n, hk, -1, D)
    k = s["k_cache"].float().permute(0, 2, 3, 1)
    v = s["v_cache"].float().transpose(1, 2)
    p = torch.matmul(q, k).mul_(1.0 / math.sqrt(D))
    seen = torch.arange(c["capacity"], device=q.device) < s["lens"][:, None]
    p.masked_fill_(~seen[:, None, None], -math.inf)
    m = p.amax(-1, keepdim=True)
    p.sub_(torch.where(m == -math.inf, 0.0, m)).exp_()
    p.div_(p.sum(-1, keepdim=True).clamp_min_(1e-37))
    return torch.matmul(p, v).view(n, c["heads"], D).to(BF16)


def run(s):
    if own:
        return _run_own(s)
    c = s["case"]
    if c["kind"] == "decode":
        return _plain_decode(s)
    if c["kind"] in ("packed", "packed_train"):
        return _plain_attention(s)
    rows = s["pos"].long()[:, s["axis_of"]]
    cos, sin = s["cos"].gather(0, rows)[:, None], s["sin"].gather(0, rows)[:, None]
    q2 = _plain_norm(s, s["q"], s["wq"], cos, sin).to(BF16)
    k2 = _plain_norm(s, s["k"], s["wk"], cos, sin).to(BF16)
    if c["kind"] == "append":
        b = torch.arange(len(rows), device=rows.device)
        s["k_cache"][b, s["lens"].long()] = k2
        s["v_cache"][b, s["lens"].long()] = s["v"]
        s["q_out"].copy_(q2)
        return s["q_out"], s["k_cache"], s["v_cache"]
    dq, dwq = _plain_norm_grad(s, s["q"], s["wq"], s["dq"], cos, sin)
    dk, dwk = _plain_norm_grad(s, s["k"], s["wk"], s["dk"], cos, sin)
    return q2, k2, dq, dk, dwq, dwk


# ---- the definitions in 64 bits

def _exact_norm(c, x, w, angle, dy=None):
    """One tensor [tokens, heads, dim]: the rotation as a complex product of its pairs."""
    rot, h = c["rot"], c["rot"] // 2
    first = torch.arange(h, device=x.device) * (2 if c["inter"] else 1)
    second = first + (1 if c["inter"] else h)
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]
    x, w = x.detach().double(), w.detach().double()
    rms = (x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt()
    unit = x / rms
    y = unit * w
    z = torch.complex(y[..., first], y[..., second]) * turn
    out = y.clone()
    out[..., first], out[..., second] = z.real, z.imag
    if dy is None:
        return out
    g = dy.double()
    z = torch.complex(g[..., first], g[..., second]) * turn.conj()
    g = g.clone()
    g[..., first], g[..., second] = z.real, z.imag
    dw = (g * unit).sum((0, 1))
    g = g * w
    dx = g / rms - unit * (g * unit).sum(-1, keepdim=True) / (x.shape[-1] * rms)
    return out, dx, dw


def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["kind"] in ("append", "norm_train"):
        at = s["pos"].long()
        angle = torch.stack([s["angles"].double()[at[:, a], i]
                             for i, a in enumerate(s["axis_of"].tolist())], 1)
        if c["kind"] == "append":
            k, v = s["k_cache"].double(), s["v_cache"].double()
            k2 = _exact_norm(c, s["k"], s["wk"], angle)
            for b, row in enumerate(s["lens"].tolist()):
                k[b, row], v[b, row] = k2[b], s["v"][b].double()
            return _exact_norm(c, s["q"], s["wq"], angle), k, v
        q2, dq, dwq = _exact_norm(c, s["q"], s["wq"], angle, s["dq"])
        k2, dk, dwk = _exact_norm(c, s["k"], s["wk"], angle, s["dk"])
        return q2, k2, dq, dk, dwq, dwk
    hq, hk = c["heads"], c["kv_heads"]
    if c["kind"] == "decode":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
        for b, n in enumerate(s["lens"].tolist()):
            for h in range(hk if n else 0):
                mine = slice(h * (hq // hk), (h + 1) * (hq // hk))
                x = s["q"][b, mine].double() @ s["k_cache"][b, :n, h].double().T / D ** 0.5
                out[b, mine] = torch.softmax(x, -1) @ s["v_cache"][b, :n, h].double()
        return out
    train = c["kind"] == "packed_train"
    q, k, v = (s[x].detach().double() for x in ("q", "k", "v"))
    out, dq = torch.zeros_like(q), torch.zeros_like(q)
    dk, dv = torch.zeros_like(k), torch.zeros_like(v)
    q0 = k0 = 0
    for lq, lk in zip(_lens(c["q_lens"]), _lens(c["k_lens"])):
        rows, keys = slice(q0, q0 + lq), slice(k0, k0 + lk)
        q0, k0 = q0 + lq, k0 + lk
        if not lq or not lk:
            continue
        hide = torch.ones(lq, lk, dtype=torch.bool, device=q.device).triu(lk - lq + 1)
        for h in range(hq):
            kk, vv = k[keys, h // (hq // hk)], v[keys, h // (hq // hk)]
            x = q[rows, h] @ kk.T / D ** 0.5
            if c["causal"]:
                x = x.masked_fill(hide, -math.inf)
            p = torch.softmax(x, -1).nan_to_num(0.0)  # (a row that sees no key)
            out[rows, h] = p @ vv
            if train:
                do = s["dout"][rows, h].double()
                dv[keys, h // (hq // hk)] += p.T @ do
                dp = do @ vv.T
                ds = p * (dp - (do * out[rows, h]).sum(-1, keepdim=True)) / D ** 0.5
                dq[rows, h] = ds @ kk
                dk[keys, h // (hq // hk)] += ds.T @ q[rows, h]
    return (out, dq, dk, dv) if train else out
