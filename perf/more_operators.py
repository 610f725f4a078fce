"""Cases of the operators over a paged key/value cache, for timing and comparing.

Four operators of a serving loop, one new token per sequence unless said otherwise:

- ``paged_append_``: new tokens' q and k rotated by their positions (with RMSNorm per head or
  without), k and v put into their rows of the cache's pages, and the bounds of every page they
  touch -- the smallest and largest value of each key component -- kept up ("append": one token per
  sequence, "prompt": several);
- ``attention_paged``: one query token per sequence over its pages ("paged");
- the same for a batch whose sequences all go on from one prefix, whose keys are read once for all
  of them ("shared");
- ``paged_select`` and ``attention_paged`` over what it selects: the pages whose keys can score
  highest by their bounds, with the first and last pages always among them ("sparse").

Head counts are those of the 1.3B (12 heads x 128) and 14B (40 heads x 128) models, as they are
and with grouped key/value heads; lengths are those of their frames (1560 tokens at 480p, 3600 at
720p), chunks (4680) and windows (14040, 46800), and odd and ragged ones.

With ``own`` false, run() computes the operators from elementary torch operations in 32 bits (the
pages' scores in 64: a selection hangs on their order) on gathered, padded keys; with ``own`` true
it makes the library's calls.
"""
import math
import os
import random
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
        # one decoded token into a cache that also serves sparse attention; nothing but latency
        {"name": "append_1", "kind": "append", "batch": 1, "heads": 40, "kv_heads": 8, "dim": 128,
         "rot": 128, "axes": 1, "inter": False, "norm": False, "page": 64, "capacity": 1024,
         "bounds": True},
        # a batch of 64 sequences, one token each, normalised and turned by video positions
        {"name": "append_64", "kind": "append", "batch": 64, "heads": 40, "kv_heads": 8,
         "dim": 128, "rot": 128, "axes": 3, "inter": True, "norm": True, "page": 16,
         "capacity": 257, "bounds": True},
        # a handful of short prompts that go on inside begun pages, one of them empty
        {"name": "prompt_short", "kind": "prompt", "heads": 12, "kv_heads": 4, "dim": 128,
         "rot": 128, "axes": 1, "inter": False, "norm": True, "page": 16, "bounds": True,
         "new": "17,1,60,0,33", "old": "0,63,5,40,1000"},
        # whole prompts of a chunk's size
        {"name": "prompt_14b", "kind": "prompt", "heads": 40, "kv_heads": 8, "dim": 128,
         "rot": 128, "axes": 3, "inter": True, "norm": True, "page": 64, "bounds": True,
         "new": "4680,3600,1561", "old": "0,4681,77"},
        # one sequence of a few hundred tokens: a step's latency
        {"name": "paged_1", "kind": "paged", "heads": 40, "kv_heads": 8, "page": 64, "batch": 1,
         "own": 500},
        # long windows: eight sequences, up to the 14B 720p window
        {"name": "paged_8_long", "kind": "paged", "heads": 40, "kv_heads": 8, "page": 64,
         "batch": 8, "own": 46800},
        # four continuations of one 480p frame, a few tokens each (1.3B, grouped)
        {"name": "shared_4", "kind": "shared", "heads": 12, "kv_heads": 4, "page": 32, "batch": 4,
         "prefix": 1560, "own": 40},
        # sixteen branches of a 480p history of nine frames, equal heads (1.3B)
        {"name": "shared_16_13b", "kind": "shared", "heads": 12, "kv_heads": 12, "page": 16,
         "batch": 16, "prefix": 14040, "own": 1560},
        # 64 branches of the 14B 720p window, up to a frame each
        {"name": "shared_64_14b", "kind": "shared", "heads": 40, "kv_heads": 8, "page": 64,
         "batch": 64, "prefix": 46800, "own": 3600},
        # short sequences, a quarter of their pages
        {"name": "sparse_4_short", "kind": "sparse", "heads": 12, "kv_heads": 4, "page": 16,
         "batch": 4, "own": 1560, "count": 24, "first": 1, "last": 2},
        # one sequence of the 14B 720p window, 64 of its 732 pages
        {"name": "sparse_1_14b", "kind": "sparse", "heads": 40, "kv_heads": 8, "page": 64,
         "batch": 1, "own": 46800, "count": 64, "first": 1, "last": 8},
        # eight long windows, small pages, an eighth of them
        {"name": "sparse_8_14b", "kind": "sparse", "heads": 40, "kv_heads": 8, "page": 32,
         "batch": 8, "own": 46800, "count": 180, "first": 4, "last": 12},
    ]


def _log(rng, a, b):
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


_HEADS = [(40, 8), (40, 40), (12, 12), (12, 4), (5, 1), (16, 2), (6, 3), (3, 3)]


def _text(lens):
    return ",".join(str(x) for x in lens)


def _lens(text):
    return [int(x) for x in text.split(",")]


def _ragged(c):
    """Lengths of a case's sequences: the first the longest, the others down to a third of it, an
    empty one and one of a single key among the larger batches."""
    rng = random.Random(1000003 * c["batch"] + c["own"])
    lens = [c["own"]] + [rng.randint(c["own"] // 3, c["own"]) for _ in range(c["batch"] - 1)]
    if c["batch"] >= 12:
        lens[-1], lens[-2] = 0, 1
    return lens


def _pages(n, page):
    return (n + page - 1) // page


def draw(rng):
    top = {}
    for c in listed():
        w = work(c)
        for m in ("bytes", "flops"):
            top[m] = max(top.get(m, 0), w[m])
    while True:
        c = _draw(rng)
        w = work(c)
        # (and the plain form's gathered keys, twice in 32 bits: at most about 20 GB)
        keys = c.get("batch", 1) * c.get("own", 1) * c["kv_heads"] * D * 8
        if w["bytes"] <= top["bytes"] and w["flops"] <= top["flops"] and keys <= 20e9:
            return c


def _draw(rng):
    kind = rng.choice(["append", "prompt", "paged", "shared", "shared", "sparse", "sparse"])
    heads, kv = rng.choice(_HEADS)
    c = {"kind": kind, "heads": heads, "kv_heads": kv,
         "page": rng.choice([16, 32, 64, 64, 128, 256])}
    if kind in ("append", "prompt"):
        dim = rng.choice([64, 128, 128, 256])
        c.update(dim=dim, rot=dim if rng.random() < 0.7 else dim // 2, axes=rng.choice([1, 2, 3]),
                 inter=rng.random() < 0.5, norm=rng.random() < 0.5, bounds=rng.random() < 0.7)
        if kind == "append":
            return {**c, "batch": _log(rng, 1, 256), "capacity": _log(rng, 2, 600)}
        n, most = rng.randint(1, 8), _log(rng, 2, 4680)
        new = [most] + [rng.randint(0, most) for _ in range(n - 1)]
        old = [rng.choice([0, rng.randint(0, 2000)]) for _ in range(n)]
        return {**c, "new": _text(new), "old": _text(old)}
    c["batch"] = _log(rng, 1, 64)
    if kind == "paged":
        return {**c, "own": _log(rng, 2, 46800)}
    if kind == "shared":
        return {**c, "prefix": _log(rng, 16, 46800), "own": _log(rng, 2, 3600)}
    most = _log(rng, 100, 46800)
    pages = _pages(most, c["page"])
    count = _log(rng, 4, max(5, pages // 2))
    first = rng.randint(0, 2)
    return {**c, "own": most, "count": count, "first": first,
            "last": rng.randint(0, max(1, count // 4))}


def work(c):
    hq, hk = c["heads"], c["kv_heads"]
    if c["kind"] in ("append", "prompt"):
        d = c["dim"]
        if c["kind"] == "append":
            tokens = runs = c["batch"]
            begun = runs
        else:
            new, old = _lens(c["new"]), _lens(c["old"])
            tokens = sum(new)
            runs = sum(_pages(o + n, c["page"]) - o // c["page"] for n, o in zip(new, old) if n)
            begun = sum(1 for n, o in zip(new, old) if n and o % c["page"])
        edge = 2 * 2 * d * hk * (runs + begun) if c["bounds"] else 0
        return {"bytes": 2 * tokens * d * (2 * hq + 4 * hk) + edge,
                "flops": (8 if c["norm"] else 4) * tokens * d * (hq + hk)}
    lens, b = _ragged(c), c["batch"]
    rows = 2 * D * 2 * hq * b
    if c["kind"] == "paged":
        return {"bytes": 4 * D * hk * sum(lens) + rows, "flops": 4 * D * hq * sum(lens)}
    if c["kind"] == "shared":
        return {"bytes": 4 * D * hk * (c["prefix"] + sum(lens)) + rows,
                "flops": 4 * D * hq * (b * c["prefix"] + sum(lens))}
    pages = [_pages(n, c["page"]) for n in lens]
    keys = sum(min(n, c["count"] * c["page"]) for n in lens)
    return {"bytes": 4 * D * hk * (sum(pages) + keys) + rows + 4 * b * hk * c["count"],
            "flops": 4 * D * hq * (sum(pages) + keys)}


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


def _table(g, dev, pages, width, spare):
    """Page table: the sequences' pages in no order among a pool of some more, -1 behind them."""
    total = sum(pages) + spare
    order = torch.randperm(total, generator=g, device=dev).int()
    table = torch.full((len(pages), max(1, width)), -1, dtype=torch.int32, device=dev)
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = order[at:at + n]
        at += n
    return table, order[at:], total


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)

    def rnd(*shape, gain=1.0):
        return torch.randn(*shape, generator=g, device=dev, dtype=BF16) * gain

    c = case
    hq, hk, page = c["heads"], c["kv_heads"], c["page"]
    s = {"case": c}

    def pool(total, d):
        # a page holds the rows of each key/value head together; [pages, page, heads, d] for the calls
        s["k_pages"] = rnd(total, hk, page, d).transpose(1, 2)
        s["v_pages"] = rnd(total, hk, page, d).transpose(1, 2)

    if c["kind"] in ("append", "prompt"):
        d = c["dim"]
        if c["kind"] == "append":
            t = c["batch"]
            s["lens"] = torch.randint(0, c["capacity"], (t,), generator=g, device=dev,
                                      dtype=torch.int32)
            most = c["capacity"]
            pages = [_pages(most, page)] * t
        else:
            new, old = _lens(c["new"]), _lens(c["old"])
            t, most = sum(new), max(o + n for n, o in zip(new, old))
            s["lens"] = torch.tensor(old, dtype=torch.int32, device=dev)
            s["starts"] = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)],
                                       dtype=torch.int32, device=dev)
            pages = [_pages(o + n, page) for n, o in zip(new, old)]
        s["table"], _, total = _table(g, dev, pages, _pages(most, page), 3)
        pool(total, d)
        if c["bounds"]:
            # of the rows so far, as earlier calls left them (here: of all rows of the pool)
            s["bounds"] = torch.stack((s["k_pages"].amin(1), s["k_pages"].amax(1)), 2)
        rows = max(64, most) if c["axes"] == 1 else 64
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
        s["wq"] = 1 + rnd(d, gain=0.1) if c["norm"] else None
        s["wk"] = 1 + rnd(d, gain=0.1) if c["norm"] else None
        # positions on several axes come with the tokens; on one axis a token's row is its position
        s["pos"] = None if c["axes"] == 1 else torch.randint(0, 64, (t, c["axes"]), generator=g,
                                                             device=dev, dtype=torch.int32)
        s["q_out"] = torch.empty(t, hq, d, dtype=BF16, device=dev)
        if own:
            s["rope"] = _lbw().axis_rope(s["angles"], s["axes"], interleaved=c["inter"])
    else:
        lens, pre = _ragged(c), c.get("prefix", 0)
        pages = [_pages(n, page) for n in lens]
        # (a serving loop's table is as wide as its longest sequence may become: one page more)
        s["table"], spare, total = _table(g, dev, pages, max(pages) + 1, _pages(pre, page) + 3)
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
        pool(total, D)
        if pre:
            s["prefix_table"] = spare[:_pages(pre, page)].contiguous()
            s["prefix_len"] = torch.tensor([pre], dtype=torch.int32, device=dev)
        # heads of different temperature: some of them attend to a few keys, others to all
        heat = 0.5 + 1.5 * torch.rand(hq, 1, generator=g, device=dev)
        s["q"] = (rnd(c["batch"], hq, D).float() * heat).to(BF16)
        if c["kind"] == "sparse":
            # keys of one page are alike, as neighbouring tokens' are
            s["k_pages"] += rnd(total, hk, 1, D, gain=0.7).transpose(1, 2)
            s["bounds"] = _bounds_of(s, lens)
    if own:
        s["cache"] = _lbw().PagedKV(s["k_pages"], s["v_pages"], s.get("bounds"))
    return s


def _bounds_of(s, lens):
    """[pages, kv heads, 2, D]: of every page the smallest and largest value of each key component
    over the rows that hold keys."""
    lo, hi = s["k_pages"].amin(1), s["k_pages"].amax(1)
    page = s["case"]["page"]
    for b, n in enumerate(lens):
        if n % page:
            at = s["table"][b, n // page].long()
            lo[at] = s["k_pages"][at, :n % page].amin(0)
            hi[at] = s["k_pages"][at, :n % page].amax(0)
    return torch.stack((lo, hi), 2)


# ---- the library's calls

def _run_own(s):
    lbw, c = _lbw(), s["case"]
    if c["kind"] in ("append", "prompt"):
        lbw.paged_append_(s["cache"], s["q"], s["k"], s["v"], s["table"], s["lens"], s["rope"],
                          s["pos"], starts=s.get("starts"), q_out=s["q_out"], wq=s["wq"],
                          wk=s["wk"], eps=EPS if c["norm"] else None)
        return _written(s)
    if c["kind"] == "paged":
        return lbw.attention_paged(s["q"], s["cache"], s["table"], s["lens"])
    if c["kind"] == "shared":
        return lbw.attention_paged(s["q"], s["cache"], s["table"], s["lens"],
                                   prefix_table=s["prefix_table"], prefix_len=s["prefix_len"])
    sel = lbw.paged_select(s["q"], s["cache"], s["table"], s["lens"], c["count"],
                           first=c["first"], last=c["last"])
    return sel, lbw.attention_paged(s["q"], s["cache"], s["table"], s["lens"], selected=sel)


def _written(s):
    out = (s["q_out"], s["k_pages"], s["v_pages"])
    return out + (s["bounds"],) if s["case"]["bounds"] else out


# ---- the plain forms

def _turn(x, cos, sin, rot, inter):
    """The first `rot` values of each head turned by their pairs' angles."""
    h = rot // 2
    y = x[..., :rot]
    a, b = (y[..., 0::2], y[..., 1::2]) if inter else (y[..., :h], y[..., h:])
    u, w = a * cos - b * sin, a * sin + b * cos
    y = torch.stack((u, w), -1).flatten(-2) if inter else torch.cat((u, w), -1)
    return torch.cat((y, x[..., rot:]), -1)


def _plain_turned(s, x, w, cos, sin):
    c, x = s["case"], x.float()
    if c["norm"]:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
    return _turn(x, cos, sin, c["rot"], c["inter"]).to(BF16)


def _rows(s):
    """(sequence, row) of every new token."""
    t = torch.arange(s["q"].shape[0], device=s["q"].device)
    if "starts" not in s:
        return t, s["lens"].long()
    b = torch.searchsorted(s["starts"], t.int(), right=True) - 1
    return b, s["lens"].long()[b] + t - s["starts"].long()[b]


def _plain_append(s):
    c, page = s["case"], s["case"]["page"]
    b, row = _rows(s)
    pos = row[:, None] if s["pos"] is None else s["pos"].long()
    at = pos[:, s["axis_of"]]
    cos, sin = s["cos"].gather(0, at)[:, None], s["sin"].gather(0, at)[:, None]
    k2 = _plain_turned(s, s["k"], s["wk"], cos, sin)
    s["q_out"].copy_(_plain_turned(s, s["q"], s["wq"], cos, sin))
    to = s["table"][b, row // page].long()
    s["k_pages"][to, row % page] = k2
    s["v_pages"][to, row % page] = s["v"]
    if c["bounds"]:
        # a page whose first row is written starts anew
        x, lo, hi = k2.float(), s["bounds"][:, :, 0].float(), s["bounds"][:, :, 1].float()
        new = torch.zeros(len(lo), device=x.device).index_add_(0, to, (row % page == 0).float())
        lo.masked_fill_(new[:, None, None] > 0, math.inf)
        hi.masked_fill_(new[:, None, None] > 0, -math.inf)
        lo.index_reduce_(0, to, x, "amin")
        hi.index_reduce_(0, to, x, "amax")
        s["bounds"].copy_(torch.stack((lo, hi), 2))
    return _written(s)


def _attend(q, k, v, seen):
    """q [n, rows, D], k, v [n, keys, D] in 32 bits, seen [n, 1 or rows, keys]."""
    p = torch.bmm(q, k.transpose(1, 2).contiguous()).mul_(1.0 / math.sqrt(D))
    p.masked_fill_(~seen, -math.inf)
    m = p.amax(-1, keepdim=True)
    p.sub_(torch.where(m == -math.inf, 0.0, m)).exp_()
    p.div_(p.sum(-1, keepdim=True).clamp_min_(1e-37))
    return torch.bmm(p, v)


def _gathered(s, pages):
    """k, v of a table's pages [n, width]: [n, kv heads, keys, D] in 32 bits."""
    at = pages.clamp_min(0).long()
    return [s[x][at].permute(0, 3, 1, 2, 4).flatten(2, 3).float() for x in ("k_pages", "v_pages")]


def _plain_dense(s):
    c = s["case"]
    n, hk = c["batch"], c["kv_heads"]
    q = s["q"].float().view(n, hk, -1, D)
    grp = q.shape[2]
    k, v = _gathered(s, s["table"])
    seen = torch.arange(k.shape[2], device=q.device) < s["lens"][:, None]
    if c["kind"] == "paged":
        out = _attend(q.reshape(n * hk, grp, D), k.flatten(0, 1), v.flatten(0, 1),
                      seen[:, None].expand(-1, hk, -1).reshape(n * hk, 1, -1))
        return out.view(n, c["heads"], D).to(BF16)
    # the prefix's scores for all sequences' rows at once, then each sequence's own keys
    pk, pv = (x[0] for x in _gathered(s, s["prefix_table"][None]))
    rows = q.transpose(0, 1).reshape(hk, n * grp, D)
    scale = 1.0 / math.sqrt(D)
    p = torch.bmm(rows, pk.transpose(1, 2).contiguous()).mul_(scale)
    p.masked_fill_(torch.arange(pk.shape[1], device=q.device) >= s["prefix_len"], -math.inf)
    p = p.view(hk, n, grp, -1).transpose(0, 1)
    o = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(scale)
    o.masked_fill_(~seen[:, None, None], -math.inf)
    m = torch.maximum(p.amax(-1, keepdim=True), o.amax(-1, keepdim=True))
    m = torch.where(m == -math.inf, 0.0, m)
    p, o = (p - m).exp_(), (o - m).exp_()
    total = (p.sum(-1, keepdim=True) + o.sum(-1, keepdim=True)).clamp_min_(1e-37)
    out = torch.bmm(p.transpose(0, 1).reshape(hk, n * grp, -1), pv)
    out = out.view(hk, n, grp, D).transpose(0, 1) + torch.matmul(o, v)
    return (out / total).reshape(n, c["heads"], D).to(BF16)


def _plain_select(s):
    c = s["case"]
    n, hk, page = c["batch"], c["kv_heads"], c["page"]
    q = s["q"].double().view(n, hk, -1, D)
    edge = s["bounds"][s["table"].clamp_min(0).long()].permute(0, 2, 3, 4, 1).double().contiguous()
    x = torch.matmul(q.clamp_min(0.0), edge[:, :, 1]) + torch.matmul(q.clamp_max(0.0), edge[:, :, 0])
    x = x.amax(2)
    x.masked_fill_(x.isnan(), math.inf)
    pages = ((s["lens"] + page - 1) // page)[:, None, None]
    i = torch.arange(x.shape[2], device=x.device)
    there = i < pages
    kept = there & ((i < c["first"]) | (i >= pages - c["last"]))
    # kept pages, then by score, the lower page first among equals; pages that are not there last
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices
    rank = (~kept).int() + 2 * (~there).int()
    rank = rank.expand_as(x).gather(2, order)
    order = order.gather(2, torch.sort(rank, dim=-1, stable=True).indices)[..., :c["count"]]
    count = order.shape[-1]
    order = torch.where(torch.arange(count, device=x.device) < pages, order, x.shape[2])
    order = torch.sort(order, -1).values
    sel = torch.full((n, hk, c["count"]), -1, dtype=torch.int32, device=x.device)
    sel[..., :count] = torch.where(order < x.shape[2], order, -1)
    return sel


def _plain_sparse(s):
    c = s["case"]
    n, hk, page = c["batch"], c["kv_heads"], c["page"]
    sel = _plain_select(s)
    at = s["table"][torch.arange(n, device=sel.device)[:, None, None], sel.clamp_min(0).long()]
    at, head = at.clamp_min(0).long(), torch.arange(hk, device=sel.device)[:, None]
    k, v = (s[x].transpose(1, 2)[at, head].float().view(n * hk, -1, D) for x in ("k_pages", "v_pages"))
    row = sel[..., None] * page + torch.arange(page, device=sel.device)
    seen = (sel[..., None] >= 0) & (row < s["lens"][:, None, None, None])
    out = _attend(s["q"].float().view(n * hk, -1, D), k, v, seen.view(n * hk, 1, -1))
    return sel, out.view(n, c["heads"], D).to(BF16)


def run(s):
    if own:
        return _run_own(s)
    kind = s["case"]["kind"]
    if kind in ("append", "prompt"):
        return _plain_append(s)
    return _plain_sparse(s) if kind == "sparse" else _plain_dense(s)


# ---- the definitions in 64 bits

def _exact_turned(c, x, w, angle):
    """One tensor [tokens, heads, dim]: the rotation as a complex product of its pairs."""
    h = c["rot"] // 2
    first = torch.arange(h, device=x.device) * (2 if c["inter"] else 1)
    second = first + (1 if c["inter"] else h)
    y = x.double()
    if c["norm"]:
        y = y / (y.square().sum(-1, keepdim=True) / y.shape[-1] + EPS).sqrt() * w.double()
    z = torch.complex(y[..., first], y[..., second])
    z = z * torch.polar(torch.ones_like(angle), angle)[:, None]
    y = y.clone()
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_append(s):
    c, page = s["case"], s["case"]["page"]
    old = s["lens"].tolist()
    starts = s["starts"].tolist() if "starts" in s else list(range(len(old) + 1))
    rows = [o + i for b, o in enumerate(old) for i in range(starts[b + 1] - starts[b])]
    pos = s["pos"].long() if s["pos"] is not None else torch.tensor(rows, device=s["q"].device)[:, None]
    angle = torch.stack([s["angles"].double()[pos[:, a], i]
                         for i, a in enumerate(s["axis_of"].tolist())], 1)
    k2 = _exact_turned(c, s["k"], s["wk"], angle)
    k, v = s["k_pages"].double(), s["v_pages"].double()
    edge = s["bounds"].double() if c["bounds"] else None
    table = s["table"].tolist()
    for b, o in enumerate(old):
        t, end = starts[b], starts[b + 1]
        while t < end:  # the tokens of one page at a time
            row = o + t - starts[b]
            at, n = table[b][row // page], min(page - row % page, end - t)
            here = slice(row % page, row % page + n)
            k[at, here], v[at, here] = k2[t:t + n], s["v"][t:t + n].double()
            if edge is not None:
                lo, hi = k2[t:t + n].amin(0), k2[t:t + n].amax(0)
                if row % page:
                    lo, hi = torch.minimum(lo, edge[at, :, 0]), torch.maximum(hi, edge[at, :, 1])
                edge[at, :, 0], edge[at, :, 1] = lo, hi
            t += n
    out = (_exact_turned(c, s["q"], s["wq"], angle), k, v)
    return out if edge is None else out + (edge,)


def _keys(s, pages, n, h):
    """The first n keys and values of key/value head h in the given pages, in 64 bits."""
    at = torch.tensor(pages, dtype=torch.long, device=s["q"].device)
    return [s[x][at, :, h].reshape(-1, D)[:n].double() for x in ("k_pages", "v_pages")]


def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["kind"] in ("append", "prompt"):
        return _exact_append(s)
    hq, hk, page = c["heads"], c["kv_heads"], c["page"]
    grp = hq // hk
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    sel = torch.full((c["batch"], hk, c.get("count", 0)), -1, dtype=torch.int32, device=out.device)
    table = s["table"].tolist()
    pre = {}
    for b, n in enumerate(_ragged(c)):
        pages = table[b][:_pages(n, page)]
        for h in range(hk):
            mine = slice(h * grp, (h + 1) * grp)
            q = s["q"][b, mine].double()
            if c["kind"] == "sparse":
                if not n:
                    continue
                lo, hi = s["bounds"][torch.tensor(pages, device=out.device), h].double().unbind(1)
                score = torch.maximum(q[:, None] * lo, q[:, None] * hi).sum(-1).amax(0).tolist()
                always = [i < c["first"] or i >= len(pages) - c["last"] for i in range(len(pages))]
                best = sorted(range(len(pages)), key=lambda i: (not always[i], -score[i], i))
                best = sorted(best[:c["count"]])
                sel[b, h, :len(best)] = torch.tensor(best, dtype=torch.int32)
                short = page * len(pages) - n if best[-1] == len(pages) - 1 else 0
                k, v = _keys(s, [pages[i] for i in best], page * len(best) - short, h)
            else:
                k, v = _keys(s, pages, n, h)
                if c["kind"] == "shared":
                    if h not in pre:
                        pre[h] = _keys(s, s["prefix_table"].tolist(), c["prefix"], h)
                    k, v = torch.cat((pre[h][0], k)), torch.cat((pre[h][1], v))
            if len(k):
                out[b, mine] = torch.softmax(q @ k.T / D ** 0.5, -1) @ v
    return (sel, out) if c["kind"] == "sparse" else out
