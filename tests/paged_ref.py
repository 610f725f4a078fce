"""Plain 64-bit forms of the operators over a paged cache, with the error each kernel may make, and their inputs.

Allowances as in packed_ref: they count roundings, and nothing in them was fitted to a result. A selection and the
bounds of a page are exact."""
import math

import torch

import packed_ref as R

BF = torch.bfloat16
D = 128


def pages_of(n, page):
    return (n + page - 1) // page


def make_table(lens, page, g, spare=3, width=None, fill=-1):
    """A table whose sequences' pages lie in no order in a pool of `spare` pages more; `fill` behind them."""
    need = [pages_of(n, page) for n in lens]
    total = sum(need) + spare
    order = torch.randperm(total, generator=g).int()
    table = torch.full((len(lens), max(need + [0]) + 1 if width is None else width), fill, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, order[at:].clone(), total


def make_pool(total, page, heads, d, g, head_major=True):
    """k, v [pages, page, heads, d] on the GPU, as two memory layouts of the same shape."""
    shape = (total, heads, page, d) if head_major else (total, page, heads, d)
    kv = [torch.randn(shape, generator=g).to(BF).cuda() for _ in range(2)]
    return [x.transpose(1, 2) if head_major else x for x in kv]


def rows(pool, pages, n):
    """The first n tokens [n, heads, d] of a list of pages."""
    return pool[pages.long()].flatten(0, 1)[:n]


def attention(q, k, v, table, lens, scale, prefix=None, prefix_len=0, selected=None):
    """(out, allowed error) of one query token per sequence, in 64 bits."""
    page, hk = k.shape[1], k.shape[2]
    grp = q.shape[1] // hk
    out, allow = torch.zeros_like(q, dtype=torch.float64), torch.zeros_like(q, dtype=torch.float64)
    pk, pv = (rows(x, prefix, prefix_len) if prefix is not None else x[0, :0] for x in (k, v))
    for b, n in enumerate(lens):
        n = max(0, min(int(n), table.shape[1] * page))
        if selected is None:
            ks, vs = (rows(x, table[b, :pages_of(n, page)], n) for x in (k, v))
            _one(q[b], torch.cat((pk, ks)), torch.cat((pv, vs)), scale, out[b], allow[b])
            continue
        for h in range(hk):
            at = []
            for e in selected[b, h].tolist():
                if e < 0:
                    break
                at += range(min(e * page, n), min((e + 1) * page, n))
            at = torch.tensor(at, dtype=torch.long, device=k.device)
            own = [x[table[b].long()[at // page], at % page, h:h + 1] if len(at) else x[0, :0, h:h + 1]
                   for x in (k, v)]
            mine = slice(h * grp, (h + 1) * grp)
            _one(q[b, mine], torch.cat((pk[:, h:h + 1], own[0])), torch.cat((pv[:, h:h + 1], own[1])), scale,
                 out[b, mine], allow[b, mine])
    return out, allow


def _one(q, k, v, scale, out, allow):
    if len(k):
        r = R.attention(q[None], k, v, [1], [len(k)], False, scale)
        out.copy_(r["out"][0])
        allow.copy_(r["out_a"][0])


def select(q, bounds, table, lens, page, count, first, last):
    """The selection, in 64 bits and on the host."""
    q, bounds, table = q.double().cpu(), bounds.double().cpu(), table.cpu()
    hk = bounds.shape[1]
    grp = q.shape[1] // hk
    sel = torch.full((q.shape[0], hk, count), -1, dtype=torch.int32)
    for b, n in enumerate(lens):
        n = pages_of(max(0, min(int(n), table.shape[1] * page)), page)
        for h in range(hk if n else 0):
            at = table[b, :n].long()
            bad = (at < 0) | (at >= bounds.shape[0])
            e = bounds[at.clamp(0, bounds.shape[0] - 1), h]
            x = q[b, h * grp:(h + 1) * grp]
            s = (x.clamp_min(0)[:, None] * e[:, 1] + x.clamp_max(0)[:, None] * e[:, 0]).sum(-1)
            s = torch.where(s.isnan(), math.inf, s).amax(0)
            s = torch.where(bad, math.inf, s).tolist()
            best = sorted(range(n), key=lambda i: (not (i < first or i >= n - last), -s[i], i))
            best = sorted(best[:count])
            sel[b, h, :len(best)] = torch.tensor(best, dtype=torch.int32)
    return sel


def turned(x, w, ang, inter, eps, scale):
    """Append's q or k in 64 bits: normalised per head when eps is not None."""
    x = x.double()
    if eps is not None:
        return R.head_norm(x, None if w is None else w.double(), ang, inter, eps, scale)
    return R.rotate(x, ang.cos(), ang.sin(), inter) * scale
