"""Plain 64-bit forms of the operators on packed sequences, with the error each kernel may make.

The allowances count roundings. A rounding to bf16 is off by at most half a step, H = eps(bf16) / 2 =
2^-8 of the value; fp32 arithmetic by 2^-24 per operation. They are sums of absolute values, so they
hold for every input, and nothing in them was fitted to a result.
"""
import math

import torch

H = torch.finfo(torch.bfloat16).eps / 2
E = torch.finfo(torch.float32).eps / 2


# ---- per-head norm + rotation

def rotate(y, cos, sin, inter):
    """cos, sin [tokens, pairs]; y [tokens, heads, D]."""
    n = cos.shape[1]
    a, b = (y[..., 0:2 * n:2], y[..., 1:2 * n:2]) if inter else (y[..., :n], y[..., n:2 * n])
    c, s = cos[:, None], sin[:, None]
    u, w = a * c - b * s, a * s + b * c
    head = torch.stack((u, w), -1).flatten(-2) if inter else torch.cat((u, w), -1)
    return torch.cat((head, y[..., 2 * n:]), -1)


def token_angles(angles, axes, pos):
    pos = pos[:, None] if pos.dim() == 1 else pos
    cols, at = [], 0
    for a, n in enumerate(axes):
        cols.append(angles.double()[pos[:, a].long(), at:at + n])
        at += n
    return torch.cat(cols, 1)


def head_norm(x, w, ang, inter, eps, scale):
    """The definition in 64 bits (x, w may require gradients)."""
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)
    if w is not None:
        y = y * w
    return rotate(y, ang.cos(), ang.sin(), inter) * scale


def head_norm_allow(y):
    """Forward: fp32 up to the one rounding. Before the rotation a value carries a relative error of a
    few E (the sum of squares D/2 E at worst in its halved exponent, rsqrt, two products), the table's
    cos and sin half a step each, and the rotation mixes the two values of a pair: 2^10 E of the largest
    value of the head covers D <= 256."""
    return H * y.abs() + 2 ** 10 * E * y.abs().amax(-1, keepdim=True)


# ---- attention

def attention(q, k, v, q_lens, k_lens, causal, scale, dout=None):
    """Packed attention of bf16 (or wider) tensors in 64 bits: a dict of out, lse and, with dout, dq, dk,
    dv, and the allowed absolute error of each ("out_a", ...)."""
    q, k, v = q.double(), k.double(), v.double()
    hq, hk = q.shape[1], k.shape[1]
    r = {n: torch.zeros_like(q) for n in ("out", "out_a")}
    r["lse"] = torch.full((hq, q.shape[0]), -math.inf, dtype=torch.float64, device=q.device)
    r["lse_a"] = torch.zeros_like(r["lse"])
    if dout is not None:
        dout = dout.double()
        for n in ("dq", "dq_a"):
            r[n] = torch.zeros_like(q)
        for n in ("dk", "dk_a", "dv", "dv_a"):
            r[n] = torch.zeros_like(k)
    q0 = k0 = 0
    for lq, lk in zip(q_lens, k_lens):
        qs, ks = slice(q0, q0 + lq), slice(k0, k0 + lk)
        q0, k0 = q0 + lq, k0 + lk
        if lq == 0 or lk == 0:
            continue
        i = torch.arange(lq, device=q.device)[:, None]
        j = torch.arange(lk, device=q.device)[None, :]
        seen = (j <= i + lk - lq) if causal else torch.ones(lq, lk, dtype=torch.bool, device=q.device)
        for h in range(hq):
            g = h // (hq // hk)
            Q, K, V = q[qs, h], k[ks, g], v[ks, g]
            S = (scale * Q @ K.T).masked_fill(~seen, -math.inf)
            lse = torch.logsumexp(S, -1)
            P = torch.exp(S - lse[:, None]).nan_to_num(0.0)
            O = P @ V
            # a score is an fp32 sum of 128 exact products (128 E of their absolute sum), scaled and
            # referred to the row's reference (a few E of the score); exp2 and the log add E's:
            # the relative error of a probability, or the absolute one of lse
            mag = (scale * Q.abs() @ K.abs().T).masked_fill(~seen, 0.0)
            rel = (136 * E * mag.amax(-1, keepdim=True) + (64 + lk) * E)
            # P is rounded to bf16 for the product with V (its sum is not), then the output is rounded
            PV = P @ V.abs()
            r["out"][qs, h] = O
            r["out_a"][qs, h] = H * O.abs() + (H + 2 * rel) * (1 + H) * PV
            r["lse"][h, qs] = lse
            r["lse_a"][h, qs] = 2 * rel[:, 0] + 4 * E * lse.abs().nan_to_num(0.0, 0.0, 0.0)
            if dout is None:
                continue
            dO = dout[qs, h]
            dP = dO @ V.T
            delta = (dO * O).sum(-1, keepdim=True)
            dS = P * (dP - delta)
            # delta is taken from the rounded output: its error is the output's, against |dO|
            e_delta = (dO.abs() * r["out_a"][qs, h]).sum(-1, keepdim=True)
            # dS is rounded to bf16 once; before that P's relative error, dP's and delta's fp32 errors
            e_ds = H * dS.abs() + (1 + H) * (P * (e_delta + (136 * E + 4 * rel) *
                                                  (dO.abs() @ V.abs().T + (dO * O).abs().sum(-1, keepdim=True))))
            r["dq"][qs, h] = scale * dS @ K
            r["dk"][ks, g] += scale * dS.T @ Q
            r["dv"][ks, g] += P.T @ dO
            # (fp32 sums over the keys or queries: their count in E's)
            r["dq_a"][qs, h] = scale * (e_ds + lk * E * dS.abs()) @ K.abs()
            r["dk_a"][ks, g] += scale * (e_ds + lq * hq * E * dS.abs()).T @ Q.abs()
            r["dv_a"][ks, g] += (P * (H + 4 * rel + lq * hq * E)).T @ dO.abs()
    if dout is not None:
        for n in ("dq", "dk", "dv"):
            r[n + "_a"] = r[n + "_a"] * (1 + H) + H * r[n].abs()
    return r


def decode(q, k, v, lens, scale):
    """Single-token attention in 64 bits: (out, allowed error)."""
    out, allow = torch.zeros_like(q, dtype=torch.float64), torch.zeros_like(q, dtype=torch.float64)
    for b, n in enumerate(lens):
        n = max(0, min(int(n), k.shape[1]))
        if n == 0:
            continue
        r = attention(q[b:b + 1], k[b, :n], v[b, :n], [1], [n], False, scale)
        out[b], allow[b] = r["out"][0], r["out_a"][0]
    return out, allow


def assert_within(name, got, want, allow):
    got = got.double()
    assert torch.isfinite(got).all(), f"{name}: not finite"
    over = (got - want).abs() - allow
    # (an exact zero has no allowance: it has to come out as one)
    worst = over.max().item() if over.numel() else 0.0
    assert worst <= 0.0, f"{name}: {worst:.3e} beyond the allowance; worst ratio " \
        f"{((got - want).abs() / allow.clamp_min(1e-300)).max().item():.3f}"
