"""Plain 64-bit forms of the attention operators, and bounds of what 32-bit sums and roundings to the storage type may change.

A result is compared element by element with a bound that is summed up in the same way as the result itself, over absolute
values: half a step of the storage type for each rounding to it (weights of the softmax and dS in bf16, the results), and
the rounding of fp32 sums."""
import math

import torch

HALF = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8}  # half a step, relative


def heads(x, n, d):
    """[B, N, n * d] -> [B, n, N, d] in 64 bits"""
    return x.detach().double().unflatten(-1, (n, d)).transpose(1, 2)


def flat(x):
    return x.transpose(1, 2).flatten(2)


def visible(B, Nq, Nk, window, n_sink, ctxlen, start, device):
    """[B, 1, Nq, Nk].  ctxlen, start: ints or [B]"""
    ctx = torch.as_tensor(ctxlen, device=device).long().expand(B).clamp(0, Nk)[:, None, None]
    p = torch.as_tensor(start, device=device).long().expand(B)[:, None, None] + torch.arange(Nq, device=device)[None, :, None]
    j = torch.arange(Nk, device=device)[None, None, :]
    return ((j < ctx) & (j <= p) & (p < ctx) & ((p - j < window) | (j < n_sink)))[:, None]


def clean(x, rows):
    """x [B, n, N, d] with zeros where a row takes part in nothing (it may hold NaN there)"""
    return torch.where(rows[:, :, :, None], x, 0.0)


def attention(q, k, v, n_head, window, n_sink, scale, ctxlen, start, dy=None):
    """-> {name: (value, bound)} of y and, with dy, dq, dk, dv."""
    dtype = q.dtype
    B, Nq, E = q.shape
    Nk, d = k.shape[1], E // n_head
    n_kv = k.shape[2] // d
    G = n_head // n_kv
    see = visible(B, Nq, Nk, window, n_sink, ctxlen, start, q.device)
    lively_q, lively_k = see.any(-1), see.any(-2)
    Q = clean(heads(q, n_head, d), lively_q)
    K = clean(heads(k, n_kv, d), lively_k).repeat_interleave(G, 1)
    V = clean(heads(v, n_kv, d), lively_k).repeat_interleave(G, 1)
    half = HALF[dtype]
    u = 2.0**-24
    S = scale * (Q @ K.mT)
    m = torch.where(see, S, -math.inf).amax(-1, keepdim=True)
    m = torch.where(m.isinf(), 0.0, m)
    P = torch.where(see, torch.exp(S - m), 0.0)
    total = P.sum(-1, keepdim=True)
    P = torch.where(total > 0, P / total, 0.0)
    Y = P @ V
    # what a weight may be off by, relatively: the score's sum of d products and its scaling (absolute, times two: the score and
    # the row's largest, and as much for the sum that divides), the exponential and the sums' terms
    count = float(see.sum(-1).max().clamp(min=1))
    ds = ((d + 6) * u * scale * (Q.abs() @ K.abs().mT) * see).amax(-1, keepdim=True)
    w32 = 4 * ds + (2 * math.sqrt(count) + 32) * u + 2.0**-21
    rounded = half if dtype != torch.float32 else 0.0
    A = P @ V.abs()
    ey = (w32 + rounded) * A
    out = {"y": (flat(Y), flat(ey + half * (Y.abs() + ey) + 1e-30))}
    if dy is None:
        return out
    dO = clean(heads(dy, n_head, d), lively_q)
    dP = dO @ V.mT
    D = (dO * Y).sum(-1, keepdim=True)
    dS = P * (dP - D)
    e_delta = (dO.abs() * (ey + half * half * (Y.abs() + ey))).sum(-1, keepdim=True) + (d + 2) * u * (dO * Y).abs().sum(-1, keepdim=True)
    e_dp = (d + 2) * u * (dO.abs() @ V.abs().mT)
    e_ds = dS.abs() * (w32 + rounded) + P * (e_dp + e_delta) * (1 + rounded)
    acc_q, acc_k = (2 * math.sqrt(count) + 32) * u, (2 * math.sqrt(float(G * Nq)) + 32) * u

    def group(x):
        return x.unflatten(1, (n_kv, G)).sum(2)

    def add(name, value, err):
        out[name] = (flat(value), flat(err + half * (value.abs() + err) + 1e-30))

    add("dq", scale * (dS @ K), scale * (e_ds + acc_q * dS.abs()) @ K.abs())
    add("dk", scale * group(dS.mT @ Q), scale * group((e_ds + acc_k * dS.abs()).mT @ Q.abs()))
    add("dv", group(P.mT @ dO), group(((w32 + rounded + acc_k) * P).mT @ dO.abs()))
    return out


def turn(x, positions, freqs, interleaved, magnitude, inverse=False):
    """x [B, N, n, d] in 64 bits; positions [B, N]"""
    R = 2 * freqs.numel()
    a = positions.double()[..., None, None] * freqs.double()
    c, s = magnitude * a.cos(), magnitude * a.sin()
    if inverse:
        s = -s
    if interleaved:
        u, w = x[..., 0:R:2], x[..., 1:R:2]
        head = torch.stack([u * c - w * s, w * c + u * s], -1).flatten(-2)
    else:
        u, w = x[..., : R // 2], x[..., R // 2 : R]
        head = torch.cat([u * c - w * s, w * c + u * s], -1)
    return torch.cat([head, x[..., R:]], -1)


def norm_rotary(x, w, n, positions, freqs, interleaved, magnitude, eps=1e-6, dy=None):
    """-> {"y": (value, bound)} and, with dy, "dx" and (with a weight) "dw"."""
    B, N, E = x.shape
    d = E // n
    half, u = HALF[x.dtype], 2.0**-24
    X = x.detach().double().reshape(B, N, n, d)
    turned = lambda t, inv=False: turn(t, positions, freqs, interleaved, magnitude, inv)  # noqa: E731
    # a pair's two features each gain u of each other's size, times a few roundings
    size = lambda t: turn_sizes(t, freqs, interleaved, magnitude)  # noqa: E731
    e_rel = (0.25 * d + 24) * u  # the norm's sum of squares (half of it after the root), products, sine and cosine
    U = X
    if w is not None:
        W = w.detach().double()
        r = 1 / torch.sqrt(X.square().mean(-1, keepdim=True) + eps)
        U = X * r * W
    Y, e = turned(U), e_rel * size(U)
    flatten = lambda t: t.reshape(B, N, E)  # noqa: E731
    out = {"y": (flatten(Y), flatten(e + half * (Y.abs() + e) + 1e-30))}
    if dy is None:
        return out
    g0 = dy.detach().double().reshape(B, N, n, d)
    G, eg = turned(g0, True), e_rel * size(g0)
    if w is None:
        out["dx"] = (flatten(G), flatten(eg + half * (G.abs() + eg) + 1e-30))
        return out
    xh = X * r
    gw = G * W
    c = (gw * xh).mean(-1, keepdim=True)
    dx = r * (gw - xh * c)
    ec = (eg * W.abs() * xh.abs() + (d + 2 * e_rel / u) * u * (gw * xh).abs()).mean(-1, keepdim=True)
    e = r * (eg * W.abs() + 2 * e_rel * (gw.abs() + (xh * c).abs()) + xh.abs() * ec)
    out["dx"] = (flatten(dx), flatten(e + half * (dx.abs() + e) + 1e-30))
    terms = G * xh
    e = (eg * xh.abs() + (2 * e_rel + (2 * math.sqrt(B * N * n) + 32) * u) * terms.abs()).sum((0, 1, 2))
    out["dw"] = (terms.sum((0, 1, 2)), e + u * terms.sum((0, 1, 2)).abs() + 1e-30)
    return out


def turn_sizes(x, freqs, interleaved, magnitude):
    """|a| + |b| of each feature's pair, |a| of a feature that passes"""
    R = 2 * freqs.numel()
    x = x.abs()
    m = max(abs(magnitude), 1.0)
    if interleaved:
        s = (x[..., 0:R:2] + x[..., 1:R:2]).repeat_interleave(2, -1)
    else:
        s = x[..., : R // 2] + x[..., R // 2 : R]
        s = torch.cat([s, s], -1)
    return torch.cat([m * s, x[..., R:]], -1)


def close(name, got, want):
    value, bound = want
    assert got.shape == value.shape, (name, got.shape, value.shape)
    assert torch.isfinite(got).all(), name
    over = (got.double() - value).abs() / bound
    worst = float(over.max()) if over.numel() else 0.0
    assert worst <= 1.0, f"{name}: {worst:.3f} times its bound at {int(over.argmax())}"
