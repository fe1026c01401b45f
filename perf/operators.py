"""Performance cases of the attention operators: rotary positions, norms of queries and keys with the rotation in the same
pass, attention with a sliding window and sink tokens in training and prefill, and the same over a cache for single tokens.

Tensors have the package's layout: [B, N, E], head h of a row in the features h * d .. h * d + d - 1; keys and values may
have fewer heads than queries. Random inputs are N(0, 1), which is what normalised queries and keys look like.
"""
import math

import torch

own = False


def _rot(name, B, N, H, Hk, d, R, dtype="bf16", interleaved=False, norm=False, train=False, start=0, scaling="none"):
    return {"name": name, "kind": "rotary", "B": B, "N": N, "H": H, "Hk": Hk, "d": d, "R": R, "dtype": dtype,
            "interleaved": interleaved, "norm": norm, "train": train, "start": start, "scaling": scaling}


def _att(name, B, Nq, Nk, H, Hk, d, window, sinks, dtype="bf16", train=False, ragged=False):
    return {"name": name, "kind": "attention", "B": B, "Nq": Nq, "Nk": Nk, "H": H, "Hk": Hk, "d": d, "window": window,
            "sinks": sinks, "dtype": dtype, "train": train, "ragged": ragged}


def _dec(name, B, Nq, S, H, Hk, d, window, sinks, dtype="bf16"):
    return {"name": name, "kind": "decode", "B": B, "Nq": Nq, "S": S, "H": H, "Hk": Hk, "d": d, "window": window,
            "sinks": sinks, "dtype": dtype}


def listed():
    return [
        # One new token of each of four sequences, far into their contexts: the rotation in a serving step. The smallest call.
        _rot("rotary_step", 4, 1, 32, 8, 128, 128, start=100000, scaling="yarn"),
        # A training batch whose heads are rotated in part, neighbouring features paired, fp32.
        _rot("rotary_part_train", 2, 4096, 16, 4, 128, 64, dtype="f32", interleaved=True, train=True, scaling="linear"),
        # Norm and rotation at the token shape of the reference's own gradient test, fp32: launches count.
        _rot("norm_tokens_train", 4, 256, 4, 4, 32, 32, dtype="f32", norm=True, train=True),
        # Norm and rotation of a prefill of odd length with heads of 96 features.
        _rot("norm_ragged", 3, 1999, 12, 6, 96, 96, norm=True, scaling="ntk"),
        # Norm and rotation in a training step of ordinary size in mixed precision.
        _rot("norm_train", 4, 8192, 32, 8, 128, 128, norm=True, train=True),
        # The token shape of the reference's gradient test, windows of its group size: the smallest training step of the attention.
        _att("window_tokens_train", 4, 256, 256, 4, 4, 32, 32, 0, dtype="f32", train=True),
        # A local layer in training: 4096 tokens, windows of 1024, four sinks, grouped key and value heads.
        _att("window_train", 2, 4096, 4096, 16, 4, 128, 1024, 4, train=True),
        # A padded batch of odd length with a head per key and value head, heads of 64, an odd window.
        _att("window_padded_train", 3, 1999, 1999, 12, 12, 64, 333, 5, train=True, ragged=True),
        # A long prompt through a local layer. The largest.
        _att("window_prefill", 1, 16384, 16384, 16, 4, 128, 4096, 4),
        # A chunk of a prompt behind what the cache holds already.
        _att("window_chunk", 2, 512, 8192, 32, 8, 128, 2048, 16),
        # Serving: one token of one sequence. Latency counts.
        _dec("decode_one", 1, 1, 4096, 32, 8, 128, 1024, 4),
        # Serving: one token each of 64 sequences of mixed lengths.
        _dec("decode_64", 64, 1, 8192, 32, 8, 128, 4096, 4),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rotary", "rotary", "attention", "attention", "attention", "decode", "decode"])
    Hk = rng.choice([1, 2, 3, 4, 8])
    H = Hk * rng.choice([1, 1, 2, 3, 4, 8])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    if kind == "rotary":
        d = rng.choice([32, 40, 64, 64, 80, 96, 128, 128])
        N = _log(rng, 1, 8192)
        B = max(1, min(_log(rng, 1, 64), 100_000_000 // (N * (H + Hk) * d)))
        R = d if rng.random() < 0.6 else rng.choice([d // 2, d // 4 * 2])
        return {"kind": kind, "B": B, "N": N, "H": H, "Hk": Hk, "d": d, "R": R, "dtype": dtype, "interleaved": rng.random() < 0.3,
                "norm": rng.random() < 0.6, "train": rng.random() < 0.5, "start": rng.choice([0, _log(rng, 1, 1_000_000)]),
                "scaling": rng.choice(["none", "linear", "ntk", "yarn"])}
    d = rng.choice([32, 64, 64, 80, 96, 128, 128, 128])
    if kind == "decode":
        S = _log(rng, 16, 16384)
        B = max(1, min(_log(rng, 1, 64), 400_000_000 // (S * Hk * d)))
        return {"kind": kind, "B": B, "Nq": rng.choice([1, 1, 1, 2, 4]), "S": S, "H": H, "Hk": Hk, "d": d,
                "window": _log(rng, 1, 8192), "sinks": rng.choice([0, 1, 4, 16]), "dtype": dtype}
    train = rng.random() < 0.6
    Nk = _log(rng, 16, 8192)
    Nq = Nk if train or rng.random() < 0.5 else rng.randint(1, Nk)
    cap = (5e8 if dtype == "f32" else 1e9) if train else (1e9 if dtype == "f32" else 3e9)
    B = max(1, min(_log(rng, 1, 16), int(cap / (Nq * Nk * H))))
    while B * H * Nq * Nk > cap:
        Hk, H = max(1, Hk // 2), max(1, Hk // 2) * (H // Hk)
        if Hk == 1 and B * H * Nq * Nk > cap:
            Nq = Nk = Nk // 2
    return {"kind": kind, "B": B, "Nq": Nq, "Nk": Nk, "H": H, "Hk": Hk, "d": d, "window": _log(rng, 1, 8192),
            "sinks": rng.choice([0, 0, 1, 4, 16, 130]), "dtype": dtype, "train": train, "ragged": rng.random() < 0.3}


def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def _frequencies(R, scaling):
    """Radians per position of the R / 2 pairs, and the factor of the rotated features, for contexts eight times as long as trained."""
    i = torch.arange(0, R, 2, dtype=torch.float64)
    base, factor, trained, magnitude = 10000.0, 8.0, 4096, 1.0
    f = base ** (-i / max(R, 1))
    if scaling == "linear":
        f = f / factor
    elif scaling == "ntk":
        f = (base * factor ** (R / max(R - 2, 1))) ** (-i / max(R, 1))
    elif scaling == "yarn":  # fast pairs keep their frequency, slow ones are interpolated, a ramp between
        turns = trained * f / (2 * math.pi)
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0, 1)
        f = f * keep + f / factor * (1 - keep)
        magnitude = 0.1 * math.log(factor) + 1.0
    return f.cuda(), magnitude


def _lengths(B, lo, hi, g):
    """A length for each row, spread over lo .. hi; the first has the whole length."""
    n = torch.randint(lo, hi + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    n[0] = hi
    return n


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    B, H, Hk, d, dtype = case["B"], case["H"], case["Hk"], case["d"], _dtype(case)

    def randn(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)

    s = {"case": case}
    if case["kind"] == "rotary":
        N = case["N"]
        s["q"], s["k"] = randn(B, N, H * d), randn(B, N, Hk * d)
        s["freqs"], s["magnitude"] = _frequencies(case["R"], case["scaling"])
        s["positions"] = case["start"] + torch.arange(N, device="cuda") + torch.randint(0, 100, (B, 1), generator=g, device="cuda")
        if case["norm"]:
            s["wq"] = 1.0 + 0.1 * torch.randn(d, generator=g, device="cuda")
            s["wk"] = 1.0 + 0.1 * torch.randn(d, generator=g, device="cuda")
        if case["train"]:
            s["dq"], s["dk"] = randn(B, N, H * d), randn(B, N, Hk * d)
        leaves = [s[n] for n in ("q", "k", "wq", "wk") if n in s]
    elif case["kind"] == "attention":
        Nq, Nk = case["Nq"], case["Nk"]
        s["q"], s["k"], s["v"] = randn(B, Nq, H * d), randn(B, Nk, Hk * d), randn(B, Nk, Hk * d)
        s["ctxlen"] = _lengths(B, max(1, Nk // 4), Nk, g) if case["ragged"] else None
        if case["train"]:
            s["dy"] = randn(B, Nq, H * d)
        leaves = [s["q"], s["k"], s["v"]]
    else:
        s["q"], s["k"], s["v"] = randn(B, case["Nq"], H * d), randn(B, case["S"], Hk * d), randn(B, case["S"], Hk * d)
        s["ctxlen"] = _lengths(B, max(1, case["S"] // 4), case["S"], g)
    if case.get("train"):
        for t in leaves:
            t.requires_grad_(True)
    return s


# ---------------------------------------------------------------- the plain forms
def _pairs(x, R, interleaved):
    return (x[..., 0:R:2], x[..., 1:R:2]) if interleaved else (x[..., : R // 2], x[..., R // 2 : R])


def _unpairs(a, b, x, R, interleaved):
    ab = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([ab, x[..., R:]], -1)


def _turn(x, cos, sin, R, interleaved):
    a, b = _pairs(x, R, interleaved)
    return _unpairs(a * cos - b * sin, b * cos + a * sin, x, R, interleaved)


def _plain_rotary_one(x, w, dy, cos, sin, case, heads, eps=1e-6):
    """Norm (where there is a weight) and rotation of one tensor, and the gradients of its input and weight for dy."""
    R, il, d = case["R"], case["interleaved"], case["d"]
    u = x.detach().float().unflatten(-1, (heads, d))
    if w is not None:
        r = torch.rsqrt(u.square().mean(-1, keepdim=True) + eps)
        xhat = u * r
        u = xhat * w.detach()
    y = [_turn(u, cos, sin, R, il).flatten(-2).to(x.dtype)]
    if dy is not None:
        g = _turn(dy.float().unflatten(-1, (heads, d)), cos, -sin, R, il)
        if w is None:
            return y + [g.flatten(-2).to(x.dtype)]
        gw = g * w.detach()
        dx = r * (gw - xhat * (gw * xhat).mean(-1, keepdim=True))
        return y + [dx.flatten(-2).to(x.dtype), (g * xhat).flatten(0, -2).sum(0)]
    return y


def _plain_rotary(s):
    c = s["case"]
    angle = s["positions"].double()[..., None, None] * s["freqs"]
    cos, sin = (angle.cos() * s["magnitude"]).float(), (angle.sin() * s["magnitude"]).float()
    q = _plain_rotary_one(s["q"], s.get("wq"), s.get("dq"), cos, sin, c, c["H"])
    k = _plain_rotary_one(s["k"], s.get("wk"), s.get("dk"), cos, sin, c, c["Hk"])
    return {"y": [q[0], k[0]], "dx": [q[1], k[1]] if len(q) > 1 else [], "dw": [q[2], k[2]] if len(q) > 2 else []}


def _hidden(p, Nk, n, window, sinks):
    """True where the query at position p [B, Nq] does not see key j: [B, 1, 1, Nq, Nk]. n [B]: keys of each row."""
    j = torch.arange(Nk, device=p.device)
    p, n = p[:, :, None], n.view(-1, 1, 1)
    seen = (j < n) & (p < n) & (j <= p) & ((p - j < window) | (j < sinks))
    return ~seen[:, None, None]


def _heads(x, Hk, groups, d):
    """[B, N, heads * d] -> [B, Hk, groups, N, d] in 32 bits."""
    return x.detach().float().unflatten(-1, (Hk, groups, d)).permute(0, 2, 3, 1, 4)


def _flat(x, dtype):
    return x.permute(0, 3, 1, 2, 4).flatten(2).to(dtype)


def _plain_attention(s):
    c = s["case"]
    B, H, Hk, d = c["B"], c["H"], c["Hk"], c["d"]
    Nq, Nk = s["q"].shape[1], s["k"].shape[1]
    n = s["ctxlen"] if s["ctxlen"] is not None else torch.full((B,), Nk, device="cuda")
    start = (n - Nq).view(B, 1) if c["kind"] == "decode" else torch.full((B, 1), Nk - Nq, device="cuda")
    hidden = _hidden(start + torch.arange(Nq, device="cuda"), Nk, n, c["window"], c["sinks"])
    scale = 1 / math.sqrt(d)
    q, k, v = _heads(s["q"], Hk, H // Hk, d), _heads(s["k"], Hk, 1, d), _heads(s["v"], Hk, 1, d)
    p = (q @ k.mT).mul_(scale).masked_fill_(hidden, -math.inf)
    p = p.sub_(p.amax(-1, keepdim=True).clamp_(min=-1e30)).exp_()
    total = p.sum(-1, keepdim=True)
    inv = torch.where(total > 0, 1 / total, 0.0)
    if not c.get("train"):
        return {"y": _flat((p @ v) * inv, s["q"].dtype)}
    p = p.mul_(inv)
    o = p @ v
    do = _heads(s["dy"], Hk, H // Hk, d)
    dv = (p.mT @ do).sum(2, keepdim=True)
    ds = (do @ v.mT).sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq, dk = ds @ k, (ds.mT @ q).sum(2, keepdim=True)
    t = s["q"].dtype
    return {"y": _flat(o, t), "dq": _flat(dq, t), "dk": _flat(dk, t), "dv": _flat(dv, t)}


# ---------------------------------------------------------------- the package's operators
def _own_rotary(s):
    import ncn_cuda_b200 as ncn

    c = s["case"]
    if c["norm"]:
        y = ncn.fused_qk_norm_rotary(s["q"], s["k"], s["wq"], s["wk"], s["freqs"], c["H"], positions=s["positions"],
                                     interleaved=c["interleaved"], magnitude=s["magnitude"], eps=1e-6)
    else:
        y = ncn.fused_rotary(s["q"], s["k"], s["freqs"], c["H"], positions=s["positions"], interleaved=c["interleaved"],
                             magnitude=s["magnitude"])
    out = {"y": [y[0].detach(), y[1].detach()], "dx": [], "dw": []}
    if c["train"]:
        leaves = [s["q"], s["k"]] + ([s["wq"], s["wk"]] if c["norm"] else [])
        grads = torch.autograd.grad(y, leaves, [s["dq"], s["dk"]])
        out["dx"], out["dw"] = list(grads[:2]), list(grads[2:])
    return out


def _own_attention(s):
    import ncn_cuda_b200 as ncn

    c = s["case"]
    if c["kind"] == "decode":
        return {"y": ncn.window_attention_decode(s["q"], s["k"], s["v"], s["ctxlen"], c["H"], c["window"], n_sink=c["sinks"])}
    y = ncn.fused_window_attention(s["q"], s["k"], s["v"], c["H"], c["window"], n_sink=c["sinks"], ctxlen=s["ctxlen"])
    if not c["train"]:
        return {"y": y}
    dq, dk, dv = torch.autograd.grad(y, [s["q"], s["k"], s["v"]], s["dy"])
    return {"y": y.detach(), "dq": dq, "dk": dk, "dv": dv}


def run(state):
    rotary = state["case"]["kind"] == "rotary"
    if own:
        return _own_rotary(state) if rotary else _own_attention(state)
    with torch.no_grad():
        return _plain_rotary(state) if rotary else _plain_attention(state)


# ---------------------------------------------------------------- what a pass cannot do without
def _visible(n, start, Nq, window, sinks):
    """Pairs of query and key that see each other in a row of n keys whose first query is at `start`; the keys seen by any."""
    pairs, lo = 0, n
    for i in range(Nq):
        p = start + i
        if 0 <= p < n:
            first = max(0, p - window + 1)
            pairs += p - first + 1 + min(sinks, first)
            lo = min(lo, first)
    return pairs, n - lo + min(sinks, lo)


def work(case):
    w = 2 if case["dtype"] == "bf16" else 4
    B, H, Hk, d = case["B"], case["H"], case["Hk"], case["d"]
    if case["kind"] == "rotary":
        x = B * case["N"] * (H + Hk) * d
        moved = 4 if case["train"] else 2  # x in, y out; dy in, dx out
        return {"bytes": x * w * moved + B * case["N"] * 8, "flops": x * (3 + (4 if case["norm"] else 0)) * (3 if case["train"] else 1)}
    if case["kind"] == "decode":
        # lengths are spread over a quarter of the cache to all of it: the middle
        n = case["S"] if B == 1 else max(1, case["S"] * 5 // 8)
        pairs, keys = _visible(n, n - case["Nq"], case["Nq"], case["window"], case["sinks"])
        return {"bytes": w * d * B * (2 * Hk * keys + 2 * H * case["Nq"]), "flops": 4 * d * B * H * pairs}
    Nq, Nk = case["Nq"], case["Nk"]
    n = (Nk + max(1, Nk // 4)) // 2 if case["ragged"] and B > 1 else Nk
    pairs, keys = _visible(n, Nk - Nq, Nq, case["window"], case["sinks"])
    one = {"q": H * Nq, "kv": 2 * Hk * max(keys, 1)}
    if case["train"]:  # q, k, v, dy in; y and three gradients out
        return {"bytes": w * d * B * (4 * one["q"] + 2 * one["kv"]), "flops": 14 * d * B * H * max(pairs, 1)}
    return {"bytes": w * d * B * (2 * one["q"] + one["kv"]), "flops": 4 * d * B * H * max(pairs, 1)}


# ---------------------------------------------------------------- the definitions in 64 bits
def _exact_rotary(case, s):
    """Pair by pair as complex numbers; the gradients by automatic differentiation in 64 bits."""
    B, N, d, R = case["B"], case["N"], case["d"], case["R"]
    phase = torch.polar(torch.full((B, N, 1, R // 2), s["magnitude"], dtype=torch.float64, device="cuda"),
                        torch.remainder(s["positions"].double()[..., None, None] * s["freqs"], 2 * math.pi))
    ys, dxs, dws = [], [], []
    for name, heads in (("q", case["H"]), ("k", case["Hk"])):
        x = s[name].detach().double().requires_grad_(case["train"])
        u, leaves = x.view(B, N, heads, d), [x]
        if case["norm"]:
            w = s["w" + name].detach().double().requires_grad_(case["train"])
            leaves.append(w)
            u = w * u / torch.sqrt((u * u).sum(-1, keepdim=True) / d + 1e-6)
        head, tail = u[..., :R], u[..., R:]
        if case["interleaved"]:
            z = torch.view_as_complex(head.reshape(B, N, heads, R // 2, 2).contiguous()) * phase
            head = torch.view_as_real(z).reshape(B, N, heads, R)
        else:
            z = torch.complex(head[..., : R // 2], head[..., R // 2 :]) * phase
            head = torch.cat([z.real, z.imag], -1)
        y = torch.cat([head, tail], -1).reshape(B, N, heads * d)
        ys.append(y.detach())
        if case["train"]:
            got = torch.autograd.grad(y, leaves, s["d" + name].double())
            dxs.append(got[0])
            dws += got[1:]
        del x, u, head, tail, z, y
    return {"y": ys, "dx": dxs, "dw": dws}


def _exact_attention(case, s):
    """Head by head: the softmax over the keys that each query sees, and its gradients."""
    B, H, Hk, d = case["B"], case["H"], case["Hk"], case["d"]
    Nq, Nk, train = s["q"].shape[1], s["k"].shape[1], case.get("train", False)
    y = torch.zeros(B, Nq, H * d, dtype=torch.float64, device="cuda")
    dq = torch.zeros_like(y)
    dk = torch.zeros(B, Nk, Hk * d, dtype=torch.float64, device="cuda")
    dv = torch.zeros_like(dk)
    i, j = torch.arange(Nq, device="cuda")[:, None], torch.arange(Nk, device="cuda")[None, :]
    for b in range(B):
        n = int(s["ctxlen"][b]) if s["ctxlen"] is not None else Nk
        p = i + (n - Nq if case["kind"] == "decode" else Nk - Nq)
        seen = (j < n) & (p < n) & (j <= p) & ((j > p - case["window"]) | (j < case["sinks"]))
        for h in range(H):
            a, c = slice(h * d, h * d + d), slice(h // (H // Hk) * d, h // (H // Hk) * d + d)
            q, k, v = s["q"][b, :, a].detach().double(), s["k"][b, :, c].detach().double(), s["v"][b, :, c].detach().double()
            score = torch.where(seen, q @ k.T / math.sqrt(d), -1e300)
            w = torch.where(seen, torch.softmax(score, -1), 0.0)
            o = w @ v
            y[b, :, a] = o
            if train:
                do = s["dy"][b, :, a].double()
                dv[b, :, c] += w.T @ do
                ds = w * (do @ v.T - (do * o).sum(-1, keepdim=True)) / math.sqrt(d)
                dq[b, :, a] = ds @ k
                dk[b, :, c] += ds.T @ q
    return {"y": y, "dq": dq, "dk": dk, "dv": dv} if train else {"y": y}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rotary":
        return _exact_rotary(case, s)
    with torch.no_grad():
        return _exact_attention(case, s)
