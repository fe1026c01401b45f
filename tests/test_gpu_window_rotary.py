"""Rotary positions, norms of queries and keys with the rotation, and the run of these with windowed attention; against 64 bits."""
import math

import pytest
import torch

import ncn_cuda_b200 as ncn
from ncn_cuda_b200 import ops
from tests import window_oracle as O

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def make(seed, B, N, H, Hk, d, dtype):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda h: torch.randn(B, N, h * d, generator=g, device="cuda").to(dtype)  # noqa: E731
    w = lambda: 1 + 0.2 * torch.randn(d, generator=g, device="cuda")  # noqa: E731
    return r(H), r(Hk), r(H), r(Hk), w(), w()


def grid_of(positions, B, N):
    if positions is None:
        positions = 0
    if isinstance(positions, int):
        return (positions + torch.arange(N, device="cuda")).expand(B, N)
    return torch.as_tensor(positions, device="cuda").expand(B, N)


def check(q, k, dq, dk, wq, wk, freqs, H, positions=None, interleaved=False, magnitude=1.0):
    B, N, E = q.shape
    d = E // H
    pos = grid_of(positions, B, N)
    norm = wq is not None
    leaves = [t.clone().requires_grad_(True) for t in ([q, k, wq, wk] if norm else [q, k])]
    if norm:
        y = ncn.fused_qk_norm_rotary(*leaves, freqs, H, positions=positions, interleaved=interleaved, magnitude=magnitude)
    else:
        y = ncn.fused_rotary(*leaves, freqs, H, positions=positions, interleaved=interleaved, magnitude=magnitude)
    grads = torch.autograd.grad(y, leaves, [dq, dk])
    torch.cuda.synchronize()
    f = freqs.cuda()
    for i, (x, w, g, n) in enumerate(((q, wq, dq, H), (k, wk, dk, k.shape[2] // d))):
        want = O.norm_rotary(x, w, n, pos, f, interleaved, magnitude, dy=g)
        O.close(f"y{i}", y[i].detach(), want["y"])
        O.close(f"dx{i}", grads[i], want["dx"])
        if norm:
            O.close(f"dw{i}", grads[2 + i], want["dw"])
    return y, grads


SHAPES = [  # B, N, H, Hk, d, R
    (1, 1, 1, 1, 64, 64), (4, 1, 32, 8, 128, 128), (2, 77, 3, 1, 96, 96), (1, 300, 4, 2, 128, 64), (2, 65, 2, 2, 32, 16),
    (1, 50, 5, 5, 16, 16), (2, 33, 4, 2, 80, 0), (1, 40, 2, 1, 256, 128), (2, 31, 3, 1, 40, 20), (1, 30, 2, 2, 34, 34), (1, 30, 2, 1, 33, 6),
    (1, 20, 2, 1, 512, 512), (3, 9, 2, 1, 2, 2), (1, 9, 2, 1, 1, 0), (2, 2000, 2, 1, 64, 64),
]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,N,H,Hk,d,R", SHAPES)
def test_both_directions(dtype, norm, interleaved, B, N, H, Hk, d, R):
    q, k, dq, dk, wq, wk = make(N + d, B, N, H, Hk, d, dtype)
    freqs, _ = ncn.rotary_frequencies(R, device="cuda")
    check(q, k, dq, dk, wq if norm else None, wk if norm else None, freqs, H, interleaved=interleaved)


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("d,R", [(64, 64), (34, 34)])
@pytest.mark.parametrize("scaling", ncn.attention.SCALINGS)
def test_far_positions(norm, d, R, scaling):
    """Angles of a million turns: in 32 bits nothing of them would be left."""
    q, k, dq, dk, wq, wk = make(7, 3, 50, 4, 2, d, F32)
    freqs, magnitude = ncn.rotary_frequencies(R, scaling=scaling, factor=8.0 if scaling else 1.0, device="cuda")
    w = (wq, wk) if norm else (None, None)
    far = torch.arange(50) + torch.tensor([[0], [1_000_000], [40_000_000]])
    for positions in (far, far.cuda(), far[1].to(torch.int32), far[1:2], 123_456_789, -77, far.flip(-1)):
        check(q, k, dq, dk, *w, freqs, 4, positions=positions, magnitude=magnitude)
    check(q, k, dq, dk, *w, freqs.float().cpu(), 4, positions=5)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_views(dtype):
    g = torch.Generator(device="cuda").manual_seed(3)
    H, Hk, d, B, N = 4, 2, 64, 2, 100
    _, _, dq, dk, wq, wk = make(1, B, N, H, Hk, d, dtype)
    freqs, _ = ncn.rotary_frequencies(d, device="cuda")
    for extra in (0, 3):  # 3: no 16-byte access reaches a row
        joint = torch.randn(B, N, (H + 2 * Hk) * d + extra, generator=g, device="cuda").to(dtype)[..., extra:]
        q, k = joint[..., : H * d], joint[..., H * d : (H + Hk) * d]
        for w in ((None, None), (wq, wk)):
            check(q, k, dq, dk, *w, freqs, H)
            check(q, k, dq[:, :1].expand_as(dq), dk[:1].expand_as(dk), *w, freqs, H)
    flat = torch.randn(B * N * H * d + 1, generator=g, device="cuda").to(dtype)[1:].view(B, N, H * d)  # contiguous, off the boundary
    check(flat, k, dq, dk, wq, wk, freqs, H)


def test_one_tensor_weights_of_other_types_and_missing_gradients():
    q, k, dq, dk, wq, wk = make(4, 2, 60, 4, 2, 64, BF16)
    freqs, _ = ncn.rotary_frequencies(64, device="cuda")
    y, none = ncn.fused_rotary(q, None, freqs, 4)
    both = ncn.fused_rotary(q, k, freqs, 4)
    assert none is None and torch.equal(y, both[0])
    leaves = [q.clone().requires_grad_(True), wq.to(BF16).requires_grad_(True)]
    y, none = ncn.fused_qk_norm_rotary(leaves[0], None, leaves[1], None, freqs, 4)
    gx, gw = torch.autograd.grad(y, leaves, dq)
    want = O.norm_rotary(q, leaves[1], 4, grid_of(None, 2, 60), freqs, False, 1.0, dy=dq)
    assert none is None and gw.dtype == BF16
    O.close("dx", gx, want["dx"])
    value, bound = want["dw"]
    O.close("dw", gw, (value, bound + 2.0**-8 * (value.abs() + bound)))  # rounded to the weight's type once more
    # a gradient for one of the two results only
    leaves = [t.clone().requires_grad_(True) for t in (q, k, wq, wk)]
    y = ncn.fused_qk_norm_rotary(*leaves, freqs, 4)
    grads = torch.autograd.grad(y[1], leaves, dk, allow_unused=True)
    want = O.norm_rotary(k, wk, 2, grid_of(None, 2, 60), freqs, False, 1.0, dy=dk)
    O.close("dk", grads[1], want["dx"])
    assert (grads[0] == 0).all() and (grads[2] == 0).all()


def test_nothing_to_do():
    freqs, _ = ncn.rotary_frequencies(64, device="cuda")
    for B, N in ((0, 3), (2, 0)):
        q, k, dq, dk, wq, wk = make(1, B, N, 2, 1, 64, F32)
        leaves = [t.requires_grad_(True) for t in (q, k, wq, wk)]
        y = ncn.fused_qk_norm_rotary(*leaves, freqs, 2)
        g = torch.autograd.grad(y, leaves, [dq, dk])
        assert y[0].shape == q.shape and (g[2] == 0).all() and (g[3] == 0).all()
        assert ncn.fused_rotary(q, k, freqs, 2)[0].shape == q.shape


def test_a_row_of_zeros_and_values_that_are_not_finite():
    q, k, dq, dk, wq, wk = make(5, 1, 40, 2, 1, 64, F32)
    q[0, 3] = 0
    freqs, _ = ncn.rotary_frequencies(64, device="cuda")
    check(q, k, dq, dk, wq, wk, freqs, 2)
    clean = ncn.fused_qk_norm_rotary(q, k, wq, wk, freqs, 2)[0]
    q[0, 7, 5] = math.nan  # head 0 of position 7
    y = ncn.fused_qk_norm_rotary(q, k, wq, wk, freqs, 2)[0]
    assert y[0, 7, :64].isnan().all()
    y[0, 7, :64] = clean[0, 7, :64]
    assert torch.equal(y, clean)


@pytest.mark.parametrize("d,N", [(64, 100), (96, 37), (33, 37)])
def test_eps_of_zero(d, N):
    q, k, dq, dk, wq, wk = make(5, 3, N, 3, 1, d, F32)
    freqs, _ = ncn.rotary_frequencies(32, device="cuda")
    leaves = [t.requires_grad_(True) for t in (q, k, wq, wk)]
    y = ncn.fused_qk_norm_rotary(*leaves, freqs, 3, eps=0.0)
    grads = torch.autograd.grad(y, leaves, [dq, dk])
    for i, (x, w, g, n) in enumerate(((q, wq, dq, 3), (k, wk, dk, 1))):
        want = O.norm_rotary(x, w, n, grid_of(None, 3, N), freqs, False, 1.0, eps=0.0, dy=g)
        O.close(f"y{i}", y[i].detach(), want["y"])
        O.close(f"dx{i}", grads[i], want["dx"])
        O.close(f"dw{i}", grads[2 + i], want["dw"])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_same_bits_captured(dtype):
    q, k, dq, dk, wq, wk = make(8, 2, 500, 4, 2, 128, dtype)
    freqs, _ = ncn.rotary_frequencies(128, device="cuda")
    leaves = [t.requires_grad_(True) for t in (q, k, wq, wk)]
    positions = torch.arange(500, device="cuda").expand(2, 500).contiguous()

    def step():
        y = ncn.fused_qk_norm_rotary(*leaves, freqs, 4, positions=positions)
        return (*[t.detach() for t in y], *torch.autograd.grad(y, leaves, [dq, dk]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    graph.replay()
    torch.cuda.synchronize()
    for x, y in zip(a, out):
        assert torch.equal(x, y)
    positions += 1000
    graph.replay()
    torch.cuda.synchronize()
    for x, y in zip(out, step()):
        assert torch.equal(x, y)


def test_gradient_against_differences():
    q, k, dq, dk, wq, wk = make(6, 1, 20, 2, 1, 32, F32)
    freqs, _ = ncn.rotary_frequencies(32, device="cuda")
    _, grads = check(q, k, dq, dk, wq, wk, freqs, 2)
    g = torch.Generator(device="cuda").manual_seed(8)
    for i, t in enumerate((q, k, wq, wk)):
        u = torch.randn(t.shape, generator=g, device="cuda")
        f = []
        for h in (1e-2, -1e-2):
            args = [q, k, wq, wk]
            args[i] = t + h * u
            y = ncn.fused_qk_norm_rotary(*args, freqs, 2)
            f.append((y[0].double() * dq).sum() + (y[1].double() * dk).sum())
        slope = float(f[0] - f[1]) / 2e-2
        want = float((grads[i].double() * u).sum())
        assert abs(slope - want) <= 1e-2 * float((grads[i].double().abs() * u.abs()).sum()), (i, slope, want)


def test_function_form_agrees():
    q, k, dq, dk, wq, wk = make(9, 2, 30, 4, 2, 64, BF16)
    freqs, _ = ncn.rotary_frequencies(64, device="cuda")
    pos = torch.arange(30, device="cuda")
    for w in ((None, None), (wq, wk)):
        leaves = [t.clone().requires_grad_(True) for t in (q, k, *w) if t is not None]
        args = (*leaves, *w[: 4 - len(leaves)], freqs, pos, 4, 0, False, 1e-6, 1.5)
        a = ncn.RotaryFunction.apply(*args)
        b = torch.autograd.Function.apply.__func__(ncn.RotaryFunction, *args)
        ga, gb = torch.autograd.grad(a, leaves, [dq, dk]), torch.autograd.grad(b, leaves, [dq, dk])
        for x, y in zip((*a, *ga), (*b, *gb)):
            assert torch.equal(x, y)


# ---------------------------------------------------------------- the operators in a run, as a layer uses them
@pytest.mark.parametrize("dtype,d", [(F32, 32), (BF16, 64), (BF16, 128)])
def test_layer_in_training_and_serving(dtype, d):
    """Norm and rotation, windowed attention and an NCN stage behind it; then the same token by token over a cache."""
    B, N, H, Hk, window, sinks, n_cache = 2, 192, 4, 2, 40, 3, 4
    g = torch.Generator(device="cuda").manual_seed(d)
    joint = torch.randn(B, N, (H + 2 * Hk) * d, generator=g, device="cuda").to(dtype).requires_grad_(True)
    wq, wk = ((1 + 0.1 * torch.randn(d, generator=g, device="cuda")).requires_grad_(True) for _ in range(2))
    W = (torch.randn(2 * H * d, generator=g, device="cuda") * 0.1).requires_grad_(True)
    freqs, _ = ncn.rotary_frequencies(d, device="cuda")
    dy = torch.randn(B, N, H * d, generator=g, device="cuda").to(dtype)

    q, k, v = joint.split([H * d, Hk * d, Hk * d], -1)
    qr, kr = ncn.fused_qk_norm_rotary(q, k, wq, wk, freqs, H)
    y = ncn.fused_window_attention(qr, kr, v, H, window, n_sink=sinks)
    z, za = ncn.fused_ncn_cuda_v2(y, torch.zeros_like(y), W, 0.9, 0, n_cache, H, 0)
    grads = torch.autograd.grad(z, [joint, wq, wk, W], dy, retain_graph=True)
    assert all(torch.isfinite(t).all() for t in grads)

    # the attention part against 64 bits, from the same rotated queries and keys and the same cotangent
    gy, = torch.autograd.grad(ncn.fused_ncn_cuda_v2(y, torch.zeros_like(y), W, 0.9, 0, n_cache, H, 0)[0], y, dy, retain_graph=True)
    want = O.attention(qr, kr, v, H, window, sinks, 1 / math.sqrt(d), N, 0, gy)
    O.close("y", y.detach(), want["y"])
    gq, gk, gv = torch.autograd.grad(y, [qr, kr, v], gy, retain_graph=True)
    for name, t in (("dq", gq), ("dk", gk), ("dv", gv)):
        O.close(name, t, want[name])
    pos = torch.arange(N, device="cuda").expand(B, N)
    nq, nk = O.norm_rotary(q, wq, H, pos, freqs, False, 1.0, dy=gq), O.norm_rotary(k, wk, Hk, pos, freqs, False, 1.0, dy=gk)
    gj, gwq, gwk = torch.autograd.grad(y, [joint, wq, wk], gy)
    O.close("d joint", gj, tuple(torch.cat(t, -1) for t in zip(nq["dx"], nk["dx"], (gv.double(), torch.full_like(gv, 1e-30).double()))))
    O.close("dwq", gwq, nq["dw"])
    O.close("dwk", gwk, nk["dw"])

    # serving: a prompt of 100 tokens in one call, a chunk of 50 behind it, then single tokens
    with torch.no_grad():
        kc, vc = torch.full((B, N, Hk * d), math.nan, dtype=dtype, device="cuda"), torch.full((B, N, Hk * d), math.nan, dtype=dtype, device="cuda")
        for lo, hi in [(0, 100), (100, 150)] + [(t, t + 1) for t in range(150, N)]:
            a, b = ncn.fused_qk_norm_rotary(q[:, lo:hi], k[:, lo:hi], wq, wk, freqs, H, positions=lo)
            kc[:, lo:hi], vc[:, lo:hi] = b, v[:, lo:hi]
            ctxlen = torch.full((B,), hi, dtype=torch.int32, device="cuda")
            if hi - lo > 1:
                out = ncn.fused_window_attention(a, kc, vc, H, window, n_sink=sinks, ctxlen=ctxlen, q_start=lo)
            else:
                out = ncn.window_attention_decode(a, kc, vc, ctxlen, H, window, n_sink=sinks)
            assert torch.equal(a, qr[:, lo:hi]) and torch.equal(b, kr[:, lo:hi])
            O.close(f"serving {lo}", out, tuple(t[:, lo:hi] for t in want["y"]))
    ops.device_status()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kw", [{}, {"qk_norm": False, "rot_dim": 32, "interleaved": True}, {"n_kv_head": 4, "scaling": "yarn", "factor": 4.0}])
def test_layer_module(dtype, kw):
    """forward against the operators one by one; step by step against forward, rows of different lengths."""
    torch.manual_seed(3)
    B, N, E, H = 3, 90, 256, 4
    layer = ncn.NCNWindowAttention(E, H, 20, n_sink=2, **{"n_kv_head": 2, **kw}).cuda().to(dtype)
    x = torch.randn(B, N, E, device="cuda").to(dtype)
    y = layer(x)
    y.float().square().mean().backward()
    for name, p in layer.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all() and p.grad.abs().sum() > 0, name
    q, k, v = layer._rotated(x, None)
    inner = ncn.fused_window_attention(q, k, v, H, 20, n_sink=2)
    assert torch.equal(y, layer.out(inner))
    want = O.attention(q, k, v, H, 20, 2, 1 / 8, N, 0)["y"]
    O.close("inner", inner.detach(), want)

    # rows of 40, 7 and 1 positions, padded in front to a prompt of 40, then 30 more each, one by one
    lens = torch.tensor([40, 7, 1], device="cuda")
    cache = layer.new_cache(B, N)
    prompt = torch.full((B, 40, E), math.nan, device="cuda", dtype=dtype)
    for b, n in enumerate(lens.tolist()):
        prompt[b, 40 - n :] = x[b, :n]
    got = layer.step(prompt, cache, lens)
    # The same projections in other batches may be summed in another order.  bf16: roundings of the projection, the rotated heads, the inner
    # result and the last one, 2^-8 of the largest each, on both sides: 8 * 2^-8.  fp32: three sums of 256 terms on both sides, 2^-24 of
    # the terms each: 6 * 256 * 2^-24 of the terms, which are no larger than 1.1 times the results' largest here.
    tol = {F32: 1.1 * 6 * 256 * 2.0**-24, BF16: 8 * 2.0**-8}[dtype]
    for b, n in enumerate(lens.tolist()):
        assert (got[b, 40 - n :] - y[b, :n]).abs().max() <= tol * y.abs().max()
        assert (got[b, : 40 - n] == 0).all()
        assert torch.isfinite(cache[0][b, :N]).all()
    for t in range(30):
        lens += 1
        one = torch.stack([x[b, n - 1 : n] for b, n in enumerate(lens.tolist())])
        got = layer.step(one, cache, lens)
        for b, n in enumerate(lens.tolist()):
            assert (got[b, 0] - y[b, n - 1]).abs().max() <= tol * y.abs().max(), (t, b)
