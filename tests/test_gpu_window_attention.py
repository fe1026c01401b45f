"""Windowed attention with sinks: training, chunks of a prompt, padded batches, single tokens over a cache; against 64 bits."""
import math
import subprocess
import sys

import pytest
import torch

import ncn_cuda_b200 as ncn
from ncn_cuda_b200 import ops
from tests import window_oracle as O
from tests.kernels_util import kernels_of, launched

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def make(seed, B, Nq, Nk, H, Hk, d, dtype, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda n, h: (spread * torch.randn(B, n, h * d, generator=g, device="cuda")).to(dtype)  # noqa: E731
    return r(Nq, H), r(Nk, Hk), r(Nk, Hk), r(Nq, H)


def check(q, k, v, dy, H, window, sinks, ctxlen=None, q_start=None, scale=None):
    d = q.shape[2] // H
    Nq, Nk = q.shape[1], k.shape[1]
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    y = ncn.fused_window_attention(*leaves, H, window, n_sink=sinks, scale=scale, ctxlen=ctxlen, q_start=q_start)
    grads = torch.autograd.grad(y, leaves, dy)
    torch.cuda.synchronize()
    ops.device_status()
    want = O.attention(q, k, v, H, window if window else 1 << 40, sinks, scale or 1 / math.sqrt(d), Nk if ctxlen is None else ctxlen,
                       Nk - Nq if q_start is None else q_start, dy)
    O.close("y", y.detach(), want["y"])
    for name, g in zip(("dq", "dk", "dv"), grads):
        O.close(name, g, want[name])
    return y.detach(), grads


SHAPES = [  # B, N, H, Hk, d, window, sinks
    (1, 1, 1, 1, 64, 1, 0),
    (2, 1, 4, 2, 128, 5, 1),
    (1, 5, 2, 1, 64, 2, 1),
    (2, 127, 2, 2, 64, 16, 0),
    (1, 128, 2, 1, 128, 128, 4),
    (1, 129, 2, 2, 128, 129, 1),
    (1, 257, 4, 1, 128, 64, 3),
    (2, 300, 3, 3, 96, 100, 5),
    (1, 385, 2, 1, 32, 1, 0),
    (1, 640, 2, 2, 128, 200, 130),
    (1, 640, 4, 2, 64, 1, 300),
    (1, 1000, 2, 1, 128, None, 0),
    (1, 1000, 2, 1, 80, 333, 1),
    (1, 1300, 1, 1, 8, 128, 4),
    (3, 256, 4, 4, 32, 32, 0),
]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,N,H,Hk,d,window,sinks", SHAPES)
def test_training(dtype, B, N, H, Hk, d, window, sinks):
    q, k, v, dy = make(N + d, B, N, N, H, Hk, d, dtype)
    check(q, k, v, dy, H, window, sinks)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d", [1, 20, 33, 72, 136, 160, 256])
def test_other_head_sizes(dtype, d):
    q, k, v, dy = make(d, 2, 150, 150, 2, 1, d, dtype)
    check(q, k, v, dy, 2, 50, 2)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d", [40, 64, 128])
def test_large_scores_and_scale(dtype, d):
    q, k, v, dy = make(d + 1, 1, 400, 400, 2, 1, d, dtype, spread=3.0)
    check(q, k, v, dy, 2, 150, 2, scale=0.5)
    # the largest score grows along the row: the running maximum is followed
    grow = torch.linspace(0.1, 6, 400, device="cuda")[None, :, None].to(dtype)
    check(q, k * grow, v, dy, 2, None, 0)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d", [64, 128, 20])
@pytest.mark.parametrize("N,ctx", [(300, [300, 1, 0, 129]), (520, [400, 256, 128, 511]), (70, [70, 64, 63, 1000])])
def test_padded_rows_hold_anything(dtype, d, N, ctx):
    q, k, v, dy = make(N, 4, N, N, 4, 2, d, dtype)
    ctxlen = torch.tensor(ctx, device="cuda")
    for b, n in enumerate(ctx):
        for t, x in ((q, math.nan), (k, math.inf), (v, math.nan), (dy, -math.inf)):
            t[b, n:] = x
    y, (dq, dk, dv) = check(q, k, v, dy, 4, 90, 3, ctxlen=ctxlen)
    for b, n in enumerate(ctx):
        for t in (y, dq, dk, dv):
            assert (t[b, n:] == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d", [64, 128, 20])
@pytest.mark.parametrize("window", [300, 600, None])
def test_padding_behind_tiles_that_all_see(dtype, d, window):
    """Contexts that end inside a tile of queries whose other rows see whole tiles of keys."""
    ctx = [700, 390, 513, 640]
    q, k, v, dy = make(d, 4, 700, 700, 2, 1, d, dtype)
    y, grads = check(q, k, v, dy, 2, window, 2, ctxlen=torch.tensor(ctx))
    for b, n in enumerate(ctx):
        for t in (y, *grads):
            assert (t[b, n:] == 0).all()


def test_backward_first_in_a_new_thread():
    """The first CUDA call that a thread of the autograd engine makes may be a backward."""
    code = """
import torch, ncn_cuda_b200 as ncn
q, k, v = (torch.randn(1, 200, n * 64, device='cuda').bfloat16().requires_grad_(True) for n in (2, 1, 1))
y = ncn.fused_window_attention(q, k, v, 2, 50, n_sink=1)
y.backward(torch.ones_like(y))
torch.cuda.synchronize()
print('done', bool(torch.isfinite(q.grad).all()))
"""
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "done True" in out.stdout, out.stderr[-2000:]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d", [64, 128, 24])
def test_chunks_at_an_offset(dtype, d):
    q, k, v, dy = make(d, 4, 200, 500, 4, 2, d, dtype)
    check(q, k, v, dy, 4, 130, 4)                                             # the last 200 positions
    check(q, k, v, dy, 4, 130, 4, q_start=37)
    check(q, k, v, dy, 4, 130, 4, q_start=torch.tensor([0, 37, 299, 300], dtype=torch.int64))
    check(q, k, v, dy, 4, 130, 4, q_start=torch.tensor([-50, -200, 450, 1 << 30], device="cuda"),
          ctxlen=torch.tensor([500, 500, 480, 500], device="cuda"))           # rows that see nothing among them
    check(q, k, v, dy, 4, 10, 0, q_start=250, ctxlen=[500, 260, 250, 0])
    check(q[:, :150], k[:, :40], v[:, :40], dy[:, :150], 4, 7, 2)             # more queries than keys: positions below zero


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_views_of_a_joint_projection(dtype):
    g = torch.Generator(device="cuda").manual_seed(3)
    H, Hk, d, B, N = 4, 2, 64, 2, 333
    joint = torch.randn(B, N, (H + 2 * Hk) * d, generator=g, device="cuda").to(dtype)
    q, k, v = joint.split([H * d, Hk * d, Hk * d], -1)
    dy = torch.randn(B, N, H * d, generator=g, device="cuda").to(dtype)
    assert not q.is_contiguous()
    a = check(q, k, v, dy, H, 77, 2)
    b = check(q.contiguous(), k.contiguous(), v.contiguous(), dy, H, 77, 2)
    assert torch.equal(a[0], b[0])
    check(q.transpose(0, 1).contiguous().transpose(0, 1), k, v, dy.expand(B, N, H * d), H, 77, 2)
    # rows that no 16-byte access reaches, broadcast rows, features apart
    odd = torch.randn(B, N, (H + 2 * Hk) * d + 3, generator=g, device="cuda").to(dtype)[..., 3:]
    check(odd[..., : H * d], odd[..., H * d : (H + Hk) * d], odd[..., (H + Hk) * d :], dy, H, 77, 2)
    one = k[:1].expand(B, N, Hk * d)
    check(q, one, one, dy, H, 77, 2)
    apart = torch.randn(B, N, Hk * d, 2, generator=g, device="cuda").to(dtype)[..., 0]
    check(q, apart, v, dy[:, :1].expand(B, N, H * d), H, 77, 2)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_nothing_to_do(dtype):
    for B, Nq, Nk in ((0, 4, 4), (2, 0, 4), (2, 4, 0), (2, 0, 0)):
        q, k, v, dy = make(1, B, Nq, Nk, 2, 1, 64, dtype)
        leaves = [t.requires_grad_(True) for t in (q, k, v)]
        y = ncn.fused_window_attention(*leaves, 2, 3)
        assert y.shape == q.shape and (y == 0).all()
        for g, t in zip(torch.autograd.grad(y, leaves, dy), leaves):
            assert g.shape == t.shape and (g == 0).all()


def test_the_tensor_cores_are_reached():
    q, k, v, dy = make(1, 1, 256, 256, 2, 1, 128, BF16)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]

    def steps():  # (a profiler that has been in use for a minute may miss the first milliseconds)
        for _ in range(200):
            torch.autograd.grad(ncn.fused_window_attention(*leaves, 2, 64, n_sink=2), leaves, dy)

    _, names = kernels_of(steps)
    for part in ("attn_tensor_fwd", "attn_tensor_dq", "attn_tensor_dkv", "attn_sink_sum"):
        assert launched(names, part), (part, names)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_same_bits_again_and_on_another_stream(dtype):
    q, k, v, dy = make(2, 2, 700, 700, 4, 2, 64, dtype)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]

    def step():
        y = ncn.fused_window_attention(*leaves, 4, 100, n_sink=5)
        return (y, *torch.autograd.grad(y, leaves, dy))

    a, b = step(), step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for x, y, z in zip(a, b, c):
        assert torch.equal(x, y) and torch.equal(x, z)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_captured(dtype):
    q, k, v, dy = make(4, 2, 300, 300, 4, 2, 64, dtype)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    ctxlen = torch.tensor([300, 200], dtype=torch.int32, device="cuda")

    def step():
        y = ncn.fused_window_attention(*leaves, 4, 100, n_sink=5, ctxlen=ctxlen)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    other = make(5, 2, 300, 300, 4, 2, 64, dtype)
    with torch.no_grad():
        for t, x in zip((*leaves, dy), other):
            t.copy_(x)
        ctxlen.copy_(torch.tensor([150, 299], dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    for x, y in zip(out, step()):
        assert torch.equal(x, y)


def test_gradient_against_differences():
    q, k, v, dy = make(6, 1, 40, 40, 2, 1, 16, F32)
    _, grads = check(q, k, v, dy, 2, 9, 2)
    g = torch.Generator(device="cuda").manual_seed(8)
    for i, t in enumerate((q, k, v)):
        u = torch.randn(t.shape, generator=g, device="cuda")
        f = []
        for h in (1e-2, -1e-2):
            args = [q, k, v]
            args[i] = t + h * u
            f.append((ncn.fused_window_attention(*args, 2, 9, n_sink=2).double() * dy).sum())
        slope = float(f[0] - f[1]) / 2e-2
        want = float((grads[i].double() * u).sum())
        # third derivative: 1e-4 / 6 of a scale of the sums' size; rounding: 2^-24 of the output's terms over the step
        assert abs(slope - want) <= 1e-2 * float((grads[i].double().abs() * u.abs()).sum()), (i, slope, want)


def test_saved_tensors_are_guarded():
    q, k, v, dy = make(7, 1, 64, 64, 2, 2, 64, BF16)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    y = ncn.fused_window_attention(*leaves, 2, 9)
    y.backward(dy)
    with pytest.raises(RuntimeError, match="second time|already been freed"):
        y.backward(dy)
    y = ncn.fused_window_attention(*leaves, 2, 9)
    with torch.no_grad():
        leaves[1].add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(dy)


def test_function_form_agrees():
    """What the native node declines goes through the Python Function: the same kernels."""
    q, k, v, dy = make(9, 2, 130, 130, 2, 1, 64, BF16)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    ctxlen = torch.tensor([130, 77], device="cuda")
    args = (2, 20, 3, 0.125, ctxlen, None, 0)
    a = ncn.WindowAttentionFunction.apply(*leaves, *args)
    b = torch.autograd.Function.apply.__func__(ncn.WindowAttentionFunction, *leaves, *args)
    assert torch.equal(a, b)
    for x, y in zip(torch.autograd.grad(a, leaves, dy), torch.autograd.grad(b, leaves, dy)):
        assert torch.equal(x, y)


def test_far_offsets():
    """Rows more than 2^31 elements into a cache."""
    H, d, S, B = 1, 64, 1 << 20, 36
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    k = torch.zeros(B, S, d, dtype=BF16, device="cuda")
    v = torch.zeros(B, S, d, dtype=BF16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    k[-1, -300:] = torch.randn(300, d, generator=g, device="cuda").to(BF16)
    v[-1, -300:] = torch.randn(300, d, generator=g, device="cuda").to(BF16)
    q = torch.randn(B, 130, d, generator=g, device="cuda").to(BF16)
    y = ncn.fused_window_attention(q, k, v, H, 150)
    want = O.attention(q[-1:], k[-1:, -300:], v[-1:, -300:], H, 150, 0, 1 / 8, 300, 170)
    O.close("y", y[-1:], want["y"])
    last = ncn.window_attention_decode(q[:, -1:], k, v, torch.full((B,), S, device="cuda"), H, 150)
    O.close("decode", last[-1:], tuple(t[:, -1:] for t in want["y"]))


# ---------------------------------------------------------------- single tokens over a cache
def check_decode(q, k, v, H, window, sinks, ctxlen):
    d = q.shape[2] // H
    ctx = torch.as_tensor(ctxlen, device="cuda").clamp(0, k.shape[1])
    y = ncn.window_attention_decode(q, k, v, ctxlen, H, window, n_sink=sinks)
    torch.cuda.synchronize()
    want = O.attention(q, k, v, H, window if window else 1 << 40, sinks, 1 / math.sqrt(d), ctx, ctx - q.shape[1])
    O.close("y", y, want["y"])
    return y


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,Nq,S,H,Hk,d,window,sinks", [
    (1, 1, 1, 1, 1, 64, 1, 0), (1, 1, 4096, 32, 8, 128, 1024, 4), (3, 1, 500, 8, 8, 64, 100, 1), (2, 1, 300, 12, 1, 96, 64, 20),
    (2, 3, 700, 16, 2, 128, 200, 130), (2, 4, 64, 4, 4, 80, 1000, 0), (5, 2, 1000, 40, 2, 128, 17, 5), (1, 1, 20000, 4, 1, 64, None, 0),
    (2, 1, 257, 2, 1, 20, 31, 2), (2, 1, 257, 4, 2, 256, 31, 2), (2, 2, 257, 4, 2, 33, 31, 2), (300, 1, 40, 2, 2, 32, 8, 1),
])
def test_decode(dtype, B, Nq, S, H, Hk, d, window, sinks):
    q, k, v, _ = make(S + d, B, Nq, S, H, Hk, d, dtype)
    g = torch.Generator(device="cuda").manual_seed(2)
    ctxlen = torch.randint(1, S + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    ctxlen[0] = S
    check_decode(q, k, v, H, window, sinks, ctxlen)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d", [64, 128, 20])
def test_decode_reads_only_what_is_seen(dtype, d):
    H, window, sinks, S = 4, 50, 3, 400
    q, k, v, _ = make(d, 5, 1, S, H, 2, d, dtype)
    ctx = [400, 200, 52, 1, 0]
    for b, n in enumerate(ctx):
        for t, x in ((k, math.nan), (v, math.inf)):
            t[b, n:] = x
            t[b, min(sinks, n) : max(n - window, min(sinks, n))] = x
    y = check_decode(q, k, v, H, window, sinks, torch.tensor(ctx))
    assert (y[4] == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_decode_continues_training_form(dtype):
    q, k, v, _ = make(3, 2, 333, 333, 8, 2, 64, dtype)
    y = ncn.fused_window_attention(q, k, v, 8, 60, n_sink=4)
    for n in (1, 61, 64, 65, 200, 333):
        one = ncn.window_attention_decode(q[:, n - 1 : n], k, v, torch.full((2,), n), 8, 60, n_sink=4)
        want = O.attention(q[:, n - 1 : n], k, v, 8, 60, 4, 1 / 8, n, n - 1)["y"]
        O.close("decode", one, want)
        O.close("training form", y[:, n - 1 : n], want)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_ring_cache(dtype):
    H, Hk, d, window, sinks, N = 4, 2, 64, 48, 4, 130
    q, k, v, _ = make(11, 2, N, N, H, Hk, d, dtype)
    kc, vc = (torch.full((2, sinks + window, Hk * d), math.nan, dtype=dtype, device="cuda") for _ in range(2))
    for p in range(N):
        at = p if p < sinks else sinks + (p - sinks) % window
        kc[:, at], vc[:, at] = k[:, p], v[:, p]
        if p % 13 and p != N - 1:
            continue
        y = ncn.window_attention_decode(q[:, p : p + 1], kc, vc, torch.full((2,), min(p + 1, sinks + window)), H, None)
        O.close("y", y, O.attention(q[:, p : p + 1], k, v, H, window, sinks, 1 / 8, p + 1, p)["y"])


def test_decode_captured_and_strided():
    H, d, S = 8, 128, 1000
    q, k, v, _ = make(13, 4, 1, S, H, 2, d, BF16)
    cache = torch.randn(2, 4, S + 8, 2 * d, device="cuda").to(BF16)
    kc, vc = cache[0][:, :S], cache[1][:, 8:]
    ctxlen = torch.tensor([1000, 10, 500, 0], dtype=torch.int32, device="cuda")
    check_decode(q, kc, vc, H, 300, 4, ctxlen)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ncn.window_attention_decode(q, kc, vc, ctxlen, H, 300, n_sink=4)
    ctxlen.copy_(torch.tensor([900, 11, 0, 1], dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, check_decode(q, kc, vc, H, 300, 4, ctxlen))


@pytest.mark.parametrize("d", [24, 50, 64, 100, 128])
def test_fp32_features_of_all_sizes(d):
    """fp32 heads of 17 to 128 features go through products of two parts each: small features beside large ones keep their bits."""
    q, k, v, dy = make(d, 1, 200, 200, 2, 1, d, F32)
    g = torch.Generator(device="cuda").manual_seed(d)
    e = torch.randint(-30, 31, (2, 1, 1, d), generator=g, device="cuda").float()
    q, dy = q * torch.exp2(e[0]).repeat(1, 1, 2), dy * torch.exp2(-e[1]).repeat(1, 1, 2)
    k, v = k * torch.exp2(-e[0]), v * torch.exp2(e[1])
    check(q, k, v, dy, 2, 60, 3)


def test_fp32_many_sinks_and_chunks():
    q, k, v, dy = make(8, 2, 700, 1500, 4, 2, 40, F32)
    check(q, k, v, dy, 4, 30, 900, ctxlen=torch.tensor([1500, 1033], device="cuda"))


# ---------------------------------------------------------------- refusals, and calls side by side
@pytest.mark.parametrize("dtype,d", [(F32, 16), (BF16, 64), (BF16, 12)])
def test_many_sinks(dtype, d):
    """More tiles of sinks than the far queries are cut for: fewer pieces each."""
    q, k, v, dy = make(d, 1, 4000, 4000, 1, 1, d, dtype)
    check(q, k, v, dy, 1, 8, 3500)


@pytest.mark.parametrize("native", [True, False])
def test_no_second_derivative(native):
    q, k, v, dy = make(3, 1, 40, 40, 2, 1, 32, F32)
    freqs, _ = ncn.rotary_frequencies(32, device="cuda")
    q, k, v, dy = (t.requires_grad_(True) for t in (q, k, v, dy))

    def apply(f, *args):
        return f.apply(*args) if native else torch.autograd.Function.apply.__func__(f, *args)

    y = apply(ncn.WindowAttentionFunction, q, k, v, 2, 9, 1, 0.2, None, None, 0)
    r, _ = apply(ncn.RotaryFunction, q, k, None, None, freqs, None, 2, 0, False, 0.0, 1.0)
    w = torch.ones(32, device="cuda", requires_grad=True)
    n, _ = apply(ncn.RotaryFunction, q, k, w, w, freqs, None, 2, 0, False, 1e-6, 1.0)
    for out in (y, r, n) if native else (y, n):  # (of a rotation the gradient does not depend on what was turned)
        g, = torch.autograd.grad(out, q, dy, create_graph=True)
        for loss in (g.sum(), g.sum() + (q * q).sum()):
            with pytest.raises(RuntimeError, match="derivative of its own"):
                torch.autograd.grad(loss, q, retain_graph=True)


def test_lengths_beyond_32_bits():
    """A length that means "no limit" stays one; lengths are whole numbers."""
    q, k, v, dy = make(5, 2, 70, 70, 2, 1, 64, BF16)
    whole = ncn.fused_window_attention(q, k, v, 2, 9)
    for most in (2**31 - 1, 2**32, 2**40, 2**63 - 1):
        ctxlen = torch.full((2,), most, device="cuda")
        assert torch.equal(whole, ncn.fused_window_attention(q, k, v, 2, 9, ctxlen=ctxlen, q_start=0))
        assert torch.equal(whole, ops.window_fwd(q, k, v, 2, 9, 0, 0.125, 0, ctxlen=ctxlen)[0])
        last = ncn.window_attention_decode(q[:, -1:], k, v, ctxlen, 2, 9)
        assert torch.equal(last, ncn.window_attention_decode(q[:, -1:], k, v, torch.tensor([70, 70]), 2, 9))
        assert not ncn.fused_window_attention(q, k, v, 2, 9, q_start=ctxlen).any()
        assert not ncn.fused_window_attention(q, k, v, 2, 9, ctxlen=-ctxlen).any()
    for bad in (torch.tensor([3.0, 4.0]), torch.tensor([True, False])):
        for call in (lambda: ncn.fused_window_attention(q, k, v, 2, 9, ctxlen=bad), lambda: ncn.fused_window_attention(q, k, v, 2, 9, q_start=bad),
                     lambda: ncn.window_attention_decode(q[:, :1], k, v, bad, 2, 9), lambda: ops.window_fwd(q, k, v, 2, 9, 0, 1.0, 0, ctxlen=bad)):
            with pytest.raises(TypeError, match="whole numbers"):
                call()


def test_refusals_on_the_device():
    q, k, v, _ = make(1, 2, 8, 8, 4, 2, 32, BF16)
    freqs, _ = ncn.rotary_frequencies(32, device="cuda")
    half = q.half()
    for call in (lambda: ncn.fused_window_attention(half, half, half, 4, 3), lambda: ncn.fused_rotary(half, half, freqs, 4),
                 lambda: ncn.window_attention_decode(half, half, half, [1, 1], 4, 3)):
        with pytest.raises(TypeError, match="float32 or bfloat16"):
            call()
    for bad in ((q, k.float(), v), (q, k, v[:, :5]), (q, k[:1], v[:1]), (q[0], k, v), (q, k[..., :40], v[..., :40])):
        with pytest.raises(ValueError):
            ncn.fused_window_attention(*bad, 4, 3)
        with pytest.raises(ValueError):
            ncn.window_attention_decode(*bad, torch.tensor([1, 1]), 4, 3)
    with pytest.raises(ValueError, match="n_head"):
        ncn.fused_window_attention(q, k, v, 3, 3)
    with pytest.raises(ValueError, match="ctxlen has 3"):
        ncn.fused_window_attention(q, k, v, 4, 3, ctxlen=[1, 2, 3])
    with pytest.raises(ValueError, match="q_start has 1"):
        ncn.fused_window_attention(q, k, v, 4, 3, q_start=torch.tensor([1]))
    with pytest.raises(ValueError, match="positions"):
        ncn.fused_rotary(q, k, freqs, 4, positions=torch.arange(7))
    with pytest.raises(TypeError, match="whole numbers"):
        ncn.fused_rotary(q, k, freqs, 4, positions=torch.arange(8).float())
    with pytest.raises(ValueError, match="freqs"):
        ncn.fused_rotary(q, k, torch.ones(17, device="cuda"), 4)
    with pytest.raises(ValueError, match="weight has"):
        ncn.fused_qk_norm_rotary(q, k, torch.ones(31, device="cuda"), torch.ones(32, device="cuda"), freqs, 4)
    wide = torch.zeros(1, 4, 2 * 264, device="cuda")
    with pytest.raises(ncn._lib.NCNError, match="bad shape"):
        ncn.fused_window_attention(wide, wide, wide, 2, 3)
    # heads of the queries that the heads of the keys do not divide
    with pytest.raises(ncn._lib.NCNError, match="bad shape"):
        ncn.fused_window_attention(torch.zeros(1, 4, 96, device="cuda"), torch.zeros(1, 4, 64, device="cuda"), torch.zeros(1, 4, 64, device="cuda"), 3, 3)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_calls_at_once_on_two_streams(dtype):
    """Workspaces, results and saved states belong to a call."""
    sets = [make(20 + i, 1, 1500, 1500, 4, 2, 128, dtype) for i in range(2)]
    sets = [([t.requires_grad_(True) for t in s[:3]], s[3]) for s in sets]

    def step(i):
        leaves, dy = sets[i]
        y = ncn.fused_window_attention(*leaves, 4, 300, n_sink=40)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    alone = [step(i) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = step(i)
    torch.cuda.synchronize()
    for a, b in zip(alone, got):
        for x, y in zip(a, b):
            assert torch.equal(x, y)


def test_gradients_of_shared_and_broadcast_inputs():
    """The same tensor as keys and values, and one row of keys broadcast over the batch."""
    q, k, _, dy = make(30, 3, 100, 100, 2, 1, 64, BF16)
    both = k.clone().requires_grad_(True)
    y = ncn.fused_window_attention(q, both, both, 2, 30)
    g, = torch.autograd.grad(y, both, dy)
    want = O.attention(q, k, k, 2, 30, 0, 1 / 8, 100, 0, dy)
    value, bound = (a + b for a, b in zip(want["dk"], want["dv"]))
    O.close("d both", g, (value, bound + 2.0**-8 * (value.abs() + bound)))  # (the sum is rounded once more)
    row = k[:1].clone().requires_grad_(True)
    y = ncn.fused_window_attention(q, row.expand(3, 100, 64), k, 2, 30)
    g, = torch.autograd.grad(y, row, dy)
    want = O.attention(q, row.expand(3, 100, 64), k, 2, 30, 0, 1 / 8, 100, 0, dy)["dk"]
    value, bound = want[0].sum(0, keepdim=True), want[1].sum(0, keepdim=True)
    O.close("d row", g, (value, bound + 2.0**-8 * (value.abs() + bound)))
