"""Attention operators at the edges of what they take: traced and transformed calls, scores that overflow, places that nobody sees, views
off the 16-byte grid, mixed precision, many rows."""
import math
import re

import pytest
import torch

import ncn_cuda_b200 as ncn
from ncn_cuda_b200 import ops
from tests import window_oracle as O
from tests.kernels_util import kernels_of, launched

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def make(seed, B, Nq, Nk, H, Hk, d, dtype):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda n, h: torch.randn(B, n, h * d, generator=g, device="cuda").to(dtype)  # noqa: E731
    return r(Nq, H), r(Nk, Hk), r(Nk, Hk), r(Nq, H)


# ---------------------------------------------------------------- calls that are traced or transformed
def _call(kind):
    """-> a call of tensors alone, and its tensors"""
    q, k, v, _ = make(1, 2, 40, 40, 2, 1, 32, F32)
    freqs, _ = ncn.rotary_frequencies(32, device="cuda")
    lengths = torch.tensor([40, 21], device="cuda")
    w = torch.ones(32, device="cuda")
    if kind == "window":
        return lambda a, b, c: ncn.fused_window_attention(a, b, c, 2, 9, n_sink=1, ctxlen=lengths), [q, k, v]
    if kind == "rotary":
        return lambda a, b: ncn.fused_rotary(a, b, freqs, 2), [q, k]
    if kind == "norm_rotary":
        return lambda a, b, c, e: ncn.fused_qk_norm_rotary(a, b, c, e, freqs, 2, positions=3), [q, k, w, w]
    return lambda a, b, c: ncn.window_attention_decode(a, b, c, lengths, 2, 9, n_sink=1), [q[:, :2].contiguous(), k, v]


@pytest.mark.parametrize("kind", ["window", "rotary", "norm_rotary", "decode"])
def test_a_traced_call_computes(kind):
    call, args = _call(kind)
    with torch.no_grad():
        traced = torch.jit.trace(call, tuple(args), check_trace=False)
        other = [a.flip(1) if a.dim() == 3 else 2 * a for a in args]
        got, want = traced(*other), call(*other)
    for p, q in zip(got if isinstance(got, tuple) else (got,), want if isinstance(want, tuple) else (want,)):
        assert torch.equal(p, q)


def test_a_traced_step_computes():
    torch.manual_seed(1)
    layer = ncn.NCNWindowAttention(64, 2, 9, n_sink=1, n_kv_head=1).cuda().requires_grad_(False)
    x, other = torch.randn(2, 2, 1, 64, device="cuda")
    lengths = torch.tensor([1, 1], device="cuda")

    def step(x, k, v):
        return layer.step(x, (k, v), lengths)

    traced = torch.jit.trace(step, (x, *layer.new_cache(2, 8)), check_trace=False)
    assert torch.equal(traced(other, *layer.new_cache(2, 8)), step(other, *layer.new_cache(2, 8)))


@pytest.mark.parametrize("kind", ["window", "rotary", "norm_rotary", "decode"])
def test_transforms_are_refused(kind):
    """No forward-mode rule and no vmap rule: a dual tensor or a functorch transform is an error, never a lost tangent."""
    import torch.autograd.forward_ad as fwAD

    call, args = _call(kind)
    for i in range(len(args)):
        with fwAD.dual_level(), pytest.raises(NotImplementedError, match="jvp"):
            call(*[fwAD.make_dual(t, torch.ones_like(t)) if i == k else t for k, t in enumerate(args)])
    with pytest.raises(RuntimeError, match="setup_context"):
        torch.func.vmap(lambda a: call(a, *args[1:]))(torch.stack([args[0], args[0]]))
    with torch.no_grad():  # with the level left, the same tensors are taken
        call(*args)


def test_the_function_form_refuses_what_the_node_refuses():
    q, k, _, _ = make(1, 2, 8, 8, 2, 1, 32, F32)
    freqs, _ = ncn.rotary_frequencies(32, device="cuda")
    apply = torch.autograd.Function.apply.__func__
    with pytest.raises(TypeError, match="whole numbers"):
        apply(ncn.RotaryFunction, q, k, None, None, freqs, torch.arange(8).float(), 2, 0, False, 0.0, 1.0)
    with pytest.raises(ValueError, match="weights"):
        apply(ncn.RotaryFunction, q, k, torch.ones(32, device="cuda"), None, freqs, None, 2, 0, False, 0.0, 1.0)


def test_function_form_of_decode_agrees():
    for dtype, d in ((BF16, 64), (F32, 40), (BF16, 20)):
        q, k, v, _ = make(9, 3, 2, 130, 4, 1, d, dtype)
        args = (torch.tensor([130, 77, 0], device="cuda"), 4, 20, 3, 0.125)
        a = ncn.WindowDecodeFunction.apply(q, k, v, *args)
        b = torch.autograd.Function.apply.__func__(ncn.WindowDecodeFunction, q, k, v, *args)
        assert torch.equal(a, b)
    y = ncn.WindowDecodeFunction.apply(q.requires_grad_(True), k, v, *args)
    with pytest.raises(RuntimeError, match="no gradient"):
        y.sum().backward()
    with pytest.raises(TypeError, match="whole numbers"):
        ops.window_decode(q, k, v, torch.tensor([1.0, 2.0, 3.0]), 4, 20, 3, 0.125)
    with pytest.raises(ValueError, match="ctxlen has 2"):
        ops.window_decode(q, k, v, torch.tensor([1, 2]), 4, 20, 3, 0.125)


# ---------------------------------------------------------------- scores of minus infinity
BIG = 2.0**66  # BIG * -BIG overflows in 32 bits

FORMS = [(BF16, 64), (BF16, 128), (BF16, 20), (BF16, 160), (F32, 64), (F32, 16), (F32, 160)]


def overflowing(dtype, d, N, sinks):
    """The scores of keys 0 .. sinks - 1 overflow to minus infinity for every query; their values are large."""
    q, k, v, dy = make(d, 2, N, N, 2, 1, d, dtype)
    q[..., ::d], k[..., 0] = BIG, 0.0
    k[:, :sinks, 0] = -BIG
    v[:, :sinks] = 1e35
    return q, k, v, dy


@pytest.mark.parametrize("dtype,d", FORMS)
def test_scores_of_minus_infinity_weigh_nothing(dtype, d):
    """Sinks whose scores are minus infinity: a query that sees other keys too is answered from these alone, one that sees none gets
    what the formula gives, NaN.  (Sinks in places 0 and 1, so that past the window the answer is the one without sinks.)"""
    N, window, sinks = 300, 60, 2
    q, k, v, dy = overflowing(dtype, d, N, sinks)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    y = ncn.fused_window_attention(*leaves, 2, window, n_sink=sinks)
    want = O.attention(q, k, v, 2, window, 0, 1 / math.sqrt(d), N, 0, dy)
    far = window + sinks
    O.close("y", y.detach()[:, far:], tuple(t[:, far:] for t in want["y"]))
    assert y[:, :sinks].isnan().all() and y[:, sinks:].isfinite().all()
    dq, dk, dv = torch.autograd.grad(y, leaves, dy)
    O.close("dq", dq[:, far:], tuple(t[:, far:] for t in want["dq"]))
    assert dq[:, :sinks].isnan().all()
    # keys that no row of NaN sees
    assert dk[:, sinks:].isfinite().all() and dv[:, sinks:].isfinite().all()


@pytest.mark.parametrize("dtype,d", FORMS)
def test_decode_with_scores_of_minus_infinity(dtype, d):
    N, window, sinks = 300, 60, 2
    q, k, v, _ = overflowing(dtype, d, N, sinks)
    one = q[:, :1]
    y = ncn.window_attention_decode(one, k, v, torch.tensor([N, 2]), 2, window, n_sink=sinks)
    want = O.attention(one, k, v, 2, window, 0, 1 / math.sqrt(d), N, N - 1)["y"]
    O.close("y", y[:1], tuple(t[:1] for t in want))
    assert y[1].isnan().all()
    y = ncn.window_attention_decode(q[:, :2], k, v, torch.tensor([1, 0]), 2, window, n_sink=sinks)
    assert (y[0, 0] == 0).all() and y[0, 1].isnan().all() and (y[1] == 0).all()  # a position below zero; one key; none


# ---------------------------------------------------------------- places that no query of the call sees
@pytest.mark.parametrize("dtype,d", FORMS + [(F32, 128)])
@pytest.mark.parametrize("Nq,Nk,lo,window,sinks", [
    (40, 700, 300, 90, 3),      # before the window, between it and the sinks, behind the last query
    (1, 300, 299, 7, 1), (130, 700, 520, 300, 0), (5, 64, 20, 10, 4), (200, 900, 600, 128, 130), (129, 1000, 700, 1, 257), (3, 400, 140, 200, 300),
])
def test_unseen_places_hold_anything(dtype, d, Nq, Nk, lo, window, sinks):
    q, k, v, dy = make(Nk + d, 3, Nq, Nk, 4, 2, d, dtype)
    starts = torch.tensor([lo, max(lo - 37, 0), 0], device="cuda")
    ctxlen = torch.tensor([Nk, Nk, min(Nk, Nq + 2)], device="cuda")
    see = O.visible(3, Nq, Nk, window, sinks, ctxlen, starts, "cuda").any(-2)[:, 0]
    assert not see.all()
    k[~see], v[~see] = math.nan, math.inf
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    y = ncn.fused_window_attention(*leaves, 4, window, n_sink=sinks, ctxlen=ctxlen, q_start=starts)
    grads = torch.autograd.grad(y, leaves, dy)
    torch.cuda.synchronize()
    ops.device_status()
    want = O.attention(q, k, v, 4, window, sinks, 1 / math.sqrt(d), ctxlen, starts, dy)
    O.close("y", y.detach(), want["y"])
    for name, g in zip(("dq", "dk", "dv"), grads):
        O.close(name, g, want[name])
    assert (grads[1][~see] == 0).all() and (grads[2][~see] == 0).all()
    # one start for all rows, no lengths
    see = O.visible(3, Nq, Nk, window, sinks, Nk, lo, "cuda").any(-2)[:, 0]
    k, v = torch.randn_like(k), torch.randn_like(v)
    k[~see], v[~see] = -math.inf, math.nan
    y = ncn.fused_window_attention(q, k, v, 4, window, n_sink=sinks, q_start=lo)
    O.close("y", y, O.attention(q, k, v, 4, window, sinks, 1 / math.sqrt(d), Nk, lo)["y"])


# ---------------------------------------------------------------- views off the 16-byte grid
def taken(call):
    """Bytes that a call takes beyond its result"""
    call()  # (whatever the first call of its kind takes)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    base = torch.cuda.memory_allocated()
    y = call()
    return torch.cuda.max_memory_allocated() - base - y.numel() * y.element_size()


@pytest.mark.parametrize("dtype,d,extra", [(F32, 9, 0), (BF16, 20, 0), (BF16, 36, 0), (F32, 64, 1), (BF16, 64, 3), (BF16, 128, 2)])
def test_decode_takes_no_copy_of_a_cache(dtype, d, extra):
    """A slice of a longer cache, of an odd width or at an odd place of a joint cache, is read where it lies."""
    B, S = 3, 5000
    q, _, _, _ = make(d, B, 1, 1, 3, 1, d, dtype)
    g = torch.Generator(device="cuda").manual_seed(d)
    joint = torch.randn(B, S + 1, 2 * d + extra, generator=g, device="cuda").to(dtype)
    k, v = joint[:, :S, extra : d + extra], joint[:, :S, d + extra :]
    if not extra:
        k, v = (t.contiguous()[:, :S] for t in (joint[..., :d], joint[..., d:]))
    ctxlen = torch.tensor([S, 2000, 1], dtype=torch.int32, device="cuda")
    call = lambda: ncn.window_attention_decode(q, k, v, ctxlen, 3, 100, n_sink=2)  # noqa: E731
    O.close("y", call(), O.attention(q, k, v, 3, 100, 2, 1 / math.sqrt(d), ctxlen, ctxlen - 1)["y"])
    assert taken(call) < 16384 < k.numel() * k.element_size()


@pytest.mark.parametrize("dtype,d", [(F32, 9), (BF16, 20), (F32, 33)])
def test_no_copy_where_it_would_not_help(dtype, d):
    """Rows of an odd width have no 16-byte boundaries in a copy either."""
    B, S = 2, 6000
    cache = torch.randn(2, B, S + 1, d, device="cuda").to(dtype)
    q, _, _, _ = make(d, B, 4, 1, 3, 1, d, dtype)
    k, v = cache[0][:, :S], cache[1][:, :S]
    call = lambda: ncn.fused_window_attention(q, k, v, 3, 100, n_sink=2)  # noqa: E731
    O.close("y", call(), O.attention(q, k, v, 3, 100, 2, 1 / math.sqrt(d), S, S - 4)["y"])
    assert taken(call) < 16384 < k.numel() * k.element_size()


# ---------------------------------------------------------------- the layer
@pytest.mark.parametrize("dtype", ["default", F32, BF16])
def test_layer_under_autocast(dtype):
    """fp32 weights, bf16 arithmetic: forward, and step by step over a cache of either type."""
    torch.manual_seed(4)
    B, N, E, H = 2, 50, 128, 2
    layer = ncn.NCNWindowAttention(E, H, 20, n_sink=2, n_kv_head=1).cuda()
    x = torch.randn(B, N, E, device="cuda")
    with torch.autocast("cuda", torch.bfloat16), torch.no_grad():
        y = layer(x)
        cache = layer.new_cache(B, N) if dtype == "default" else layer.new_cache(B, N, dtype=dtype)
        assert cache[0].dtype == (BF16 if dtype == "default" else dtype)
        got = [layer.step(x[:, :20], cache, torch.full((B,), 20))]
        got += [layer.step(x[:, n : n + 1], cache, torch.full((B,), n + 1)) for n in range(20, N)]
    assert y.dtype == BF16 and all(t.dtype == BF16 for t in got)
    # roundings of the projection, the rotated heads, the inner result and the last one, on both sides: 8 * 2^-8 of the largest
    assert (torch.cat(got, 1) - y).abs().max() <= 8 * 2.0**-8 * y.abs().max()
    assert layer.new_cache(B, N)[0].dtype == F32  # (without autocast: the weights' type)
    assert layer.new_cache(B, N, dtype=BF16)[1].dtype == BF16


def test_layer_beyond_its_cache():
    """A position that has no place in the cache is lost, and gives out(0), whether it comes alone or with others."""
    torch.manual_seed(5)
    layer = ncn.NCNWindowAttention(64, 2, 20).cuda()
    x = torch.randn(2, 10, 64, device="cuda")
    cache = layer.new_cache(2, 8)
    y = layer(x)
    first = layer.step(x[:, :6], cache, torch.tensor([6, 6]))
    two = layer.step(x[:, 6:8], cache, torch.tensor([8, 8]))
    assert (torch.cat([first, two], 1) - y[:, :8]).abs().max() <= 1e-5 * y.abs().max() + 6 * 64 * 2.0**-24 * y.abs().max()
    kept = [t[:, :8].clone() for t in cache]
    for n in (1, 2):
        got = layer.step(x[:, 8 : 8 + n], cache, torch.tensor([8 + n, 8 + n]))
        assert (got == 0).all(), n
    assert all(torch.equal(a, b[:, :8]) for a, b in zip(kept, cache))


# ---------------------------------------------------------------- many rows
def test_more_queries_than_decode_takes():
    """Forward and backward have a CTA per tile of queries, and are not bound by what the form for single tokens would launch."""
    H, d, Nq, Nk = 128, 8, 1 << 21, 64
    if torch.cuda.mem_get_info()[0] < 48 << 30:
        pytest.skip("needs 48 GB")
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v, first, dy = (torch.randn(1, Nk, n * d, generator=g, device="cuda").to(BF16) for n in (1, 1, H, H))
    wide = lambda t: torch.cat([t, t.new_zeros(1, Nq - Nk, H * d)], 1)  # noqa: E731
    leaves = [t.requires_grad_(True) for t in (wide(first), k, v)]
    y = ncn.fused_window_attention(*leaves, H, 9, q_start=0)
    want = O.attention(first, k, v, H, 9, 0, 1 / math.sqrt(d), Nk, 0, dy)
    O.close("y", y.detach()[:, :Nk], want["y"])
    assert not y[:, Nk:].any()
    dq, dk, dv = torch.autograd.grad(y, leaves, wide(dy))
    O.close("dq", dq[:, :Nk], want["dq"])
    assert not dq[:, Nk:].any()
    O.close("dk", dk, want["dk"])
    O.close("dv", dv, want["dv"])


# ---------------------------------------------------------------- kernels by name
@pytest.mark.parametrize("kind,dtype,d,wanted", [
    ("train", F32, 64, ("attn_split_fwd_kernel<64", "attn_split_dq_kernel<64", "attn_split_dkv_kernel<64", "attn_sink_sum_kernel<float")),
    ("train", BF16, 64, ("attn_tensor_fwd_kernel<64", "attn_tensor_dq_kernel<64", "attn_tensor_dkv_kernel<64")),
    ("train", BF16, 160, ("attn_simt_fwd_kernel", "attn_simt_dq_kernel", "attn_simt_dkv_kernel")),
    ("decode", BF16, 128, ("attn_decode_kernel<128, 1>",)), ("decode", BF16, 64, ("attn_decode_kernel<64, 1>",)), ("decode", F32, 64, ("attn_decode_any_kernel<float",)),
    ("norm", BF16, 128, ("rotary_kernel<__nv_bfloat16, 8, 1>", "rotary_kernel<__nv_bfloat16, 8, 2>")), ("norm", F32, 96, ("rotary_kernel<float, 8, 1>", "rotary_kernel<float, 8, 2>")),
    ("turn", BF16, 64, ("rotary_kernel<__nv_bfloat16, 4, 0>",)), ("turn", F32, 40, ("rotary_any_kernel<float",)),
])
def test_the_kernels_are_reached(kind, dtype, d, wanted):
    q, k, v, dy = make(1, 2, 200, 200, 4, 2, d, dtype)
    freqs, _ = ncn.rotary_frequencies(d, device="cuda")
    lengths = torch.tensor([200, 90], dtype=torch.int32, device="cuda")
    w = torch.ones(d, device="cuda", requires_grad=True)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]

    def call():
        if kind == "train":
            return torch.autograd.grad(ncn.fused_window_attention(*leaves, 4, 50, n_sink=2), leaves, dy)
        if kind == "decode":
            with torch.no_grad():
                return ncn.window_attention_decode(q[:, :1], k, v, lengths, 4, 50, n_sink=2)
        if kind == "norm":
            y = ncn.fused_qk_norm_rotary(q, k, w, w, freqs, 4)
        else:
            y = ncn.fused_rotary(q, k, freqs, 4)
        return torch.autograd.grad(y, leaves[:2], (dy, dy[..., : k.shape[2]]))

    _, names = kernels_of(call)
    for part in wanted:
        assert launched(names, re.escape(part)), (part, sorted(names))
