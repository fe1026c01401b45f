"""Attention next to the NCN layers: norms of queries and keys with rotary positions, a sliding window with sink tokens, and its
form over a cache for single tokens.

An NCN stage mixes fixed groups of positions by a recurrence; a local attention layer mixes what a window holds by content.
Both take [B, N, E] activations whose features are cut into n_head heads, a context length per batch row for padded batches, and
fp32 or bf16 storage.  Keys and values may have fewer heads than the queries (their features are a smaller multiple of the head
size).  No counterpart in the reference.

In training a layer calls fused_qk_norm_rotary (or fused_rotary) and then fused_window_attention; in serving the rotated keys go
into a cache and window_attention_decode reads it.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch
from torch import nn

from . import _lib, ops

SCALINGS = (None, "linear", "ntk", "yarn")


def rotary_frequencies(rot_dim: int, base: float = 10000.0, scaling: Optional[str] = None, factor: float = 1.0,
                       trained_length: int = 4096, fast_turns: float = 32.0, slow_turns: float = 1.0,
                       device=None) -> Tuple[torch.Tensor, float]:
    """-> (frequencies, magnitude): radians per position of the rot_dim / 2 pairs, base^(-2 i / rot_dim), as a float64 tensor, and
    what the rotated features are multiplied by.  For contexts `factor` times as long as trained_length:

    "linear"  every frequency divided by factor
    "ntk"     a larger base, so that the slowest pair is slowed down by factor and the fastest not at all
    "yarn"    pairs that turn more than fast_turns times within trained_length keep their frequency, those below slow_turns are
              divided by factor, a linear ramp between; magnitude 0.1 ln(factor) + 1 (the scores are sharpened by its square)

    A program makes these once and keeps them."""
    if rot_dim < 0 or rot_dim % 2:
        raise ValueError(f"rot_dim must be even, got {rot_dim}")
    if scaling not in SCALINGS:
        raise ValueError(f"unknown scaling {scaling!r}: one of {SCALINGS}")
    if not (factor >= 1.0 and base > 0 and trained_length > 0 and fast_turns > slow_turns):
        raise ValueError("factor >= 1, base > 0, trained_length > 0 and fast_turns > slow_turns are needed")
    i = torch.arange(0, rot_dim, 2, dtype=torch.float64, device="cpu")
    magnitude = 1.0
    if scaling == "ntk":
        base = base * factor ** (rot_dim / max(rot_dim - 2, 1))
    f = base ** (-i / max(rot_dim, 1))
    if scaling == "linear":
        f = f / factor
    elif scaling == "yarn":
        turns = trained_length * f / (2 * math.pi)
        keep = ((turns - slow_turns) / (fast_turns - slow_turns)).clamp(0, 1)
        f = f * keep + f / factor * (1 - keep)
        magnitude = 0.1 * math.log(factor) + 1.0
    return (f if device is None else f.to(device=device)), magnitude


class _Once(torch.autograd.Function):
    """Gradients that have no derivative of their own: one that is asked for is an error, not a silent zero."""

    @staticmethod
    def forward(ctx, n, *tensors):
        return tensors[:n]

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("the gradient of an attention operator has no derivative of its own")


def _once(grads, *inputs):
    grads = tuple(grads)
    if not torch.is_grad_enabled():
        return grads
    have = [g for g in grads if g is not None]
    done = iter(_Once.apply(len(have), *have, *(t for t in inputs if t is not None)))
    return tuple(None if g is None else next(done) for g in grads)


class RotaryFunction(torch.autograd.Function):
    """Rotation of queries and keys, with the norm of every head where weights are given.  `apply` goes to the native node of
    csrc/attn_torch.cpp; forward and backward stand for the calls that the node declines."""

    @classmethod
    def apply(cls, *args):
        if cls is not RotaryFunction:
            return super().apply(*args)
        q, k, wq, wk, freqs, positions, n_head, start, interleaved, eps, magnitude = args
        out = _lib.native().rotary(q, k, wq, wk, freqs, positions, n_head, start, interleaved, eps, magnitude)
        return super().apply(*args) if out is None else out

    @staticmethod
    def forward(ctx, q, k, wq, wk, freqs, positions, n_head, start, interleaved, eps, magnitude):
        ctx.cfg = (n_head, start, interleaved, eps, magnitude)
        ctx.norm = wq is not None
        ctx.save_for_backward(q if ctx.norm else None, k if ctx.norm else None, wq, wk, freqs, positions)
        ctx.has_k = k is not None
        return ops.qk_rotary(q, k, wq, wk, freqs, positions, *ctx.cfg)

    @staticmethod
    def backward(ctx, dq, dk):
        q, k, wq, wk, freqs, positions = ctx.saved_tensors
        if not ctx.norm:
            dx = ops.qk_rotary(dq, dk if ctx.has_k else None, None, None, freqs, positions, *ctx.cfg, inverse=True)
            return (*_once(dx, dq, dk), None, None, None, None, None, None, None, None, None)
        gq, gk, dwq, dwk = ops.qk_norm_rotary_bwd(q, k, wq, wk, freqs, positions, dq, dk if ctx.has_k else None, *ctx.cfg)
        dwq = dwq.to(wq.dtype).reshape(wq.shape)
        dwk = None if dwk is None else dwk.to(wk.dtype).reshape(wk.shape)
        return (*_once((gq, gk, dwq, dwk), q, k, wq, wk, dq, dk), None, None, None, None, None, None, None)


def _positions(positions):
    """-> (tensor or None, first position)"""
    if positions is None:
        return None, 0
    if isinstance(positions, int):
        return None, positions
    return torch.as_tensor(positions), 0


def fused_rotary(q, k, freqs, n_head, positions=None, interleaved=False, magnitude=1.0):
    """q [B, N, E] and k [B, N, Ek] (or None) with the first 2 * len(freqs) features of every head turned by their positions; returns both.
    freqs: from rotary_frequencies.  positions: None (0, 1, ...), the first position as an int, or whole numbers [N] or [B, N].
    Pair i of a head: features i and i + len(freqs), or 2 i and 2 i + 1 with interleaved=True.  Differentiable in q and k."""
    pos, start = _positions(positions)
    return RotaryFunction.apply(q, k, None, None, freqs, pos, n_head, start, interleaved, 0.0, magnitude)


def fused_qk_norm_rotary(q, k, wq, wk, freqs, n_head, positions=None, interleaved=False, magnitude=1.0, eps=1e-6):
    """fused_rotary of the normalised queries and keys: every head of q is divided by its root mean square (eps under the root) and
    multiplied by wq [E / n_head], k likewise by wk, in the pass that turns them.  freqs of length 0: norms alone.
    Differentiable in q, k, wq and wk."""
    if wq is None:
        raise ValueError("fused_qk_norm_rotary needs weights; fused_rotary turns without a norm")
    pos, start = _positions(positions)
    return RotaryFunction.apply(q, k, wq, wk, freqs, pos, n_head, start, interleaved, eps, magnitude)


class WindowAttentionFunction(torch.autograd.Function):
    """Windowed attention; `apply` goes to the native node, as in RotaryFunction."""

    @classmethod
    def apply(cls, *args):
        if cls is not WindowAttentionFunction:
            return super().apply(*args)
        out = _lib.native().window(*args)
        return super().apply(*args) if out is None else out

    @staticmethod
    def forward(ctx, q, k, v, n_head, window, n_sink, scale, ctxlen, q_start, start):
        ctx.cfg = (n_head, window, n_sink, scale, start)
        y, state = ops.window_fwd(q, k, v, *ctx.cfg, ctxlen=ctxlen, q_start=q_start, want_state=True)
        ctx.save_for_backward(q, k, v, y, state, ctxlen, q_start)
        return y

    @staticmethod
    def backward(ctx, dy):
        q, k, v, y, state, ctxlen, q_start = ctx.saved_tensors
        dq, dk, dv = ops.window_bwd(q, k, v, y, dy, state, *ctx.cfg, ctxlen=ctxlen, q_start=q_start)
        return (*_once((dq, dk, dv), q, k, v, dy), None, None, None, None, None, None, None)


class WindowDecodeFunction(torch.autograd.Function):
    """Windowed attention over a cache; `apply` goes to the native form, as in RotaryFunction.  It has no gradient: the Function is there
    for calls that are traced, and refuses transforms and forward gradients as any custom Function does."""

    @classmethod
    def apply(cls, *args):
        if cls is not WindowDecodeFunction:
            return super().apply(*args)
        out = _lib.native().window_decode(*args)
        return super().apply(*args) if out is None else out

    @staticmethod
    def forward(ctx, q, k_cache, v_cache, ctxlen, n_head, window, n_sink, scale):
        return ops.window_decode(q, k_cache, v_cache, ctxlen, n_head, window, n_sink, scale)

    @staticmethod
    def backward(ctx, dy):
        raise RuntimeError("window_attention_decode has no gradient: use fused_window_attention")


def _window(window, n_sink, scale, q, n_head):
    window = ops.NO_WINDOW if window is None else int(window)
    if window < 1 or n_sink < 0:
        raise ValueError(f"window must be at least 1 and n_sink at least 0, got {window} and {n_sink}")
    if scale is None:
        scale = 1.0 / math.sqrt(max(q.shape[-1] // max(n_head, 1), 1))
    if not (math.isfinite(scale) and scale > 0):
        raise ValueError(f"scale must be positive, got {scale}")
    return window, float(scale)


def fused_window_attention(q, k, v, n_head, window, n_sink=0, scale=None, ctxlen=None, q_start=None):
    """Causal attention in which a query sees the last `window` positions up to its own, and the first n_sink.

    q [B, Nq, E], k and v [B, Nk, Ek] -> [B, Nq, E].  window None: all positions before.  scale: 1 / sqrt(E / n_head) unless given.
    ctxlen (int tensor [B], None: Nk): the keys of each row that count; queries at or behind it are padding and give zeros.
    q_start: the position of the first query, an int or an int tensor [B]; None: Nk - Nq, so that the last query is at the last key (a
    chunk of a prompt behind a cache; 0 where both have one length).  Differentiable in q, k and v."""
    window, scale = _window(window, n_sink, scale, q, n_head)
    if ctxlen is not None:
        ctxlen = torch.as_tensor(ctxlen)
    start = 0
    if q_start is None:
        start = k.shape[1] - q.shape[1]
    elif isinstance(q_start, int):
        start, q_start = q_start, None
    else:
        q_start = torch.as_tensor(q_start)
    return WindowAttentionFunction.apply(q, k, v, n_head, window, n_sink, scale, ctxlen, q_start, start)


def window_attention_decode(q, k_cache, v_cache, ctxlen, n_head, window, n_sink=0, scale=None):
    """fused_window_attention of the last Nq positions of each row, for serving: q [B, Nq, E] (Nq = 1: one new token, already in the
    cache), k_cache and v_cache [B, S, Ek], ctxlen int tensor [B] with the new tokens counted.  Reads only the visible keys.
    No gradient.

    A ring cache (sinks in the first n_sink places, position p at n_sink + (p - n_sink) % window) holds just what one new token
    sees, in an order that does not matter: call with window=None and ctxlen = the number of places in use."""
    window, scale = _window(window, n_sink, scale, q, n_head)
    if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k_cache, v_cache)):
        raise RuntimeError("window_attention_decode has no gradient: use fused_window_attention, or torch.no_grad()")
    return WindowDecodeFunction.apply(q, k_cache, v_cache, torch.as_tensor(ctxlen), n_head, window, n_sink, scale)


class NCNWindowAttention(nn.Module):
    """A local attention layer to stand between NCN layers: [B, N, embed_dim] -> [B, N, embed_dim].

    One projection to queries, keys and values, the norm of every head of queries and keys (qk_norm) with the rotation of its first
    rot_dim features (None: all of them, 0: none), windowed attention with sinks, a projection back.  n_kv_head: heads of
    keys and values (None: n_head).  base, scaling, factor, trained_length: as in rotary_frequencies.

    forward(x, ctxlen=None) is the training form.  For serving, new_cache(B, length) and step(x, cache, ctxlen)."""

    def __init__(self, embed_dim, n_head, window, n_sink=0, n_kv_head=None, rot_dim=None, base=10000.0, scaling=None, factor=1.0,
                 trained_length=4096, interleaved=False, qk_norm=True, eps=1e-6):
        super().__init__()
        n_kv_head = n_head if n_kv_head is None else n_kv_head
        if n_head < 1 or n_kv_head < 1 or embed_dim % n_head or n_head % n_kv_head:
            raise ValueError(f"n_head = {n_head} must divide embed_dim = {embed_dim}, and n_kv_head = {n_kv_head} n_head")
        self.embed_dim, self.n_head, self.n_kv_head = embed_dim, n_head, n_kv_head
        self.window, self.n_sink, self.interleaved, self.eps = window, n_sink, interleaved, eps
        d = embed_dim // n_head
        self.qkv = nn.Linear(embed_dim, (n_head + 2 * n_kv_head) * d, bias=False)
        self.out = nn.Linear(embed_dim, embed_dim, bias=False)
        self.q_weight = nn.Parameter(torch.ones(d)) if qk_norm else None
        self.k_weight = nn.Parameter(torch.ones(d)) if qk_norm else None
        freqs, self.magnitude = rotary_frequencies(d if rot_dim is None else rot_dim, base, scaling, factor, trained_length)
        self.freqs = freqs if self.qkv.weight.is_meta else freqs.to(self.qkv.weight.device)

    def _apply(self, fn, *args, **kwargs):
        # the frequencies go where the weights go, and stay in 64 bits whatever the weights' type becomes
        super()._apply(fn, *args, **kwargs)
        if not self.qkv.weight.is_meta:
            self.freqs = self.freqs.to(self.qkv.weight.device)
        return self

    def _rotated(self, x, positions):
        d = self.embed_dim // self.n_head
        q, k, v = self.qkv(x).split([self.embed_dim, self.n_kv_head * d, self.n_kv_head * d], -1)
        if self.q_weight is None:
            q, k = fused_rotary(q, k, self.freqs, self.n_head, positions, self.interleaved, self.magnitude)
        else:
            q, k = fused_qk_norm_rotary(q, k, self.q_weight, self.k_weight, self.freqs, self.n_head, positions, self.interleaved,
                                        self.magnitude, self.eps)
        return q, k, v

    def forward(self, x, ctxlen=None):
        q, k, v = self._rotated(x, None)
        return self.out(fused_window_attention(q, k, v, self.n_head, self.window, n_sink=self.n_sink, ctxlen=ctxlen))

    def new_cache(self, B: int, length: int, dtype: Optional[torch.dtype] = None):
        """Keys and values of B rows of up to `length` positions, in `dtype`: unless given, autocast's where it is on, else the weights'.
        (The place behind them takes what has none.)"""
        w = self.qkv.weight
        if dtype is None:
            kind = w.device.type
            cast = torch.amp.is_autocast_available(kind) and torch.is_autocast_enabled(kind)
            dtype = torch.get_autocast_dtype(kind) if cast else w.dtype
        width = self.n_kv_head * (self.embed_dim // self.n_head)
        return tuple(torch.zeros(B, length + 1, width, dtype=dtype, device=w.device) for _ in range(2))

    @torch.no_grad()
    def step(self, x, cache, ctxlen):
        """The next positions of each row: x [B, n, embed_dim], ctxlen int tensor [B], the rows' lengths with these n counted.  Enters their
        keys and values into the cache, in whose type the attention is computed, and returns [B, n, embed_dim].  Rows shorter than n are
        padded in front: what stands there is not entered and gives out(0).  So do positions beyond the cache's length, which are lost: make it long enough."""
        k_cache, v_cache = cache
        B, n, _ = x.shape
        length = k_cache.shape[1] - 1
        ctxlen = torch.as_tensor(ctxlen).to(device=x.device, dtype=torch.int64)
        positions = ctxlen[:, None] - n + torch.arange(n, device=x.device)
        q, k, v = self._rotated(x, positions)
        dtype = q.dtype
        q, k, v = (t.to(k_cache.dtype) for t in (q, k, v))
        place = torch.where((positions < 0) | (positions >= length), length, positions)
        rows = torch.arange(B, device=x.device)[:, None]
        k_cache[rows, place] = k
        v_cache[rows, place] = v
        k_cache, v_cache = k_cache[:, :length], v_cache[:, :length]
        if n == 1:  # (a row whose position has no place sees nothing, as in the other form)
            ctxlen = torch.where(ctxlen > length, 0, ctxlen)
            y = window_attention_decode(q, k_cache, v_cache, ctxlen, self.n_head, self.window, n_sink=self.n_sink)
        else:
            y = fused_window_attention(q, k_cache, v_cache, self.n_head, self.window, n_sink=self.n_sink, ctxlen=ctxlen, q_start=ctxlen - n)
        return self.out(y.to(dtype))
