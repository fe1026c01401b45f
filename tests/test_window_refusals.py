"""Attention operators, without a device: what they refuse, the frequencies' scalings, the layer's arguments."""
import ctypes
import math

import pytest
import torch

import ncn_cuda_b200 as ncn
from ncn_cuda_b200 import _lib, ops

OK, SHAPE, DTYPE, NULL, UNSUPPORTED, WORKSPACE = 0, 1, 2, 8, 5, 6
P = 1 << 20  # (stands for a pointer: every call here is refused, or has nothing to do, before one is read)


def fwd(q=P, k=P, v=P, y=P, B=1, Nq=8, Nk=8, E=64, Ek=64, H=2, window=4, sinks=0, start=0, scale=1.0, dtype=0):
    return _lib.load().ncn_window_fwd(q, k, v, y, None, None, None, None, B, Nq, Nk, E, Ek, H, window, sinks, start, scale, dtype, None)


def bwd(state=P, ws=P, nbytes=1 << 40, B=1, Nq=8, dq=P, dk=P):
    return _lib.load().ncn_window_bwd(P, P, P, P, P, state, dq, dk, P, None, None, None, ws, nbytes, B, Nq, 8, 64, 64, 2, 4, 0, 0, 1.0, 0, None)


def decode(ctxlen=P, H=2, dtype=1, B=1):
    return _lib.load().ncn_window_decode(P, P, P, P, ctxlen, None, B, 1, 8, 64, 32, H, 4, 0, 1.0, dtype, None)


def rotary(q=P, k=P, wq=None, wk=None, freqs=P, B=1, N=4, E=64, Ek=64, H=2, R=32, eps=1e-6, magnitude=1.0, inverse=0, dtype=0):
    return _lib.load().ncn_qk_rotary(q, k, wq, wk, freqs, None, 0, 0, P, P, None, B, N, E, Ek, H, R, 0, eps, magnitude, inverse, dtype, None)


@pytest.mark.parametrize("status,args", [
    (DTYPE, {"dtype": 2}), (SHAPE, {"B": -1}), (SHAPE, {"Nq": -1}), (SHAPE, {"Nk": -1}), (SHAPE, {"H": 0}), (SHAPE, {"H": 3}), (SHAPE, {"E": 0}),
    (SHAPE, {"Ek": 48}), (SHAPE, {"E": 192, "Ek": 128, "H": 3}), (SHAPE, {"E": 1024, "Ek": 512}), (SHAPE, {"window": 0}), (SHAPE, {"sinks": -1}),
    (SHAPE, {"scale": 0.0}), (SHAPE, {"scale": -1.0}), (SHAPE, {"scale": math.nan}), (SHAPE, {"scale": math.inf}), (SHAPE, {"Nq": 1 << 29}),
    (SHAPE, {"Nk": 1 << 29}), (NULL, {"q": None}), (NULL, {"k": None}), (NULL, {"y": None}), (OK, {"B": 0}), (OK, {"Nq": 0}), (10, {"B": 1 << 30}),
])
def test_forward_refuses(status, args):
    assert fwd(**args) == status


@pytest.mark.parametrize("status,args", [(NULL, {"state": None}), (NULL, {"dq": None}), (NULL, {"dk": None}), (OK, {"B": 0}), (OK, {"Nq": 0})])
def test_backward_refuses(status, args):
    assert bwd(**args) == status


@pytest.mark.parametrize("off", [1, 4, 8])
def test_states_and_workspaces_off_the_boundary(off):
    """What bulk copies and 16-byte accesses read has to lie on 16 bytes: a status, not a fault."""
    ALIGN = 3
    assert bwd(ws=P + off) == ALIGN and bwd(state=P + off) == ALIGN
    assert _lib.load().ncn_window_fwd(P, P, P, P, P + off, None, None, None, 1, 8, 8, 64, 64, 2, 4, 0, 0, 1.0, 0, None) == ALIGN


def test_decode_refuses():
    assert decode(ctxlen=None) == NULL
    assert decode(H=5) == SHAPE
    assert decode(dtype=7) == DTYPE
    assert decode(B=0) == OK
    assert _lib.load().ncn_window_decode(P, P, P, P, P, None, 1 << 30, 1, 8, 64, 64, 2, 4, 0, 1.0, 1, None) == 10  # two heads of 2^30 rows
    assert _lib.load().ncn_window_decode(P, P, P, P, P, None, 1, 1 << 28, 8, 512, 64, 8, 4, 0, 1.0, 1, None) == 10  # 2^31 rows share keys


@pytest.mark.parametrize("status,args", [
    (DTYPE, {"dtype": 3}), (SHAPE, {"H": 3}), (SHAPE, {"R": 31}), (SHAPE, {"R": 34}), (SHAPE, {"R": -2}), (SHAPE, {"Ek": 40}), (SHAPE, {"E": 2048}),
    (SHAPE, {"eps": -1.0}), (SHAPE, {"eps": math.nan}), (SHAPE, {"magnitude": math.inf}), (SHAPE, {"B": -1}), (NULL, {"q": None}), (NULL, {"k": None}),
    (NULL, {"freqs": None}), (NULL, {"wq": P}), (NULL, {"wk": P}), (UNSUPPORTED, {"wq": P, "wk": P, "inverse": 1}), (OK, {"B": 0}), (OK, {"N": 0}),
])
def test_rotary_refuses(status, args):
    assert rotary(**args) == status


def test_sizes_of_buffers():
    lib = _lib.load()
    assert lib.ncn_window_state_bytes(2, 130, 64, 4, 0) == 2 * 4 * 256 * 4
    assert lib.ncn_window_state_bytes(2, 130, 64, 4, 1) == 2 * 4 * 256 * 4 + 2 * 130 * 64 * 2
    assert lib.ncn_window_state_bytes(0, 130, 64, 4, 1) == 0 and lib.ncn_window_state_bytes(1, 0, 64, 4, 1) == 0
    assert lib.ncn_window_bwd_workspace_bytes(2, 130, 130, 256, 64, 4, 200, 5, 1) == 2 * 4 * 256 * 4      # no query is beyond the window
    assert lib.ncn_window_bwd_workspace_bytes(2, 130, 130, 256, 64, 4, 16, 0, 1) == 2 * 4 * 256 * 4       # no sinks
    assert lib.ncn_window_bwd_workspace_bytes(2, 130, 130, 256, 64, 4, 16, 5, 1) > 2 * 4 * 256 * 4
    assert lib.ncn_window_bwd_workspace_bytes(2, 130, 130, 256, 100, 4, 16, 5, 1) == 0
    # many sinks: in proportion to dk and dv in fp32 (2 x 2 of them and 256 pieces of 128 x 128), not to their pieces times the tiles
    assert lib.ncn_window_bwd_workspace_bytes(1, 131072, 131072, 128, 128, 1, 1024, 65536, 1) <= (4 * 131072 + 2 * 256 * 128 + 131072) * 128 * 4
    assert lib.ncn_qk_norm_rotary_workspace_bytes(2, 3, 64, 4) == 2 * 3 * 4 * 2 * 16 * 4
    assert lib.ncn_qk_norm_rotary_workspace_bytes(1 << 20, 1 << 20, 64, 4) == 8192 * 2 * 16 * 4


def test_python_refuses():
    q = torch.randn(1, 4, 64)
    freqs, _ = ncn.rotary_frequencies(32)
    for call in (lambda: ncn.fused_window_attention(q, q, q, 2, 3), lambda: ncn.window_attention_decode(q, q, q, [4], 2, 3),
                 lambda: ncn.fused_rotary(q, q, freqs, 2), lambda: ops.window_fwd(q, q, q, 2, 3, 0, 1.0, 0),
                 lambda: ops.qk_rotary(q, q, None, None, freqs, None, 2, 0, False, 0.0, 1.0)):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            call()
    with pytest.raises(ValueError, match="window"):
        ncn.fused_window_attention(q, q, q, 2, 0)
    with pytest.raises(ValueError, match="n_sink"):
        ncn.fused_window_attention(q, q, q, 2, 3, n_sink=-1)
    with pytest.raises(ValueError, match="scale"):
        ncn.fused_window_attention(q, q, q, 2, 3, scale=-0.5)
    with pytest.raises(ValueError, match="weights"):
        ncn.fused_qk_norm_rotary(q, q, None, None, freqs, 2)
    with pytest.raises(RuntimeError, match="no gradient"):
        ncn.window_attention_decode(q.clone().requires_grad_(True), q, q, [4], 2, 3)


def test_operators_are_autograd_functions():
    for f in (ncn.WindowAttentionFunction, ncn.RotaryFunction):
        assert issubclass(f, torch.autograd.Function) and {"forward", "backward"} <= set(vars(f))


def test_frequencies():
    f, m = ncn.rotary_frequencies(64)
    assert f.dtype == torch.float64 and f.shape == (32,) and m == 1.0
    want = [10000.0 ** (-2 * i / 64) for i in range(32)]
    assert torch.allclose(f, torch.tensor(want, dtype=torch.float64), rtol=1e-15)
    lin, _ = ncn.rotary_frequencies(64, scaling="linear", factor=4.0)
    assert torch.equal(lin, f / 4)
    ntk, _ = ncn.rotary_frequencies(64, scaling="ntk", factor=4.0)
    assert ntk[0] == f[0] and math.isclose(ntk[-1] * 4, f[-1], rel_tol=1e-12) and (ntk[1:] < f[1:]).all()
    yarn, m = ncn.rotary_frequencies(64, scaling="yarn", factor=4.0, trained_length=2048)
    turns = 2048 * f / (2 * math.pi)
    assert torch.equal(yarn[turns > 32], f[turns > 32]) and torch.allclose(yarn[turns < 1], f[turns < 1] / 4, rtol=1e-15)
    assert ((yarn <= f) & (yarn >= f / 4)).all() and math.isclose(m, 0.1 * math.log(4) + 1)
    assert ncn.rotary_frequencies(0)[0].shape == (0,)
    for bad in ({"rot_dim": 3}, {"rot_dim": -2}, {"rot_dim": 8, "scaling": "other"}, {"rot_dim": 8, "factor": 0.5}, {"rot_dim": 8, "base": 0.0}):
        with pytest.raises(ValueError):
            ncn.rotary_frequencies(**bad)


def test_layer_arguments():
    for bad in ({"embed_dim": 65, "n_head": 2}, {"embed_dim": 64, "n_head": 4, "n_kv_head": 3}, {"embed_dim": 64, "n_head": 0}):
        with pytest.raises(ValueError):
            ncn.NCNWindowAttention(window=8, **bad)
    layer = ncn.NCNWindowAttention(64, 4, 8, n_kv_head=2, rot_dim=8)
    assert sorted(layer.state_dict()) == ["k_weight", "out.weight", "q_weight", "qkv.weight"]
    assert layer.qkv.weight.shape == (128, 64)
    layer.to(torch.bfloat16)
    assert layer.qkv.weight.dtype == torch.bfloat16 and layer.freqs.dtype == torch.float64 and layer.freqs.shape == (4,)
    assert ctypes.sizeof(ctypes.c_int64) == 8
    with torch.device("meta"):
        layer = ncn.NCNWindowAttention(64, 4, 8)
    assert layer.qkv.weight.is_meta and layer.freqs.device.type == "cpu"
    assert layer.to_empty(device="cpu").freqs.dtype == torch.float64


def test_types_of_a_cache():
    layer = ncn.NCNWindowAttention(64, 4, 8, n_kv_head=2)
    assert [t.dtype for t in layer.new_cache(2, 5)] == [torch.float32] * 2 and layer.new_cache(2, 5)[0].shape == (2, 6, 32)
    assert [t.dtype for t in layer.new_cache(2, 5, dtype=torch.bfloat16)] == [torch.bfloat16] * 2
    with torch.autocast("cpu", torch.bfloat16):
        assert [t.dtype for t in layer.new_cache(2, 5)] == [torch.bfloat16] * 2
        assert layer.new_cache(2, 5, dtype=torch.float32)[0].dtype == torch.float32
    cache = ncn.NCNWindowAttention(64, 4, 8).to("meta").new_cache(2, 5)  # (a device without autocast)
    assert cache[0].is_meta and cache[0].dtype == torch.float32
