"""Decaying and sliding-window attention without a GPU: refusals of the C entry points and of the tensor-level calls, layers' arguments."""
import ctypes as C

import pytest
import torch


class Decay(C.Structure):
    _fields_ = ([(n, C.c_void_p) for n in ("q", "k", "v")] + [(n, C.c_int64) for n in ("q_t", "q_b", "q_h", "k_t", "k_b", "k_h", "v_t", "v_b", "v_h")]
                + [("log_decay", C.c_void_p)] + [(n, C.c_int64) for n in ("g_t", "g_b", "g_h")] + [("s_in", C.c_void_p), ("mask", C.c_void_p), ("T", C.c_int64)]
                + [(n, C.c_int) for n in ("B", "H", "K", "D", "dtype", "decay_dtype", "per_head")] + [("scale", C.c_float)])


class Window(C.Structure):
    _fields_ = ([(n, C.c_void_p) for n in ("q", "k", "v")] + [(n, C.c_int64) for n in ("q_t", "q_b", "q_h", "k_t", "k_b", "k_h", "v_t", "v_b", "v_h")]
                + [("mask", C.c_void_p), ("T", C.c_int64)] + [(n, C.c_int) for n in ("B", "H", "G", "D", "dtype", "window", "sinks")] + [("scale", C.c_float)])


def decay(**kw):
    return Decay(**{**dict(q=16, k=16, v=16, log_decay=16, T=4, B=2, H=2, K=16, D=16, dtype=0, decay_dtype=1, scale=1.0), **kw})


def window(**kw):
    return Window(**{**dict(q=16, k=16, v=16, T=4, B=2, H=2, G=1, D=16, dtype=0, window=3, sinks=1, scale=1.0), **kw})


@pytest.mark.parametrize("kw,code", [(dict(q=None), -1), (dict(log_decay=None), -1), (dict(T=0), -1), (dict(K=-1), -1), (dict(dtype=7), -3), (dict(decay_dtype=9), -3),
                                     (dict(K=257), -3), (dict(D=300), -3), (dict(T=2 ** 31), -3), (dict(B=70000), -3), (dict(B=60000, H=60000), -3), (dict(s_in=8), -2)])
def test_decay_refusals(kw, code):
    from rfa_b200 import _lib
    lib, c = _lib.load(), decay(**kw)
    assert lib.rfa_decay_fwd(C.byref(c), 16, None, None, None, 0, None) == code
    assert lib.rfa_decay_bwd(C.byref(c), 16, None, None, 16, 16, 16, None, None, 16, 1 << 40, None) == code
    assert lib.rfa_decay_step(C.byref(c), 16, 16, None) == code


def test_decay_refusals_of_buffers():
    from rfa_b200 import _lib
    lib = _lib.load()
    c = decay()
    assert lib.rfa_decay_fwd(None, 16, None, None, None, 0, None) == -1
    assert lib.rfa_decay_fwd(C.byref(c), None, None, None, None, 0, None) == -1
    assert lib.rfa_decay_fwd(C.byref(c), 16, 8, None, None, 0, None) == -2
    assert lib.rfa_decay_step(C.byref(c), 16, 16, None) == -1                                   # four tokens
    assert lib.rfa_decay_step(C.byref(decay(T=1)), 16, 8, None) == -2
    assert lib.rfa_decay_bwd(C.byref(c), 16, None, None, 16, 16, 16, None, None, 16, 0, None) == -4   # no workspace
    assert lib.rfa_decay_bwd(C.byref(c), None, None, None, 16, 16, 16, None, None, 16, 1 << 40, None) == -1
    long = decay(T=100000, B=1, H=1)
    need = lib.rfa_decay_workspace_bytes(100000, 1, 1, 16, 16, 0, 0)
    assert need > 0 and need == lib.rfa_decay_workspace_bytes(100000, 1, 1, 16, 16, 0, 0)
    assert lib.rfa_decay_fwd(C.byref(long), 16, None, None, 16, need - 1, None) == -4
    assert lib.rfa_decay_workspace_bytes(0, 1, 1, 16, 16, 0, 0) == 0


@pytest.mark.parametrize("kw,code", [(dict(k=None), -1), (dict(T=0), -1), (dict(G=0), -1), (dict(dtype=5), -3), (dict(H=3, G=2), -3), (dict(D=257), -3), (dict(window=0), -3),
                                     (dict(sinks=-1), -3), (dict(window=2 ** 30, sinks=0), -3), (dict(window=2 ** 30 - 1, sinks=2 ** 30 - 1), -3), (dict(T=2 ** 30), -3),
                                     (dict(B=70000), -3)])
def test_window_refusals(kw, code):
    from rfa_b200 import _lib
    lib, c = _lib.load(), window(**kw)
    assert lib.rfa_window_fwd(C.byref(c), 16, None, 16, 1 << 40, None) == code
    assert lib.rfa_window_bwd(C.byref(c), 16, 16, 16, 16, 16, 16, 16, 1 << 40, None) == code
    assert lib.rfa_window_append(C.byref(c), 16, 16, 16, 0, 16, 16, 1 << 40, None) == code


def test_window_refusals_of_buffers():
    from rfa_b200 import _lib
    lib, c = _lib.load(), window()
    assert lib.rfa_window_fwd(C.byref(c), None, None, 16, 1 << 40, None) == -1
    assert lib.rfa_window_fwd(C.byref(c), 16, 8, 16, 1 << 40, None) == -2
    assert lib.rfa_window_fwd(C.byref(c), 16, None, None, 0, None) == -4
    assert lib.rfa_window_bwd(C.byref(c), 16, None, 16, 16, 16, 16, 16, 1 << 40, None) == -1
    assert lib.rfa_window_bwd(C.byref(c), 16, 16, 16, 16, 16, 16, 16, 8, None) == -4
    assert lib.rfa_window_append(C.byref(c), 16, None, 16, 0, 16, 16, 1 << 40, None) == -1
    assert lib.rfa_window_append(C.byref(c), 8, 16, 16, 0, 16, 16, 1 << 40, None) == -2
    assert lib.rfa_window_append(C.byref(c), 16, 16, 16, 0, 16, None, 0, None) == -4
    assert lib.rfa_window_append_workspace_bytes(1, 2, 2, 1, 16, 0, 3, 1, 0) == 0


def test_cpu_tensors_are_refused():
    from rfa_b200.decay_attention import decay_attention, incremental_decay_attention
    from rfa_b200.window_attention import incremental_window_attention, window_attention
    q, g = torch.zeros(4, 2, 2, 16).half(), torch.zeros(2)
    for f in (decay_attention, incremental_decay_attention):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            f(q=q, k=q, v=q, log_decay=g)
    for f in (window_attention, incremental_window_attention):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            f(q=q, k=q, v=q, window=3)


def test_layers_refuse_what_the_operators_would():
    from rfa_b200 import DecayAttention, WindowAttention
    for kw in (dict(num_heads=3), dict(num_heads=2, decay="none"), dict(num_heads=1, key_dim=300, head_dim=8)):
        with pytest.raises(AssertionError):
            DecayAttention(embed_dim=64, **kw)
    for kw in (dict(num_heads=3, window=2), dict(num_heads=4, window=0), dict(num_heads=4, num_kv_heads=3, window=2), dict(num_heads=4, window=2, sinks=-1),
               dict(num_heads=1, window=2, head_dim=257)):
        with pytest.raises(AssertionError):
            WindowAttention(embed_dim=64, **kw)
    layer = WindowAttention(embed_dim=64, num_heads=4, num_kv_heads=2, window=8, sinks=2)
    state = dict(prev_k=torch.arange(3.).view(3, 1, 1, 1), prev_len=torch.tensor([4, 5, 6]))
    layer.reorder_incremental_state(state, torch.tensor([2, 0, 0]))
    assert state["prev_len"].tolist() == [6, 4, 4] and state["prev_k"].flatten().tolist() == [2.0, 0.0, 0.0]


def test_fixed_decays_stay_fp32():
    """Of a layer that becomes 16 bits, is copied, moved, or loaded."""
    import copy
    from rfa_b200 import DecayAttention
    layer = DecayAttention(embed_dim=64, num_heads=4, decay="head")
    want = torch.log1p(-torch.exp2(-5.0 - 8.0 * torch.arange(4) / 4))
    for f in (lambda m: m.half(), lambda m: m.bfloat16(), lambda m: copy.deepcopy(m).half(), lambda m: m.to(torch.device("cpu"), torch.float16), lambda m: m.double(),
              lambda m: torch.nn.Sequential(m).bfloat16()[0], lambda m: m.float()):
        other = f(layer)
        assert other.log_decay.dtype == torch.float32 and torch.equal(other.log_decay, want)
        assert "log_decay" in dict(other.named_buffers()) and torch.equal(other.state_dict()["log_decay"], want)
    layer.half()
    layer.log_decay.fill_(-0.3)                  # a value of the user's own
    layer.bfloat16()
    assert layer.in_proj.weight.dtype == torch.bfloat16 and torch.equal(layer.log_decay, torch.full((4,), -0.3))
    fresh = DecayAttention(embed_dim=64, num_heads=4, decay="head").half()
    fresh.load_state_dict(layer.state_dict())
    assert torch.equal(fresh.log_decay, torch.full((4,), -0.3))
    meta = DecayAttention(embed_dim=64, num_heads=4, decay="head").to("meta").half().to_empty(device="cpu")
    assert meta.log_decay.dtype == torch.float32 and meta.in_proj.weight.dtype == torch.float16
    DecayAttention(embed_dim=64, num_heads=4).half()
