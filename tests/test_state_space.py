"""The state-space operators without a GPU: their oracle against autograd and differences, what the calls and the C ABI refuse."""
import ctypes as C

import pytest
import torch

from oracle import state_space_oracle as O
from rfa_b200 import SelectiveStateSpace, _lib, ops
from rfa_b200 import state_space as ss


def rand(*shape, seed=0, scale=1.0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed + sum(shape)), dtype=torch.float64) * scale


MASK = torch.tensor([[0, 0, 1, 0, 1], [1, 1, 0, 0, 0], [1, 1, 1, 1, 1]], dtype=torch.bool)


class Oracle(torch.autograd.Function):
    """An oracle's results with its own gradients, so that differences can be taken of them."""

    @staticmethod
    def forward(ctx, call, names, grads, given, *inputs):
        ctx.save_for_backward(*inputs)
        ctx.args = call, grads, given
        out = call(*inputs)
        return tuple(out[n] for n in names)

    @staticmethod
    def backward(ctx, *gs):
        call, grads, given = ctx.args
        out = call(*ctx.saved_tensors, **dict(zip(given, gs)))
        return (None, None, None, None, *(out[n] for n in grads))


@pytest.mark.parametrize("mask", [None, MASK])
@pytest.mark.parametrize("silu", [True, False])
def test_convolution_oracle(mask, silu):
    x, w, b, s = rand(5, 3, 4), rand(4, 3, seed=1), rand(4, seed=2), rand(3, 2, 4, seed=3)
    call = lambda x, w, b, s, **k: O.conv(x, w, b, s, mask, silu, **k)
    ins = [t.requires_grad_() for t in (x, w, b, s)]
    run = lambda *i: Oracle.apply(call, ("y", "state"), ("gx", "gweight", "gbias", "gstate"), ("g", "g_state"), *i)
    assert torch.autograd.gradcheck(run, ins)
    if mask is None:
        seq = torch.cat([s.transpose(0, 1), x]).permute(1, 2, 0)
        y = torch.nn.functional.conv1d(seq, w.unsqueeze(1), b, groups=4).permute(2, 0, 1)
        assert torch.allclose(run(*ins)[0], torch.nn.functional.silu(y) if silu else y)


@pytest.mark.parametrize("mask", [None, MASK])
@pytest.mark.parametrize("softplus", [True, False])
def test_scan_oracle(mask, softplus):
    T, B, D, N, G = 5, 3, 4, 3, 2
    ins = [rand(T, B, D), rand(T, B, D, seed=1, scale=0.3), -rand(D, N, seed=2).abs(), rand(T, B, G, N, seed=3), rand(T, B, G, N, seed=4), rand(D, seed=5),
           rand(D, seed=6, scale=0.3), rand(B, D, N, seed=7)]
    call = lambda *i, **k: O.scan(*i, mask, softplus, **k)
    run = lambda *i: Oracle.apply(call, ("y", "s"), ("gx", "gdt", "ga", "gb", "gc", "gd", "gbias", "gs"), ("g", "g_s"), *i)
    assert torch.autograd.gradcheck(run, [t.requires_grad_() for t in ins])


@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("silu", [True, False])
def test_norm_oracle(gated, silu):
    x, w, b, z = rand(3, 2, 6), rand(6, seed=1), rand(6, seed=2), rand(3, 2, 6, seed=3)
    call = lambda *i, **k: O.norm(i[0], 2, i[1], i[2], i[3] if gated else None, silu, 1e-5, **k)
    grads = ("gx", "gweight", "gbias", "ggate")[:4 if gated else 3]
    ins = [t.requires_grad_() for t in (x, w, b, z)[:4 if gated else 3]]
    run = lambda *i: Oracle.apply(call, ("y",), grads, ("g",), *i)
    assert torch.autograd.gradcheck(run, ins)
    n = torch.nn.functional.group_norm(x.reshape(6, 6), 2, w, b, 1e-5).view_as(x)
    act = torch.nn.functional.silu if silu else (lambda t: t)
    assert torch.allclose(run(*ins)[0], n * act(z) if gated else act(n))


def test_cpu_tensors_and_wrong_arguments_are_refused():
    x, w = torch.zeros(4, 2, 8), torch.zeros(8, 4)
    bc, a = torch.zeros(4, 2, 1, 3), torch.zeros(8, 3)
    for call in (lambda: ss.causal_conv(x=x, weight=w), lambda: ss.incremental_causal_conv(x=x, weight=w),
                 lambda: ss.selective_scan(x=x, dt=x, a=a, b=bc, c=bc), lambda: ss.incremental_selective_scan(x=x, dt=x, a=a, b=bc, c=bc),
                 lambda: ss.group_norm(x=x, num_groups=2), lambda: SelectiveStateSpace(embed_dim=8)(x)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()
    with pytest.raises(ValueError, match="activation"):
        ss.causal_conv(x=x, weight=w, activation="relu")
    with pytest.raises(AssertionError, match="norm_groups"):
        SelectiveStateSpace(embed_dim=8, norm_groups=3)


class Conv(C.Structure):
    _fields_ = [("x", C.c_void_p), ("x_t", C.c_int64), ("x_b", C.c_int64), ("weight", C.c_void_p), ("bias", C.c_void_p), ("state_in", C.c_void_p),
                ("mask", C.c_void_p), ("T", C.c_int64), ("B", C.c_int), ("D", C.c_int), ("W", C.c_int), ("dtype", C.c_int), ("silu", C.c_int)]


class Scan(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("x", "dt", "b", "c")] + [(n, C.c_int64) for n in (
        "x_t", "x_b", "dt_t", "dt_b", "b_t", "b_b", "b_g", "c_t", "c_b", "c_g")] + [(n, C.c_void_p) for n in ("a", "d", "dt_bias", "s_in", "mask")] + [
        ("T", C.c_int64)] + [(n, C.c_int) for n in ("B", "D", "N", "G", "dtype", "softplus")]


class Norm(C.Structure):
    _fields_ = [("x", C.c_void_p), ("gate", C.c_void_p), ("x_r", C.c_int64), ("gate_r", C.c_int64), ("weight", C.c_void_p), ("bias", C.c_void_p),
                ("rows", C.c_int64), ("C", C.c_int), ("groups", C.c_int), ("dtype", C.c_int), ("silu", C.c_int), ("eps", C.c_float)]


EINVAL, EALIGN, EUNSUPPORTED, EWORKSPACE = -1, -2, -3, -4


def test_c_abi_refuses_before_a_device_is_touched():
    lib = _lib.load()
    conv = dict(x=16, x_t=16, x_b=8, weight=16, T=4, B=2, D=8, W=4)
    for status, change in ((EINVAL, dict(x=None)), (EINVAL, dict(T=0)), (EINVAL, dict(D=-1)), (EUNSUPPORTED, dict(W=9)), (EUNSUPPORTED, dict(W=0)),
                           (EUNSUPPORTED, dict(dtype=3)), (EUNSUPPORTED, dict(B=65536)), (EUNSUPPORTED, dict(T=1 << 31))):
        s = Conv(**{**conv, **change})
        assert lib.rfa_causal_conv_fwd(C.addressof(s), 16, None, None) == status, change
        assert lib.rfa_causal_conv_bwd(C.addressof(s), 16, 8, 8, None, 16, None, None, None, None, 0, None) == status, change
    s = Conv(**conv, state_in=32)
    assert lib.rfa_causal_conv_fwd(C.addressof(s), 16, 32, None) == EINVAL and b"in place" in lib.rfa_last_error()
    assert lib.rfa_causal_conv_fwd(None, 16, None, None) == EINVAL
    assert lib.rfa_causal_conv_bwd(C.addressof(s), 16, 8, 8, None, 16, 16, None, None, None, 0, None) == EWORKSPACE
    scan = dict(x=16, dt=16, a=16, b=16, c=16, T=4, B=2, D=8, N=16, G=1, b_t=16)
    for status, change in ((EINVAL, dict(b=None)), (EINVAL, dict(N=0)), (EINVAL, dict(G=0)), (EUNSUPPORTED, dict(N=65)), (EUNSUPPORTED, dict(G=3)),
                           (EUNSUPPORTED, dict(dtype=7)), (EUNSUPPORTED, dict(B=1 << 17)), (EALIGN, dict(s_in=20))):
        s = Scan(**{**scan, **change})
        assert lib.rfa_selective_scan_fwd(C.addressof(s), 16, None, None, None, 0, None) == status, change
        assert lib.rfa_selective_scan_bwd(C.addressof(s), *[16] * 11, 16, 1 << 40, None) == status, change
    s = Scan(**scan)
    assert lib.rfa_selective_scan_step(C.addressof(s), 16, 16, None) == EINVAL and b"4 tokens" in lib.rfa_last_error()
    assert lib.rfa_selective_scan_fwd(C.addressof(s), None, None, None, None, 0, None) == EINVAL
    assert lib.rfa_selective_scan_bwd(C.addressof(s), *[16] * 11, 16, 0, None) == EWORKSPACE
    long = Scan(**{**scan, "T": 1 << 16})
    assert lib.rfa_selective_scan_workspace_bytes(1 << 16, 2, 8, 16, 1, 0) > 0           # few rows: cut into segments
    assert lib.rfa_selective_scan_fwd(C.addressof(long), 16, None, None, None, 0, None) == EWORKSPACE
    assert lib.rfa_selective_scan_checkpoint_bytes(17, 2, 8, 3) == 3 * 2 * 8 * 8 * 4
    assert lib.rfa_selective_scan_checkpoint_bytes(17, 2, 8, 16) == 2 * 2 * 8 * 16 * 4
    norm = dict(x=16, x_r=8, rows=3, C=8, groups=2)
    for status, change in ((EINVAL, dict(x=None)), (EINVAL, dict(rows=0)), (EINVAL, dict(groups=0)), (EUNSUPPORTED, dict(groups=3)),
                           (EUNSUPPORTED, dict(dtype=-1)), (EUNSUPPORTED, dict(C=32768, groups=1))):
        s = Norm(**{**norm, **change})
        assert lib.rfa_group_norm_fwd(C.addressof(s), 16, None) == status, change
        assert lib.rfa_group_norm_bwd(C.addressof(s), 16, 8, 16, None, None, None, None, 0, None) == status, change
    s = Norm(**norm)
    assert lib.rfa_group_norm_bwd(C.addressof(s), 16, 8, 16, None, 16, None, None, 0, None) == EWORKSPACE


def test_c_abi_refuses_more_channels_than_its_indexes_hold():
    lib, most = _lib.load(), 1 << 24
    for d in (most + 1, 1 << 28, (1 << 31) - 1):
        conv = Conv(x=16, x_t=d, x_b=d, weight=16, T=1, B=1, D=d, W=4)
        assert lib.rfa_causal_conv_fwd(C.addressof(conv), 16, None, None) == EUNSUPPORTED
        assert lib.rfa_causal_conv_bwd(C.addressof(conv), 16, d, d, None, 16, None, None, None, None, 0, None) == EUNSUPPORTED
        scan = Scan(x=16, dt=16, a=16, b=16, c=16, T=1, B=1, D=d, N=64, G=1)
        assert lib.rfa_selective_scan_fwd(C.addressof(scan), 16, None, None, None, 0, None) == EUNSUPPORTED
        assert lib.rfa_selective_scan_step(C.addressof(scan), 16, 16, None) == EUNSUPPORTED
        assert lib.rfa_selective_scan_bwd(C.addressof(scan), *[16] * 11, 16, 1 << 40, None) == EUNSUPPORTED
        norm = Norm(x=16, x_r=d, rows=1, C=d, groups=d)
        assert lib.rfa_group_norm_fwd(C.addressof(norm), 16, None) == EUNSUPPORTED
        assert lib.rfa_group_norm_bwd(C.addressof(norm), 16, d, 16, None, None, None, None, 0, None) == EUNSUPPORTED


def test_older_entry_points_refuse_bf16():
    """The code of bf16 names a type of the state-space entry points only."""
    lib = _lib.load()
    assert lib.rfa_feature_map_fwd(16, 2, 16, 16, 2, 10, 2, 64, 64, C.c_float(0.1), None) == EUNSUPPORTED
    assert lib.rfa_decode_step(16, 16, 16, 2, 16, 16, 1, 16, 4, 128, 64, None) == EUNSUPPORTED
    assert lib.rfa_decode_step(16, 16, 16, 0, 16, 16, 2, 16, 4, 128, 64, None) == EUNSUPPORTED
    assert lib.rfa_decode_step_fused(16, 16, 16, 2, 16, 0.1, 16, 16, 1, 16, 4, 2, 64, 64, None) == EUNSUPPORTED
    assert lib.rfa_gather_random_matrices(16, 2, 4, 16, 2, None, None, 16, 8, 8, 16, None) == EUNSUPPORTED
    assert lib.rfa_cross_decode_step(16, 2, 16, 16, 16, 2, 4, 128, 64, None) == EUNSUPPORTED


def test_reordering_keeps_the_state_of_the_old_slot():
    state = dict(prev_conv=torch.arange(3.)[:, None, None].expand(3, 2, 4), prev_s=torch.arange(3.)[:, None, None].expand(3, 4, 5))
    out = SelectiveStateSpace.reorder_incremental_state(state, torch.tensor([2, 0, 0]))
    assert out["prev_conv"][:, 0, 0].tolist() == out["prev_s"][:, 0, 0].tolist() == [2, 0, 0]
    assert SelectiveStateSpace.reorder_incremental_state({}, torch.tensor([0])) == {}


def test_tensor_calls_are_exported():
    for name in ("causal_conv_fwd", "causal_conv_bwd", "selective_scan_fwd", "selective_scan_bwd", "group_norm_fwd", "group_norm_bwd"):
        assert callable(getattr(ops, name)) and callable(getattr(_lib.native(), name))


def test_wide_accesses_are_taken_of_addresses_that_hold_them(tmp_path):
    """The host's rule, by itself: a run of `nv` elements is taken in words of 16, 8 or 4 bytes, whichever divides it; an address that is
    not a multiple of them is refused, and none that is."""
    import os
    import subprocess
    csrc = os.path.join(os.path.dirname(_lib.__file__), "csrc")
    src, exe = tmp_path / "wide.cpp", tmp_path / "wide"
    src.write_text('#include "wide.h"\n#include <cstdio>\n#include <initializer_list>\n'
                   "int main() {\n"
                   "  for (int size : {2, 4}) for (int nv = 2; nv <= 32; nv += 2) for (int at = 0; at < 32; at += size)\n"
                   '    std::printf("%d %d %d %d\\n", size, nv, at, (int)rfa::wide_ok(reinterpret_cast<const void*>((uintptr_t)4096 + at), 0, 0, size, nv));\n'
                   "}\n")
    subprocess.run(["g++", "-std=c++17", "-I" + csrc, str(src), "-o", str(exe)], check=True)
    rows = [tuple(map(int, line.split())) for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines()]
    assert len(rows) == 16 * (16 + 8)
    for size, nv, at, taken in rows:
        words = nv * size // 4                                    # a run in 32-bit words: four, two or one of them at a time
        access = 16 if words % 4 == 0 else 8 if words % 2 == 0 else 4
        assert bool(taken) == (at % access == 0), (size, nv, at)
    # the convolution's weights: 4 channels of `width` taps; 8 modulo 16 holds them in 16 bits only where the width is odd
    assert {w: dict(((s, n, a), t) for s, n, a, t in rows)[2, 4 * w, 8] for w in range(1, 9)} == {1: 1, 2: 0, 3: 1, 4: 0, 5: 1, 6: 0, 7: 1, 8: 0}


def test_c_abi_refuses_a_scan_whose_last_state_is_its_first():
    lib = _lib.load()
    for T in (1, 4, 1 << 16):                                     # in one segment and in several
        s = Scan(x=16, dt=16, a=16, b=16, c=16, T=T, B=2, D=8, N=16, G=1, b_t=16, s_in=32)
        assert lib.rfa_selective_scan_fwd(C.addressof(s), 16, 32, None, 16, 1 << 40, None) == EINVAL
        assert b"s_out is s_in" in lib.rfa_last_error()


def test_c_abi_refuses_outputs_in_place_of_what_other_ctas_read():
    lib = _lib.load()
    conv = Conv(x=16, x_t=16, x_b=8, weight=32, T=400, B=2, D=8, W=4, state_in=48)
    assert lib.rfa_causal_conv_fwd(C.addressof(conv), 16, None, None) == EINVAL and b"y is x" in lib.rfa_last_error()
    back = lambda g, g_state, gx, gs: lib.rfa_causal_conv_bwd(C.addressof(conv), g, 16, 8, g_state, gx, None, None, gs, None, 0, None)
    for gx in (16, 64):
        assert back(64, None, gx, None) == EINVAL and b"gx is g or x" in lib.rfa_last_error()
    for gs in (48, 80):
        assert back(64, 80, 96, gs) == EINVAL and b"g_state_in is g_state or state_in" in lib.rfa_last_error()
    scan = Scan(x=16, dt=16, a=16, b=16, c=16, T=4, B=2, D=8, N=16, G=1, b_t=16)
    assert lib.rfa_selective_scan_bwd(C.addressof(scan), 16, 32, *[16] * 8, 32, 16, 1 << 40, None) == EINVAL
    assert b"gs_in is g_s" in lib.rfa_last_error()


@pytest.mark.parametrize("wrong,name", [(dict(conv_width=9), "conv_width"), (dict(conv_width=0), "conv_width"), (dict(state_dim=65), "state_dim"),
                                        (dict(state_dim=0), "state_dim"), (dict(num_groups=0), "num_groups"), (dict(norm_groups=0), "norm_groups"),
                                        (dict(norm_groups=-1), "norm_groups"), (dict(inner_dim=0), "inner_dim"),
                                        (dict(inner_dim=16400, norm_groups=1, state_dim=1, dt_rank=1), "16384")])
def test_a_layer_that_its_operators_refuse_is_not_built(wrong, name):
    with pytest.raises(AssertionError, match=name):
        SelectiveStateSpace(**{**dict(embed_dim=2), **wrong})
    SelectiveStateSpace(embed_dim=2, conv_width=8, state_dim=64, norm_groups=4)
