"""CPU: the operators round the recurrence refuse what they cannot do before anything is launched, through Python and through the C ABI,
and the Python structures mirror the header."""
import ctypes
import os
import re

import pytest
import torch

import flashkda_b200 as F
from flashkda_b200 import _layer as L

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BF16, FP32 = 1, 2
A, B, C, D, E, G = (0x10000000 * i for i in range(1, 7))         # addresses apart, 16-byte aligned, never touched


@pytest.mark.parametrize("name,struct", [("conv", L.ConvParams), ("ssm", L.SsmParams), ("gated_norm", L.GatedNormParams), ("add_norm", L.AddNormParams)])
def test_structures_mirror_the_header(name, struct):
    text = open(os.path.join(ROOT, "include", "fkda.h")).read()
    start = text.index(f"typedef struct fkda_{name}_params {{")
    body = re.sub(r"/\*.*?\*/", "", text[start:text.index(f"}} fkda_{name}_params;")], flags=re.S)
    fields = re.findall(r"(\w[\w ]*[ *]+)([A-Za-z_]+);", body)
    kinds = {"int64_t": ctypes.c_int64, "int32_t": ctypes.c_int32, "uint32_t": ctypes.c_uint32, "float": ctypes.c_float}
    want = [(n, ctypes.c_void_p if "*" in t else kinds[t.strip()]) for t, n in fields]
    assert want == [(n, t) for n, t in struct._fields_]


def refused(function, params, match):
    rc = getattr(L._lib(), function)(ctypes.byref(params), None)
    assert rc == -1 and re.search(match, F.last_error()), (rc, F.last_error())


def conv(**more):
    p = dict(x=A, weight=B, bias=None, out=C, initial_state=None, final_state=None, cu_seqlens=None, B=2, T=16, C=64, N=2, x_batch_stride=16 * 64,
             x_token_stride=64, out_batch_stride=16 * 64, out_token_stride=64, width=4, weight_dtype=BF16, silu=1)
    return L.ConvParams(**{**p, **more})


@pytest.mark.parametrize("more,match", [
    (dict(x=None), "x must be non-NULL"), (dict(out=None), "out must be non-NULL"), (dict(weight=None), "weight must be non-NULL"), (dict(C=60), "multiple of 8"), (dict(C=0), "multiple of 8"),
    (dict(width=1), "width"), (dict(width=5), "width"), (dict(weight_dtype=0), "weight_dtype"), (dict(B=0), "B must be positive"), (dict(T=-1), "non-negative"),
    (dict(N=3), "N must equal B"), (dict(cu_seqlens=D), "B must be 1"), (dict(cu_seqlens=D, B=1, N=0), "at least 2"), (dict(x=A + 2), "16-byte boundary"),
    (dict(x_token_stride=66, x_batch_stride=2048), "multiples of 16 bytes"), (dict(x_token_stride=56), "rows of x overlap"), (dict(out_batch_stride=64), "rows of out overlap"), (dict(x_token_stride=-64), "out of range"),
    (dict(x_batch_stride=1 << 60), "out of range"), (dict(out=A), "out shares memory with x"), (dict(out=A + 64), "out shares memory with x"), (dict(x_token_stride=128, x_batch_stride=2048, out=A + 64), "shares memory"),
    (dict(initial_state=D, final_state=D + 16), "overlaps initial_state"), (dict(final_state=A), "state shares memory"), (dict(initial_state=C), "state shares memory"), (dict(initial_state=D + 4), "16-byte boundary"),
    (dict(out=B), "weight or bias"), (dict(bias=C + 16), "weight or bias"), (dict(final_state=B), "weight or bias"), (dict(final_state=D, bias=D + 64), "weight or bias"), (dict(T=1 << 39, x_batch_stride=1 << 45, out_batch_stride=1 << 45, out=A << 20), "too (many|large)|out of range")])
def test_short_conv_refusals(more, match):
    refused("fkda_short_conv", conv(**more), match)


def ssm(**more):
    p = dict(x=A, dt=B, Bm=C, Cm=C + 256, out=D, A_log=E, dt_bias=E + 4096, D=None, initial_state=None, final_state=None, cu_seqlens=None, workspace=G, workspace_bytes=1 << 40, B=2, T=300,
             H=4, P=64, G=1, Ns=128, N=2, x_batch_stride=300 * 256, x_token_stride=256, dt_batch_stride=1200, dt_token_stride=4, B_batch_stride=300 * 256, B_token_stride=256,
             C_batch_stride=300 * 256, C_token_stride=256, out_batch_stride=300 * 256, out_token_stride=256, state_dtype=0, flags=0)
    return L.SsmParams(**{**p, **more})


@pytest.mark.parametrize("more,match", [
    (dict(x=None), "x must be non-NULL"), (dict(dt=None), "dt must be non-NULL"), (dict(Bm=None), "B must be non-NULL"), (dict(Cm=None), "C must be non-NULL"), (dict(out=None), "out must be non-NULL"),
    (dict(A_log=None), "A_log"), (dict(dt_bias=None), "dt_bias"), (dict(P=96), "P and the columns"), (dict(Ns=32), "P and the columns"), (dict(G=3), "multiple of G"), (dict(G=0), "multiple of G"),
    (dict(H=0), "H must lie"), (dict(H=70000, G=1), "H must lie"), (dict(N=1), "N must equal B"), (dict(initial_state=0x100000000), "state_dtype"), (dict(cu_seqlens=E), "B must be 1"),
    (dict(x=A + 8), "x must start"), (dict(Bm=C + 8), "B must start"), (dict(C_token_stride=260, C_batch_stride=1 << 17), "multiples of 16 bytes"), (dict(dt_token_stride=3), "rows of dt overlap"), (dict(out_token_stride=128), "rows of out overlap"),
    (dict(out=A), "out shares memory with x"), (dict(out=C), "out shares memory with B"), (dict(D=D + 1024), "shares memory with A_log"), (dict(dt_bias=D + 64), "shares memory with A_log"), (dict(state_dtype=FP32, final_state=E), "shares memory with A_log"), (dict(state_dtype=FP32, final_state=A), "final_state shares memory with x"),
    (dict(state_dtype=FP32, initial_state=D), "out shares memory with initial_state"), (dict(state_dtype=FP32, initial_state=0x100000000, final_state=0x100000010), "overlaps initial_state"),
    (dict(workspace=None), "workspace must be"), (dict(workspace=G + 16), "workspace must be"), (dict(T=1 << 33, x_batch_stride=1 << 41, out_batch_stride=1 << 41), "too many tokens")])
def test_ssm_refusals(more, match):
    refused("fkda_ssm_fwd", ssm(**more), match)


def test_ssm_workspace_is_asked_for_and_checked():
    need = ctypes.c_int64(-1)
    ask = lambda p: (L._lib().fkda_ssm_scratch_bytes(ctypes.byref(p), ctypes.byref(need)), need.value)
    assert ask(ssm(T=8)) == (0, 0) and ask(ssm(T=1)) == (0, 0)
    rc, few = ask(ssm(T=300))
    assert rc == 0 and few >= 256
    rc, long = ask(ssm(T=100000, B=1, N=1))
    assert rc == 0 and long > (1 << 20)                              # states between the runs
    rc, packed = ask(ssm(T=100000, B=1, N=7, cu_seqlens=E))
    assert rc == 0 and packed > 256
    assert ask(ssm(P=65))[0] == -1
    assert L._lib().fkda_ssm_fwd(ctypes.byref(ssm(workspace_bytes=few - 1)), None) == -2 and "needed" in F.last_error()


def gated(**more):
    p = dict(x=A, gate=B, weight=E, out=C, B=2, T=4, H=2, D=72, x_batch_stride=576, x_token_stride=144, gate_batch_stride=576, gate_token_stride=144, out_batch_stride=576,
             out_token_stride=144, eps=1e-6, weight_dtype=FP32, weight_per_head=0, silu=0, gate_first=0)
    return L.GatedNormParams(**{**p, **more})


@pytest.mark.parametrize("more,match", [
    (dict(x=None), "x must be"), (dict(gate=None), "gate must be"), (dict(weight=None), "weight must be"), (dict(D=70), "multiple of 8"), (dict(D=16392), "multiple of 8"), (dict(H=0), "B and H"),
    (dict(eps=float("nan")), "eps"), (dict(eps=-1.0), "eps"), (dict(weight_dtype=3), "weight_dtype"), (dict(weight=E + 4), "16-byte"), (dict(out=A + 144), "out shares memory with x"),
    (dict(out=B, out_token_stride=288, out_batch_stride=1152), "out shares memory with gate"), (dict(out=E), "weight"), (dict(gate_token_stride=100), "rows of gate overlap"),
    (dict(x_token_stride=145, x_batch_stride=580), "multiples of 16 bytes"), (dict(B=1 << 20, T=1 << 20), "too many rows")])
def test_gated_norm_refusals(more, match):
    refused("fkda_gated_norm", gated(**more), match)


def add(**more):
    p = dict(x=A, residual=B, weight=E, out=C, residual_out=D, B=2, T=4, D=72, x_batch_stride=288, x_token_stride=72, residual_batch_stride=288, residual_token_stride=72, out_batch_stride=288,
             out_token_stride=72, residual_out_batch_stride=288, residual_out_token_stride=72, scale=1.0, eps=1e-6, weight_dtype=BF16, residual_dtype=FP32)
    return L.AddNormParams(**{**p, **more})


@pytest.mark.parametrize("more,match", [
    (dict(x=None), "x must be"), (dict(residual=None), "residual must be"), (dict(residual_out=None), "residual_out must be"), (dict(D=71), "multiple of 8"), (dict(residual_dtype=0), "residual_dtype"),
    (dict(scale=float("inf")), "finite"), (dict(out=D), "out shares memory with residual_out"), (dict(residual_out=B + 16), "without being it"), (dict(out=B), "out shares memory with residual"),
    (dict(residual_out=A), "residual_out shares memory with x"), (dict(out=A + 16), "out shares memory with x without"), (dict(residual_out=E), "weight"), (dict(residual_token_stride=74, residual_batch_stride=296), "multiples of 16")])
def test_add_norm_refusals(more, match):
    refused("fkda_add_norm", add(**more), match)


def test_null_parameters():
    for f in ("fkda_short_conv", "fkda_ssm_fwd", "fkda_gated_norm", "fkda_add_norm"):
        assert getattr(L._lib(), f)(None, None) == -1
    assert L._lib().fkda_ssm_scratch_bytes(None, None) == -1


def test_cpu_tensors_are_refused_not_computed():
    z = lambda *s, dt=torch.bfloat16: torch.zeros(*s, dtype=dt)
    with pytest.raises(RuntimeError, match="x must be on CUDA"):
        F.short_conv(z(1, 4, 8), z(8, 4), z(1, 4, 8))
    with pytest.raises(RuntimeError, match="x must be on CUDA"):
        F.ssm_fwd(z(1, 4, 2, 64), z(1, 4, 2), z(1, 4, 1, 64), z(1, 4, 1, 64), z(1, 4, 2, 64), z(2, dt=torch.float32), z(2, dt=torch.float32))
    with pytest.raises(RuntimeError, match="x must be on CUDA"):
        F.gated_norm(z(1, 4, 2, 64), z(1, 4, 2, 64), z(64), z(1, 4, 2, 64))
    with pytest.raises(RuntimeError, match="x must be on CUDA"):
        F.add_norm(z(1, 4, 64), z(1, 4, 64), z(64), z(1, 4, 64), z(1, 4, 64))
    with pytest.raises(RuntimeError, match="must be a tensor"):
        F.add_norm(None, z(1, 4, 64), z(64), z(1, 4, 64), z(1, 4, 64))


def test_a_workspace_of_a_short_scan_has_to_be_aligned():
    """It holds the status word, though nothing else is asked for."""
    refused("fkda_ssm_fwd", ssm(T=4, x_batch_stride=1024, out_batch_stride=1024, workspace=G + 16, workspace_bytes=256), "256-byte aligned")
