"""The operators that a layer has round the recurrence: short convolution, selective state space scan, gated and residual norms.

No counterparts in the reference.  The manner is that of `fwd`: results go into tensors that the caller gives, nothing is returned or
synchronised, work is enqueued on the current stream of the tensors' device, and every argument problem raises RuntimeError before
anything is launched.  Forward only, like `fwd`: no gradients are recorded.  An ordinary call is checked and launched natively
(csrc/fkda_host.cpp); one that is not in order goes through the checks here, which own the messages, as do all calls where the native
host path does not fit the running torch.
"""
import ctypes

import torch

from . import _binding
from ._binding import _check, _decline, _ptr, _require, lib

_fast = None


def _rows(*names):
    return [field for n in names for field in ((f"{n}_batch_stride", ctypes.c_int64), (f"{n}_token_stride", ctypes.c_int64))]


def _fields(kind, *names):
    return [(n, kind) for n in names]


_P, _I64, _I32, _F = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32, ctypes.c_float


class ConvParams(ctypes.Structure):
    """Mirror of `fkda_conv_params` (include/fkda.h)."""
    _fields_ = (_fields(_P, "x", "weight", "bias", "out", "initial_state", "final_state", "cu_seqlens") + _fields(_I64, "B", "T", "C", "N")
                + _rows("x", "out") + _fields(_I32, "width", "weight_dtype", "silu"))


class SsmParams(ctypes.Structure):
    """Mirror of `fkda_ssm_params`."""
    _fields_ = (_fields(_P, "x", "dt", "Bm", "Cm", "out", "A_log", "dt_bias", "D", "initial_state", "final_state", "cu_seqlens", "workspace")
                + _fields(_I64, "workspace_bytes", "B", "T", "H", "P", "G", "Ns", "N") + _rows("x", "dt", "B", "C", "out")
                + _fields(_I32, "state_dtype") + [("flags", ctypes.c_uint32)])


class GatedNormParams(ctypes.Structure):
    """Mirror of `fkda_gated_norm_params`."""
    _fields_ = (_fields(_P, "x", "gate", "weight", "out") + _fields(_I64, "B", "T", "H", "D") + _rows("x", "gate", "out")
                + _fields(_F, "eps") + _fields(_I32, "weight_dtype", "weight_per_head", "silu", "gate_first"))


class AddNormParams(ctypes.Structure):
    """Mirror of `fkda_add_norm_params`."""
    _fields_ = (_fields(_P, "x", "residual", "weight", "out", "residual_out") + _fields(_I64, "B", "T", "D")
                + _rows("x", "residual", "out", "residual_out") + _fields(_F, "scale", "eps") + _fields(_I32, "weight_dtype", "residual_dtype"))


def _lib():
    L = lib()
    for name, params in (("fkda_short_conv", ConvParams), ("fkda_ssm_fwd", SsmParams), ("fkda_gated_norm", GatedNormParams), ("fkda_add_norm", AddNormParams)):
        f = getattr(L, name)
        f.argtypes, f.restype = [ctypes.POINTER(params), ctypes.c_void_p], ctypes.c_int
    L.fkda_ssm_scratch_bytes.argtypes = [ctypes.POINTER(SsmParams), ctypes.POINTER(ctypes.c_int64)]
    L.fkda_ssm_scratch_bytes.restype = ctypes.c_int
    return L


def _native(name):
    """The operator's function of the native host path, or one that declines."""
    global _fast
    if _fast is None:
        if (_binding._fwd_fast or _binding._load_host()) is _decline:
            _fast = {}
        else:
            from . import _fkda_host
            _fast = {n: getattr(_fkda_host, n + "_fast") for n in ("short_conv", "ssm_fwd", "gated_norm", "add_norm") if hasattr(_fkda_host, n + "_fast")}
    return _fast.get(name, _decline)


def _handled(done):
    """Whether the native host path did the call; raises its error message."""
    if done is True:
        return True
    if done is not False:
        raise RuntimeError(done)
    return False


_DTYPES = {torch.bfloat16: 1, torch.float32: 2}


def _tensors(**named):
    for name, t in named.items():
        _require(isinstance(t, torch.Tensor), f"{name} must be a tensor")
        _require(t.is_cuda, f"{name} must be on CUDA")
    devices = {t.device for t in named.values()}
    _require(len(devices) == 1, "all tensors must be on the same CUDA device")


def _bf16(**named):
    for name, t in named.items():
        _require(t.dtype == torch.bfloat16, f"{name} must be bfloat16")


def _tokens(t, name, shape):
    """A [B, T, ...] tensor whose tokens are dense: (batch stride, token stride)."""
    _require(tuple(t.shape) == tuple(shape), f"{name} must be {list(shape)}, is {list(t.shape)}")
    dense = 1
    for size, stride in zip(reversed(t.shape[2:]), reversed(t.stride()[2:])):
        _require(size == 1 or stride == dense, f"the last dimensions of {name} must be contiguous")
        dense *= size
    return t.stride(0), t.stride(1)


def _weight(t, name, *shapes):
    _require(t.dtype in _DTYPES, f"{name} must be bfloat16 or float32")
    _require(t.is_contiguous(), f"{name} must be contiguous")
    _require(tuple(t.shape) in shapes, f"{name} must be {' or '.join(str(list(s)) for s in shapes)}, is {list(t.shape)}")
    return _DTYPES[t.dtype]


def _sequences(cu_seqlens, batch):
    if cu_seqlens is None:
        return batch
    _require(batch == 1, "B must be 1 when cu_seqlens is provided")
    _require(cu_seqlens.dtype == torch.int64, "cu_seqlens must be int64")
    _require(cu_seqlens.dim() == 1 and cu_seqlens.is_contiguous(), "cu_seqlens must be 1D and contiguous")
    _require(cu_seqlens.numel() >= 2, "cu_seqlens must have at least 2 elements")
    return cu_seqlens.numel() - 1


def _given(**named):
    return {name: t for name, t in named.items() if t is not None}


def _launch(function, params, device):
    with torch.cuda.device(device):
        stream = ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)
        _check(getattr(_lib(), function)(ctypes.byref(params), stream))


def short_conv(x, weight, out, bias=None, initial_state=None, final_state=None, cu_seqlens=None, *, silu=True):
    """Depthwise causal convolution, as it stands before the recurrence on q, k and v (or on x, B and C of `ssm_fwd`):

        out[t, c] = act(bias[c] + sum_k weight[c, k] x[t - (W - 1) + k, c]),   act = SiLU (or none)

    x, out: bf16 [B, T, C], C a multiple of 8; columns of wider tensors will do (16-byte aligned rows).  weight: [C, W] with W of 2 to
    4, bias: [C] or None, both bf16 or both fp32.  initial_state / final_state: bf16 [N, W-1, C], the last inputs of every sequence, the
    oldest first (None: zeros / not wanted); they may be one tensor.  cu_seqlens: int64 [N+1] on the device, requires B == 1.
    A decode step is the call with T == 1.  `out` may not share memory with `x`."""
    if _handled(_native("short_conv")(x, weight, out, bias, initial_state, final_state, cu_seqlens, silu)):
        return None
    _tensors(**_given(x=x, weight=weight, out=out, bias=bias, initial_state=initial_state, final_state=final_state, cu_seqlens=cu_seqlens))
    _bf16(**_given(x=x, out=out, initial_state=initial_state, final_state=final_state))
    _require(x.dim() == 3, "x must be [B, T, C]")
    batch, T, C = x.shape
    _require(weight.dim() == 2 and weight.shape[0] == C, "weight must be [C, W]")
    W = weight.shape[1]
    dtype = _weight(weight, "weight", (C, W))
    if bias is not None:
        _require(_weight(bias, "bias", (C,)) == dtype, "bias must have the dtype of weight")
    N = _sequences(cu_seqlens, batch)
    for name, st in _given(initial_state=initial_state, final_state=final_state).items():
        _require(st.is_contiguous() and tuple(st.shape) == (N, W - 1, C), f"{name} must be a contiguous [N, W-1, C] tensor")
    p = ConvParams(_ptr(x), _ptr(weight), _ptr(bias), _ptr(out), _ptr(initial_state), _ptr(final_state), _ptr(cu_seqlens),
                   batch, T, C, N, *_tokens(x, "x", x.shape), *_tokens(out, "out", x.shape), W, dtype, int(bool(silu)))
    _launch("fkda_short_conv", p, x.device)
    return None


def _ssm_params(x, dt, Bm, Cm, out, A_log, dt_bias, D, initial_state, final_state, cu_seqlens):
    _tensors(**_given(x=x, dt=dt, B=Bm, C=Cm, out=out, A_log=A_log, dt_bias=dt_bias, D=D, initial_state=initial_state, final_state=final_state,
                      cu_seqlens=cu_seqlens))
    _bf16(x=x, dt=dt, B=Bm, C=Cm, out=out)
    _require(x.dim() == 4, "x must be [B, T, H, P]")
    batch, T, H, P = x.shape
    _require(Bm.dim() == 4, "B must be [B, T, G, Ns]")
    G, Ns = Bm.shape[2:]
    _require(P in (64, 128), "P must be 64 or 128")
    _require(Ns in (64, 128), "the columns of a state must be 64 or 128")
    _require(G > 0 and H > 0 and H % G == 0, "H must be a multiple of G")
    for name, t in _given(A_log=A_log, dt_bias=dt_bias, D=D).items():
        _require(t.dtype == torch.float32 and t.is_contiguous() and tuple(t.shape) == (H,), f"{name} must be a contiguous float32 [H] tensor")
    N = _sequences(cu_seqlens, batch)
    state_dtype = 0
    for name, st in _given(initial_state=initial_state, final_state=final_state).items():
        _require(st.dtype in _DTYPES, f"{name} must be bfloat16 or float32")
        _require(st.is_contiguous() and tuple(st.shape) == (N, H, P, Ns), f"{name} must be a contiguous [N, H, P, Ns] tensor")
        _require(state_dtype in (0, _DTYPES[st.dtype]), "initial_state and final_state must have the same dtype")
        state_dtype = _DTYPES[st.dtype]
    return SsmParams(_ptr(x), _ptr(dt), _ptr(Bm), _ptr(Cm), _ptr(out), _ptr(A_log), _ptr(dt_bias), _ptr(D), _ptr(initial_state),
                     _ptr(final_state), _ptr(cu_seqlens), None, 0, batch, T, H, P, G, Ns, N, *_tokens(x, "x", x.shape),
                     *_tokens(dt, "dt", (batch, T, H)), *_tokens(Bm, "B", (batch, T, G, Ns)), *_tokens(Cm, "C", (batch, T, G, Ns)),
                     *_tokens(out, "out", x.shape), state_dtype, 0)


def ssm_fwd(x, dt, B, C, out, A_log, dt_bias, D=None, initial_state=None, final_state=None, cu_seqlens=None, *, workspace=None):
    """Selective state space scan with one decay per head; with delta = softplus(dt + dt_bias[h]),

        S_t = exp(-exp(A_log[h]) delta) S_(t-1) + delta x_t B_t^T,     out_t = S_t C_t + D[h] x_t

    x, out: bf16 [B, T, H, P]; dt: bf16 [B, T, H]; B, C: bf16 [B, T, G, Ns], a group's shared by H / G heads; P and Ns 64 or 128.  These
    may be columns of wider tensors (16-byte aligned rows; dt any).  A_log, dt_bias, D: fp32 [H], D or None.  initial_state / final_state:
    bf16 or fp32 [N, H, P, Ns] (same dtype when both are given) or None; they may be one tensor.  cu_seqlens: int64 [N+1] on the device,
    requires B == 1.  A decode step is the call with T == 1.  `out` may not share memory with an input.  An fp32 final_state is exact to fp32; where it is
    bf16 or not asked for, prompts keep 16 bits of what each token adds to a state, in 87 % of the time.

    `workspace` (optional): a uint8 CUDA tensor of at least `ssm_workspace_size(...)` bytes, 256-byte aligned, for callers that must not allocate; by default
    scratch memory comes from torch's caching allocator, where a call needs any.  `read_status(workspace)` then has the call's status, also of calls that
    need no scratch memory, if the tensor has at least four bytes."""
    if workspace is None and _handled(_native("ssm_fwd")(x, dt, B, C, out, A_log, dt_bias, D, initial_state, final_state, cu_seqlens)):
        return None
    p = _ssm_params(x, dt, B, C, out, A_log, dt_bias, D, initial_state, final_state, cu_seqlens)
    _ssm_launch(p, x.device, workspace)
    return None


def _scratch_bytes(p, device):
    needed = ctypes.c_int64(0)
    with torch.cuda.device(device):
        _check(_lib().fkda_ssm_scratch_bytes(ctypes.byref(p), ctypes.byref(needed)))
    return needed.value


def _ssm_launch(p, device, workspace):
    if workspace is not None:
        _require(isinstance(workspace, torch.Tensor) and workspace.is_cuda and workspace.is_contiguous() and workspace.dtype == torch.uint8,
                   "workspace must be a contiguous uint8 CUDA tensor")
        _require(workspace.device == device, "workspace must be on the same CUDA device as x")
    else:
        needed = _scratch_bytes(p, device)
        if needed:
            workspace = torch.empty(needed, dtype=torch.uint8, device=device)
    if workspace is not None:
        p.workspace, p.workspace_bytes = workspace.data_ptr(), workspace.numel()
    _launch("fkda_ssm_fwd", p, device)


def ssm_workspace_size(x, dt, B, C, out, A_log, dt_bias, D=None, initial_state=None, final_state=None, cu_seqlens=None) -> int:
    """Bytes of scratch memory that `ssm_fwd` with these arguments needs (0 for many)."""
    return _scratch_bytes(_ssm_params(x, dt, B, C, out, A_log, dt_bias, D, initial_state, final_state, cu_seqlens), x.device)


_ACTS = {"sigmoid": 0, "silu": 1}


def gated_norm(x, gate, weight, out, *, eps=1e-6, act="sigmoid", gate_first=False):
    """Norm behind the recurrence with its output gate a = sigmoid(gate) or, with act="silu", gate sigmoid(gate):

        out = x / rms(x) * weight * a,   with gate_first   out = (x a) / rms(x a) * weight,    rms(u) = sqrt(mean(u^2) + eps)

    over the last dimension.  x, gate, out: bf16 [B, T, H, D] (a norm per head; H = 1 for one over all channels), D a multiple of 8 up to
    16384; columns of wider tensors will do (16-byte aligned rows).  weight: bf16 or fp32 [D], or [H, D].  `out` may be `x` or `gate`."""
    if _handled(_native("gated_norm")(x, gate, weight, out, eps, act, gate_first)):
        return None
    _tensors(x=x, gate=gate, weight=weight, out=out)
    _bf16(x=x, gate=gate, out=out)
    _require(x.dim() == 4, "x must be [B, T, H, D]")
    _require(act in _ACTS, "act must be 'sigmoid' or 'silu'")
    batch, T, H, D = x.shape
    dtype = _weight(weight, "weight", (D,), (H, D))
    p = GatedNormParams(_ptr(x), _ptr(gate), _ptr(weight), _ptr(out), batch, T, H, D, *_tokens(x, "x", x.shape), *_tokens(gate, "gate", x.shape),
                        *_tokens(out, "out", x.shape), float(eps), dtype, int(weight.dim() == 2), _ACTS[act], int(bool(gate_first)))
    _launch("fkda_gated_norm", p, x.device)
    return None


def add_norm(x, residual, weight, out, residual_out, *, scale=1.0, eps=1e-6):
    """Residual connection behind a block and norm before the next one:

        h = residual + scale * x;   residual_out = h;   out = h / rms(h) * weight

    x, out: bf16 [B, T, D]; residual, residual_out: bf16 or fp32 [B, T, D] (the same), D a multiple of 8 up to 16384; columns of wider
    tensors will do (16-byte aligned rows).  weight: bf16 or fp32 [D].  The norm is that of h before it is rounded to the residual's
    dtype.  `residual_out` may be `residual`, `out` may be `x`."""
    if _handled(_native("add_norm")(x, residual, weight, out, residual_out, scale, eps)):
        return None
    _tensors(x=x, residual=residual, weight=weight, out=out, residual_out=residual_out)
    _bf16(x=x, out=out)
    _require(x.dim() == 3, "x must be [B, T, D]")
    _require(residual.dtype in _DTYPES, "residual must be bfloat16 or float32")
    _require(residual_out.dtype == residual.dtype, "residual_out must have the dtype of residual")
    batch, T, D = x.shape
    dtype = _weight(weight, "weight", (D,))
    p = AddNormParams(_ptr(x), _ptr(residual), _ptr(weight), _ptr(out), _ptr(residual_out), batch, T, D, *_tokens(x, "x", x.shape),
                      *_tokens(residual, "residual", x.shape), *_tokens(out, "out", x.shape), *_tokens(residual_out, "residual_out", x.shape),
                      float(scale), float(eps), dtype, _DTYPES[residual.dtype])
    _launch("fkda_add_norm", p, x.device)
    return None
