"""Plain 64-bit forms of the operators round the recurrence, each with the sums of absolute values that its rounding bounds need.

Tolerances count roundings: to bf16 at most 2^-8 of the value, in fp32 2^-24 of the sum of the absolute terms per operation."""
import torch

BF16, FP32 = 2.0 ** -8, 2.0 ** -24


def lengths_of(cu, batch, T):
    return [T] * batch if cu is None else torch.as_tensor(cu).diff().tolist()


def rows_of(cu, batch, T, n, length):
    """(batch row, first token) of sequence n."""
    return (n, 0) if cu is None else (0, int(cu[n]))


def conv(x, weight, bias, initial_state, cu, silu):
    """(out, sum of |terms|, final_state), rows outside every sequence NaN."""
    x = x.double().cpu()
    batch, T, C = x.shape
    w = weight.double().cpu()
    W = w.shape[1]
    lens = lengths_of(cu, batch, T)
    out, mass = torch.full_like(x, float("nan")), torch.zeros_like(x)
    fin = torch.zeros(len(lens), W - 1, C, dtype=torch.float64)
    for n, length in enumerate(lens):
        b, t0 = rows_of(cu, batch, T, n, length)
        past = initial_state[n].double().cpu() if initial_state is not None else torch.zeros(W - 1, C, dtype=torch.float64)
        u = torch.cat([past, x[b, t0:t0 + length]])
        fin[n] = u[length:]
        y, m = torch.zeros(length, C, dtype=torch.float64), torch.zeros(length, C, dtype=torch.float64)
        for k in range(W):
            y += u[k:k + length] * w[:, k]
            m += (u[k:k + length] * w[:, k]).abs()
        if bias is not None:
            y += bias.double().cpu()
            m += bias.double().cpu().abs()
        out[b, t0:t0 + length] = y * torch.sigmoid(y) if silu else y
        mass[b, t0:t0 + length] = m
    return out, mass, fin


def softplus(z):
    return torch.logaddexp(z, torch.zeros_like(z))


def ssm(x, dt, Bm, Cm, A_log, dt_bias, D, initial_state, cu):
    """(out, sum of |terms| of out, final_state, sum of |terms| of the state), token by token; rows outside every sequence NaN."""
    x, dt, Bm, Cm = (t.double().cpu() for t in (x, dt, Bm, Cm))
    A, dt_bias = torch.exp(A_log.double().cpu()), dt_bias.double().cpu()
    batch, T, H, P = x.shape
    G, Ns = Bm.shape[2:]
    lens = lengths_of(cu, batch, T)
    out, mass = torch.full_like(x, float("nan")), torch.zeros_like(x)
    fin, fmass = (torch.zeros(len(lens), H, P, Ns, dtype=torch.float64) for _ in range(2))
    for n, length in enumerate(lens):
        b, t0 = rows_of(cu, batch, T, n, length)
        S = initial_state[n].double().cpu() if initial_state is not None else torch.zeros(H, P, Ns, dtype=torch.float64)
        M = S.abs()
        for t in range(t0, t0 + length):
            delta = softplus(dt[b, t] + dt_bias)
            decay = torch.exp(-A * delta)[:, None, None]
            kb, kc = (m[b, t].repeat_interleave(H // G, 0) for m in (Bm, Cm))
            add = delta[:, None, None] * x[b, t][:, :, None] * kb[:, None, :]
            S, M = decay * S + add, decay * M + add.abs()
            out[b, t], mass[b, t] = (S @ kc[:, :, None])[..., 0], (M @ kc.abs()[:, :, None])[..., 0]
            if D is not None:
                out[b, t] += D.double().cpu()[:, None] * x[b, t]
                mass[b, t] += (D.double().cpu()[:, None] * x[b, t]).abs()
        fin[n], fmass[n] = S, M
    return out, mass, fin, fmass


def gated(x, gate, weight, eps, act, gate_first):
    x, g, w = x.double().cpu(), gate.double().cpu(), weight.double().cpu()
    a = torch.sigmoid(g) * (g if act == "silu" else 1.0)
    u = x * a if gate_first else x
    u = u / torch.sqrt(u.square().mean(-1, keepdim=True) + eps) * w
    return u if gate_first else u * a


def add(x, residual, weight, scale, eps):
    h = residual.double().cpu() + scale * x.double().cpu()
    return h / torch.sqrt(h.square().mean(-1, keepdim=True) + eps) * weight.double().cpu(), h


def off(got, want, bound):
    """How far `got` is outside `bound` (elementwise, absolute): at most 1 where it is inside."""
    return ((got.double().cpu() - want).abs() / bound.clamp_min(1e-300)).max().item() if want.numel() else 0.0


def columns(t, left=8, right=16):
    """The same values as columns of a wider tensor (tokens a different distance apart)."""
    flat = t.reshape(*t.shape[:2], -1)
    wide = torch.full((*flat.shape[:2], left + flat.shape[2] + right), float("nan"), dtype=t.dtype, device=t.device)
    view = wide[..., left:left + flat.shape[2]]
    view.copy_(flat)
    return view.unflatten(-1, t.shape[2:]) if t.dim() > 3 else view
