"""GPU: short convolution, gated norm and residual norm against their 64-bit forms."""
import pytest
import torch

import flashkda_b200 as F
import layer_ref as R

pytestmark = pytest.mark.gpu
bf16, fp32 = torch.bfloat16, torch.float32


def randn(*shape, dtype=bf16, seed=0, std=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype).cuda()


def conv_bound(y, mass, silu):
    """One rounding to bf16; five operations in fp32 per term; SiLU: its slope is below 1.1, and its fp32 evaluation (an exponential, a
    reciprocal, two products: 16 steps of 2^-24 are ample) is relative to the sum of the terms at most."""
    return R.BF16 * y.abs() + 1.1 * 8 * R.FP32 * mass + (16 * R.FP32 * mass if silu else 0) + 1e-30


@pytest.mark.parametrize("B,T,C,W,silu,bias,wtype,state", [
    (1, 1, 8, 4, True, True, bf16, "apart"), (3, 1, 72, 4, True, False, bf16, "same"), (2, 2, 64, 4, False, True, fp32, "same"), (2, 3, 64, 3, True, True, bf16, "same"),
    (5, 5, 24, 2, True, True, fp32, "apart"), (2, 17, 1032, 4, True, True, bf16, "out"), (1, 777, 256, 4, True, True, fp32, "in"), (4, 64, 2048, 4, True, False, bf16, None),
    (2, 33, 8, 2, False, False, bf16, "apart"), (2, 0, 16, 4, True, True, bf16, "apart"), (1, 4096, 1024, 4, True, True, bf16, "same"), (64, 1, 4096, 3, True, True, bf16, "same"),
    (3, 100, 200, 3, True, True, fp32, "same")])
def test_short_conv_equal_lengths(B, T, C, W, silu, bias, wtype, state):
    x, w = randn(B, T, C, seed=1), randn(C, W, dtype=wtype, seed=2, std=0.5)
    b = randn(C, dtype=wtype, seed=3) if bias else None
    x0 = randn(B, W - 1, C, seed=4) if state in ("apart", "same", "in") else None
    fin = torch.full((B, W - 1, C), float("nan"), dtype=bf16, device="cuda") if state in ("apart", "out") else None
    want, mass, last = R.conv(x, w, b, x0, None, silu)
    if state == "same":
        fin = x0
    out = torch.full_like(x, float("nan"))
    F.short_conv(x, w, out, b, initial_state=x0, final_state=fin, silu=silu)
    assert R.off(out, want, conv_bound(want, mass, silu)) <= 1
    if fin is not None:
        assert torch.equal(fin.cpu().double(), last)                # inputs, copied


@pytest.mark.parametrize("lens,C,W,state,surplus", [
    ([1], 64, 4, "same", 0), ([5, 1, 0, 2, 40, 0, 0, 3, 1, 1, 17], 72, 4, "same", 9), ([0, 0, 300, 0], 136, 3, "apart", 5), ([3] * 50, 8, 4, "same", 0), ([2] * 33 + [0], 512, 2, "apart", 1),
    ([1] * 129, 256, 4, "same", 3), ([0, 0], 64, 4, "apart", 4), ([1000, 7, 512, 100], 2048, 4, None, 0), ([4, 4, 4, 5, 6, 7, 8, 9, 15, 16, 17], 1024, 4, "same", 2)])
def test_short_conv_packed(lens, C, W, state, surplus):
    T = sum(lens) + surplus
    cu = torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), device="cuda")
    x, w, b = randn(1, T, C, seed=1), randn(C, W, seed=2, std=0.5), randn(C, seed=3)
    x0 = randn(len(lens), W - 1, C, seed=4) if state else None
    fin = x0 if state == "same" else torch.full_like(x0, float("nan")) if state else None
    want, mass, last = R.conv(x, w, b, x0, cu.cpu(), True)
    out = torch.full_like(x, 7.0)
    F.short_conv(x, w, out, b, initial_state=x0, final_state=fin, cu_seqlens=cu)
    n = sum(lens)
    assert R.off(out[:, :n], want[:, :n], conv_bound(want, mass, True)[:, :n]) <= 1
    assert bool((out[:, n:] == 7.0).all())                          # rows behind the last sequence are left as they were
    if fin is not None:
        assert torch.equal(fin.cpu().double(), last)


def test_short_conv_first_sequence_may_start_late():
    cu = torch.tensor([5, 9, 30], device="cuda")
    x, w = randn(1, 40, 64, seed=1), randn(64, 4, seed=2)
    x[:, :5] = float("nan")                                         # nobody's rows
    out = torch.full_like(x, 3.0)
    F.short_conv(x, w, out, cu_seqlens=cu)
    want, mass, _ = R.conv(x, w, None, None, cu.cpu(), True)
    assert R.off(out[:, 5:30], want[:, 5:30], conv_bound(want, mass, True)[:, 5:30]) <= 1
    assert bool((out[:, :5] == 3.0).all()) and bool((out[:, 30:] == 3.0).all())


@pytest.mark.parametrize("B,T", [(1, 9), (3, 20), (7, 1)])
def test_short_conv_columns_of_wider_tensors(B, T):
    x, w = randn(B, T, 40, seed=1), randn(40, 4, seed=2)
    apart = torch.empty_like(x)
    F.short_conv(x, w, apart)
    xs, outs = R.columns(x), R.columns(torch.zeros_like(x))
    whole = outs._base if outs._base is not None else outs
    F.short_conv(xs, w, outs)
    assert torch.equal(outs, apart)
    assert int(torch.isnan(whole).sum()) == B * T * 24               # nothing beside the columns was written
    # x and out as columns of one tensor, beside each other
    both = torch.zeros(B, T, 80, dtype=bf16, device="cuda")
    both[..., :40] = x
    F.short_conv(both[..., :40], w, both[..., 40:])
    assert torch.equal(both[..., 40:], apart) and torch.equal(both[..., :40], x)
    # tokens first: [T][B][C] seen as [B, T, C]
    turned = x.transpose(0, 1).contiguous().transpose(0, 1)
    out = torch.empty_like(turned)
    F.short_conv(turned, w, out)
    assert torch.equal(out, apart)


def test_short_conv_not_finite_stays_in_its_sequence_and_channel():
    x, w = randn(2, 20, 16, seed=1), randn(16, 4, seed=2)
    x[0, 10, 3] = float("nan")
    out = torch.empty_like(x)
    F.short_conv(x, w, out)
    bad = torch.zeros(2, 20, 16, dtype=torch.bool)
    bad[0, 10:14, 3] = True
    assert torch.equal(torch.isnan(out).cpu(), bad)


def norm_bound(y):
    """One rounding to bf16.  In fp32: the sum of squares and its root (half of 24 + 3 steps, whatever the order: the terms are positive and a thread adds 32 and
    thirty-two threads or warps five more), the gate's exponential and reciprocal, five products: 64 steps of 2^-24 are ample."""
    return (R.BF16 + 64 * R.FP32) * y.abs() + 1e-30


@pytest.mark.parametrize("act", ["sigmoid", "silu"])
@pytest.mark.parametrize("gate_first", [False, True])
@pytest.mark.parametrize("B,T,H,D,per_head,wtype", [
    (1, 1, 1, 8, False, fp32), (1, 1, 3, 64, True, bf16), (2, 5, 3, 72, False, bf16), (1, 7, 32, 128, False, fp32), (3, 1, 2, 200, True, fp32), (2, 3, 1, 264, False, bf16), (1, 9, 5, 520, True, bf16),
    (1, 3, 1, 1024, False, fp32), (1, 5, 1, 1032, False, bf16), (2, 2, 2, 2056, True, fp32), (1, 3, 1, 4096, False, bf16), (1, 2, 1, 8200, False, fp32), (1, 1, 1, 16384, False, bf16)])
def test_gated_norm(act, gate_first, B, T, H, D, per_head, wtype):
    x, g = randn(B, T, H, D, seed=1), randn(B, T, H, D, seed=2, std=2.0)
    w = randn(*((H, D) if per_head else (D,)), dtype=wtype, seed=3)
    out = torch.full_like(x, float("nan"))
    want = R.gated(x, g, w, 1e-5, act, gate_first)
    F.gated_norm(R.columns(x), R.columns(g, 16, 0), w, out, eps=1e-5, act=act, gate_first=gate_first)
    assert R.off(out, want, norm_bound(want)) <= 1
    for into in (x.clone(), g.clone()):                             # in place, over either input
        F.gated_norm(into if torch.equal(into, x) else x, into if torch.equal(into, g) else g, w, into, eps=1e-5, act=act, gate_first=gate_first)
        assert torch.equal(into, out)


def test_gated_norm_of_zeros_and_large_values():
    x = torch.zeros(1, 3, 1, 128, dtype=bf16, device="cuda")
    x[0, 1] = 1e15
    g, w = torch.full_like(x, 200.0), torch.ones(128, device="cuda")
    g[0, 2] = -200.0
    out = torch.empty_like(x)
    F.gated_norm(x, g, w, out, eps=1e-6)
    assert bool((out[0, 0] == 0).all()) and bool((out[0, 2] == 0).all()) and bool((out[0, 1] == 1).all())


@pytest.mark.parametrize("rtype", [bf16, fp32])
@pytest.mark.parametrize("B,T,D,wtype,scale", [(1, 1, 8, bf16, 1.0), (3, 1, 72, fp32, 0.5), (2, 9, 128, bf16, 1.0), (1, 5, 1000, fp32, -0.3), (2, 3, 1032, bf16, 1.0), (1, 7, 4096, bf16, 0.22),
                                               (1, 2, 8192, fp32, 0.0), (1, 3, 16384, bf16, 1.0)])
def test_add_norm(rtype, B, T, D, wtype, scale):
    x, r, w = randn(B, T, D, seed=1), randn(B, T, D, dtype=rtype, seed=2, std=3.0), randn(D, dtype=wtype, seed=3)
    out, ro = torch.full_like(x, float("nan")), torch.full_like(r, float("nan"))
    want, h = R.add(x, r, w, scale, 1e-5)
    F.add_norm(R.columns(x), R.columns(r), w, out, ro, scale=scale, eps=1e-5)
    # h: a product with `scale` rounded to fp32 and one fused operation, where the terms may cancel; then the rounding of its type
    slack = 3 * R.FP32 * (r.double().cpu().abs() + (scale * x.double().cpu()).abs())
    assert R.off(ro, h, (R.BF16 if rtype == bf16 else R.FP32) * h.abs() + slack + 1e-30) <= 1
    root = torch.sqrt(h.square().mean(-1, keepdim=True) + 1e-5)
    assert R.off(out, want, norm_bound(want) + 2 * slack / root * w.double().cpu().abs()) <= 1
    xi, ri = x.clone(), r.clone()                                   # in place
    F.add_norm(xi, ri, w, xi, ri, scale=scale, eps=1e-5)
    assert torch.equal(xi, out) and torch.equal(ri, ro)


def test_norms_leave_what_is_not_theirs():
    x, g, w = randn(2, 3, 2, 72, seed=1), randn(2, 3, 2, 72, seed=2), randn(72, seed=3)
    wide = torch.full((2, 3, 160), float("nan"), dtype=bf16, device="cuda")
    F.gated_norm(x, g, w, wide[..., 8:152].unflatten(-1, (2, 72)))
    assert int(torch.isnan(wide).sum()) == 2 * 3 * 16
    empty = torch.empty(2, 0, 72, dtype=bf16, device="cuda")
    F.add_norm(empty, empty, w, empty.clone(), empty.clone())
