"""GPU: the selective state space scan against its 64-bit form, token by token."""
import math

import pytest
import torch

import flash_kda
import flashkda_b200 as F
import layer_ref as R

pytestmark = pytest.mark.gpu
bf16, fp32 = torch.bfloat16, torch.float32
DTYPES = {"bf16": bf16, "fp32": fp32}
STEP = 16                 # sequences of at most so many tokens are computed in fp32 throughout


def inputs(B, T, H, P, G, Ns, seed=0, regime="usual", state=None, N=None, skip=True):
    gen = torch.Generator().manual_seed(seed)

    def randn(*shape, dtype=bf16, std=1.0):
        return (torch.randn(*shape, generator=gen) * std).to(dtype).cuda()
    x, dt = randn(B, T, H, P), randn(B, T, H, std=0.5)
    Bm, Cm = randn(B, T, G, Ns), randn(B, T, G, Ns)
    step = torch.exp(torch.empty(H).uniform_(math.log(1e-3), math.log(1e-1), generator=gen))
    dt_bias = (step + torch.log(-torch.expm1(-step))).cuda()
    A_log = torch.log(torch.empty(H).uniform_(1.0, 16.0, generator=gen)).cuda()
    if regime == "forgets":                      # everything gone within a few tokens
        dt_bias = torch.full((H,), 3.0, device="cuda")
    elif regime == "keeps":                      # no decay to speak of
        A_log = torch.full((H,), -8.0, device="cuda")
    elif regime == "wide":                       # step sizes from 1e-9 to 20 from token to token
        dt = randn(B, T, H, std=8.0)
    x0 = randn(B if N is None else N, H, P, Ns, dtype=DTYPES[state], std=0.5) if state else None
    D = randn(H, dtype=fp32) if skip else None
    return x, dt, Bm, Cm, A_log, dt_bias, D, x0


def exponent_slack(A_log, dt, dt_bias, lens):
    """How far the exponents may be off, absolute: each is a sum of fp32 terms, at most a block of 128 tokens long, whose partial sums are each rounded; an exponential
    of it has that relative error where it is not negligible.  (Exponents beyond 40 weigh less than 2^-57 and do not matter.)"""
    return 160 * R.FP32 * 40


def check(got, fin, want, mass, last, lmass, longest, lens_rows, state_bf16, slack):
    """`out`: one rounding to bf16; where the scan goes in blocks, the products C B^T (with decay) and the state are operands
    rounded to bf16, half a step each of every term.  fp32: sums of up to 128 + Ns terms per block and the exponents.  The state is a sum of terms x w B with
    w and x w each split in two bf16 parts: 2^-16 of a term for what w loses, and half a step of a second part that is at most 2^-7 of the term, 2^-15; it is
    rescaled once per block in fp32."""
    blocks = max(1, -(-longest // 128))
    single = (400 + 4 * blocks) * R.FP32 + slack
    operands = 0.0 if longest <= STEP else 2 * R.BF16
    assert R.off(got, want, R.BF16 * want.abs() + (operands + single) * mass + 1e-30) <= 1
    # roundings of both signs do not add up: over all of `out`, three roundings' worth of half a step
    if longest > STEP:
        assert ((got.double().cpu() - want).norm() / want.norm().clamp_min(1e-30)).item() <= 3 * R.BF16
    if fin is not None:
        split = 0.0 if longest <= STEP else 3 * 2.0 ** -16
        assert R.off(fin, last, (R.BF16 if state_bf16 else R.FP32) * last.abs() + (split + single) * lmass + 1e-30) <= 1


CASES = [
    (1, 1, 1, 64, 1, 64, "fp32", "usual"), (2, 1, 32, 64, 1, 128, "fp32", "usual"), (3, 1, 5, 128, 5, 64, "bf16", "usual"), (2, 4, 4, 128, 2, 128, "fp32", "wide"), (2, 8, 3, 64, 1, 128, "bf16", "usual"),
    (1, 9, 2, 64, 1, 128, "fp32", "usual"), (1, 16, 2, 64, 1, 128, "fp32", "usual"), (1, 17, 2, 64, 1, 128, "fp32", "usual"), (2, 31, 3, 64, 3, 64, "fp32", "usual"), (1, 127, 2, 64, 2, 128, "bf16", "usual"), (1, 128, 1, 128, 1, 128, "fp32", "usual"), (2, 129, 4, 64, 2, 128, "fp32", "usual"),
    (1, 257, 3, 128, 1, 64, "fp32", "usual"), (2, 300, 5, 64, 1, 128, "bf16", "wide"), (1, 520, 2, 64, 1, 64, "fp32", "forgets"), (1, 777, 4, 64, 1, 128, "fp32", "keeps"), (1, 1100, 1, 128, 1, 128, "bf16", "wide"),
    (1, 333, 6, 64, 2, 128, None, "usual"), (3, 200, 7, 64, 7, 128, "fp32", "wide")]


@pytest.mark.parametrize("B,T,H,P,G,Ns,state,regime", CASES)
def test_equal_lengths(B, T, H, P, G, Ns, state, regime):
    x, dt, Bm, Cm, A_log, dt_bias, D, x0 = inputs(B, T, H, P, G, Ns, seed=T, regime=regime, state=state, skip=T % 2 == 0)
    want, mass, last, lmass = R.ssm(x, dt, Bm, Cm, A_log, dt_bias, D, x0, None)
    out = torch.full_like(x, float("nan"))
    fin = torch.full_like(x0, float("nan")) if state else None
    F.ssm_fwd(x, dt, Bm, Cm, out, A_log, dt_bias, D, initial_state=x0, final_state=fin)
    check(out, fin, want, mass, last, lmass, T, None, state == "bf16", exponent_slack(A_log, dt, dt_bias, None))
    # columns of wider tensors, and the state updated in place: the same bits
    outs = R.columns(torch.zeros_like(x), 16, 8)
    F.ssm_fwd(R.columns(x), R.columns(dt, 3, 4), R.columns(Bm), R.columns(Cm, 24, 0), outs, A_log, dt_bias, D, initial_state=x0, final_state=x0)
    assert torch.equal(outs, out) and (fin is None or torch.equal(x0, fin))


@pytest.mark.parametrize("state_in,state_out", [(None, "fp32"), (None, "bf16"), ("fp32", None), ("bf16", None)])
@pytest.mark.parametrize("T", [1, 150])
def test_state_in_or_out_alone(state_in, state_out, T):
    x, dt, Bm, Cm, A_log, dt_bias, D, x0 = inputs(2, T, 4, 64, 1, 128, seed=3, state=state_in)
    want, mass, last, lmass = R.ssm(x, dt, Bm, Cm, A_log, dt_bias, D, x0, None)
    out = torch.full_like(x, float("nan"))
    fin = torch.full((2, 4, 64, 128), float("nan"), dtype=DTYPES[state_out], device="cuda") if state_out else None
    F.ssm_fwd(x, dt, Bm, Cm, out, A_log, dt_bias, D, initial_state=x0, final_state=fin)
    check(out, fin, want, mass, last, lmass, T, None, state_out == "bf16", exponent_slack(A_log, dt, dt_bias, None))


PACKED = [
    ([1], 4, 64, 1, 128, "fp32", 0), ([0, 0], 2, 64, 1, 64, "fp32", 3), ([5, 1, 0, 2, 8, 0], 3, 64, 3, 128, "bf16", 7), ([130, 1, 0, 200, 9, 64], 4, 64, 2, 128, "fp32", 150), ([17, 16, 0, 15, 18], 4, 64, 2, 128, "fp32", 3), ([1] * 20 + [300, 129], 5, 64, 1, 128, "bf16", 5),
    ([128, 256, 1], 2, 128, 1, 64, "fp32", 1), ([17, 600, 90], 3, 128, 3, 128, None, 40), ([1000], 2, 64, 2, 64, "fp32", 0)]


@pytest.mark.parametrize("lens,H,P,G,Ns,state,surplus", PACKED)
def test_packed(lens, H, P, G, Ns, state, surplus):
    T, N = sum(lens) + surplus, len(lens)
    cu = torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), device="cuda")
    x, dt, Bm, Cm, A_log, dt_bias, D, x0 = inputs(1, T, H, P, G, Ns, seed=N, state=state, N=N)
    n = sum(lens)
    for t in (x, dt, Bm, Cm):
        t[:, n:] = float("nan")                                  # nobody's rows
    want, mass, last, lmass = R.ssm(x, dt, Bm, Cm, A_log, dt_bias, D, x0, cu.cpu())
    out = torch.full_like(x, 7.0)
    fin = torch.full_like(x0, float("nan")) if state else None
    F.ssm_fwd(x, dt, Bm, Cm, out, A_log, dt_bias, D, initial_state=x0, final_state=fin, cu_seqlens=cu)
    assert bool((out[:, n:] == 7.0).all())
    check(out[:, :n], fin, want[:, :n], mass[:, :n], last, lmass, max(lens), None, state == "bf16", exponent_slack(A_log, dt, dt_bias, None))
    if state:
        F.ssm_fwd(x, dt, Bm, Cm, torch.full_like(x, 7.0), A_log, dt_bias, D, initial_state=x0, final_state=x0, cu_seqlens=cu)
        assert torch.equal(x0, fin)


@pytest.mark.parametrize("P,Ns,H,G", [(64, 128, 32, 1), (64, 64, 19, 1), (128, 128, 16, 2)])
def test_more_walks_than_multiprocessors(P, Ns, H, G):
    """Each CTA takes one walk after the other, of different lengths: what a sequence gives alone, within the roundings of both (it may be cut into other runs)."""
    lens = [int(v) for v in torch.randint(17, 1500, (30,), generator=torch.Generator().manual_seed(P + Ns))]
    N, T = len(lens), sum(lens)
    cu = torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), device="cuda")
    x, dt, Bm, Cm, A_log, dt_bias, D, x0 = inputs(1, T, H, P, G, Ns, seed=5, state="fp32", N=N)
    results = []
    for _ in range(3):
        out, fin = torch.full_like(x, float("nan")), torch.full_like(x0, float("nan"))
        F.ssm_fwd(x, dt, Bm, Cm, out, A_log, dt_bias, D, initial_state=x0, final_state=fin, cu_seqlens=cu)
        results.append((out, fin))
    assert all(torch.equal(o, results[0][0]) and torch.equal(f, results[0][1]) for o, f in results)
    for n in range(0, N, 3):
        a, b = int(cu[n]), int(cu[n + 1])
        alone, last = torch.empty_like(x[:, a:b]), torch.empty_like(x0[n:n + 1])
        F.ssm_fwd(x[:, a:b], dt[:, a:b], Bm[:, a:b], Cm[:, a:b], alone, A_log, dt_bias, D, initial_state=x0[n:n + 1].contiguous(), final_state=last)
        # each is off by three roundings of its operands and result to bf16 at most (their norms), states by three of 2^-16
        assert ((out[:, a:b].double() - alone.double()).norm() / alone.double().norm()).item() <= 2 * 3 * R.BF16
        assert ((fin[n] - last[0]).double().norm() / last.double().norm()).item() <= 2 * 3 * 2.0 ** -16 + 2.0 ** -16


def test_no_tokens_hands_the_state_on():
    x, dt, Bm, Cm, A_log, dt_bias, D, x0 = inputs(2, 0, 4, 64, 1, 128, state="fp32")
    fin = torch.empty_like(x0)
    F.ssm_fwd(x, dt, Bm, Cm, torch.empty_like(x), A_log, dt_bias, D, initial_state=x0, final_state=fin)
    assert torch.equal(fin, x0)


def test_sequences_do_not_see_each_other():
    """What is not finite in one sequence, in the rows behind the last one or in a neighbour's state stays there."""
    lens = [140, 5, 131, 3]
    cu = torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), device="cuda")
    x, dt, Bm, Cm, A_log, dt_bias, D, x0 = inputs(1, sum(lens), 4, 64, 1, 128, seed=9, state="fp32", N=4)
    out, fin = torch.empty_like(x), torch.empty_like(x0)
    F.ssm_fwd(x, dt, Bm, Cm, out, A_log, dt_bias, D, initial_state=x0, final_state=fin, cu_seqlens=cu)
    for bad in (float("nan"), float("inf")):
        y, yout, yfin = [t.clone() for t in (x, Bm, Cm)], torch.empty_like(x), torch.empty_like(x0)
        s0 = x0.clone()
        for t in y:
            t[:, 140:145] = bad
            t[:, 276:] = bad
        s0[1] = bad
        F.ssm_fwd(y[0], dt, y[1], y[2], yout, A_log, dt_bias, D, initial_state=s0, final_state=yfin, cu_seqlens=cu)
        for a, e, n in ((0, 140, 0), (145, 276, 2)):
            assert torch.equal(yout[:, a:e], out[:, a:e]) and torch.equal(yfin[n], fin[n])
        assert not torch.isfinite(yout[:, 140:145].float()).any()


def test_chained_calls_equal_one_call():
    """A prompt in pieces with the state handed over, then single tokens: the whole prompt at once."""
    x, dt, Bm, Cm, A_log, dt_bias, D, x0 = inputs(2, 400, 4, 64, 2, 128, seed=4, state="fp32")
    whole, fin = torch.empty_like(x), torch.empty_like(x0)
    F.ssm_fwd(x, dt, Bm, Cm, whole, A_log, dt_bias, D, initial_state=x0, final_state=fin)
    want, mass, last, lmass = R.ssm(x, dt, Bm, Cm, A_log, dt_bias, D, x0, None)
    out, state = torch.empty_like(x), x0.clone()
    cuts = [0, 128, 131, 390] + list(range(391, 401))
    for a, e in zip(cuts[:-1], cuts[1:]):
        F.ssm_fwd(x[:, a:e], dt[:, a:e], Bm[:, a:e], Cm[:, a:e], out[:, a:e], A_log, dt_bias, D, initial_state=state, final_state=state)
    slack = exponent_slack(A_log, dt, dt_bias, None)
    check(out, state, want, mass, last, lmass, 400, None, False, slack)
    check(whole, fin, want, mass, last, lmass, 400, None, False, slack)
