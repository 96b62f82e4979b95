"""GPU: the operators round the recurrence where their numbers get hard - resets, products that overflow on the way, states as exact as their type - and where a call follows one that failed."""
import pytest
import torch

import flashkda_b200 as F
import layer_ref as R
from test_gpu_conv_norm import norm_bound, randn
from test_gpu_ssm import check, exponent_slack, inputs

pytestmark = pytest.mark.gpu
bf16, fp32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("act", ["sigmoid", "silu"])
@pytest.mark.parametrize("gate_first", [False, True])
@pytest.mark.parametrize("D", [64, 128, 1032])
def test_gated_norm_where_x_times_gate_overflows(act, gate_first, D):
    """|x gate| beyond the largest fp32 while the activation is 0, or in rows that are large throughout."""
    x, g, w = randn(1, 6, 3, D, seed=1), randn(1, 6, 3, D, seed=2, std=2.0), randn(D, dtype=fp32, seed=3)
    x[0, 0, :, 5], g[0, 0, :, 5] = 1e25, -1e25                      # (alone in its row, which has the rest to show that it counts as 0 with the gate first)
    x[0, 1] *= 1e8
    g[0, 1, :, ::3] = -3e38
    x[0, 2, :, ::2], g[0, 2, :, ::2] = -2e15, -2e30
    g[0, 3] = -3e38
    out = torch.full_like(x, float("nan"))
    want = R.gated(x, g, w, 1e-5, act, gate_first)
    F.gated_norm(x, g, w, out, eps=1e-5, act=act, gate_first=gate_first)
    if not gate_first:                                              # the square of 1e25 is beyond fp32 itself, whatever the gate
        out, want = out[:, 1:], want[:, 1:]
    assert R.off(out, want, norm_bound(want)) <= 1


@pytest.mark.parametrize("bad,T", [([0, 400, 0, 400, 100], 400), ([0, 9, 300], 200)])
@pytest.mark.parametrize("lens", [None, [2, 1, 4]])
def test_status_of_a_step_behind_a_call_that_failed(bad, T, lens):
    """A fixed workspace: a good step after a batch whose cu_seqlens were bad reads as good, through every route of few tokens."""
    x, dt, Bm, Cm, A_log, dt_bias, D, _ = inputs(1, T, 2, 64, 1, 128)
    cu = torch.tensor(bad, device="cuda")
    args = (x, dt, Bm, Cm, torch.empty_like(x), A_log, dt_bias, D, None, None, cu)
    ws = torch.empty(F.ssm_workspace_size(*args), dtype=torch.uint8, device="cuda")
    F.ssm_fwd(*args, workspace=ws)
    with pytest.raises(RuntimeError, match="not monotone"):
        F.read_status(ws)
    n = 1 if lens is None else sum(lens)
    cu = None if lens is None else torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), device="cuda")
    out = torch.empty_like(x[:, :n])
    F.ssm_fwd(x[:, :n], dt[:, :n], Bm[:, :n], Cm[:, :n], out, A_log, dt_bias, D, cu_seqlens=cu, workspace=ws)
    assert F.read_status(ws) == 0
    plain = torch.empty_like(out)
    F.ssm_fwd(x[:, :n], dt[:, :n], Bm[:, :n], Cm[:, :n], plain, A_log, dt_bias, D, cu_seqlens=cu)
    assert torch.equal(out, plain)


@pytest.mark.parametrize("bad", [[0, 9, 4, 12], [0, 5, 13], [-1, 4, 12], [3, 2, 12]])
def test_bad_cu_seqlens_of_few_tokens_are_reported(bad):
    x, dt, Bm, Cm, A_log, dt_bias, D, _ = inputs(1, 12, 2, 64, 1, 128)
    ws = torch.zeros(256, dtype=torch.uint8, device="cuda")
    F.ssm_fwd(x, dt, Bm, Cm, torch.empty_like(x), A_log, dt_bias, D, cu_seqlens=torch.tensor(bad, device="cuda"), workspace=ws)
    with pytest.raises(RuntimeError, match="not monotone"):
        F.read_status(ws)
    F.ssm_fwd(x, dt, Bm, Cm, torch.empty_like(x), A_log, dt_bias, D, cu_seqlens=torch.tensor([0, 5, 12], device="cuda"), workspace=ws)
    assert F.read_status(ws) == 0


def with_resets(T, H, P, G, Ns, every, size, seed):
    """Steps of `size` at every `every`th token, of some 1e-3 between: what was before is forgotten at once, what comes behind is kept.  The resets add nothing (x = 0)."""
    x, dt, Bm, Cm, A_log, dt_bias, D, x0 = inputs(1, T, H, P, G, Ns, seed=seed, state="fp32")
    dt_bias.zero_()
    dt = (torch.randn(1, T, H, generator=torch.Generator().manual_seed(seed)) * 0.5 - 7.0).to(bf16).cuda()
    at = torch.arange(T) % every == 3
    dt[:, at] = size
    x[:, at] = 0.0
    return x, dt, Bm, Cm, A_log, dt_bias, D, x0


@pytest.mark.parametrize("size", [20.0, 300.0, 1e4, 1e6, 1e12, 1e30])
@pytest.mark.parametrize("T,every,P,Ns", [(200, 37, 64, 128), (130, 9, 128, 64), (400, 150, 64, 64)])
def test_steps_that_reset_the_state(T, every, P, Ns, size):
    """The decays between the tokens behind a reset do not depend on how far the reset went."""
    args = with_resets(T, 4, P, 2, Ns, every, size, seed=T)
    x, dt, Bm, Cm, A_log, dt_bias, D, x0 = args
    want, mass, last, lmass = R.ssm(*args, None)
    out, fin = torch.full_like(x, float("nan")), torch.full_like(x0, float("nan"))
    F.ssm_fwd(x, dt, Bm, Cm, out, A_log, dt_bias, D, initial_state=x0, final_state=fin)
    check(out, fin, want, mass, last, lmass, T, None, False, exponent_slack(A_log, dt, dt_bias, None))


@pytest.mark.parametrize("size", [1e6, 1e9, 1e12, 1e18, 1e25])
def test_large_steps_with_rates_as_small(size):
    """Steps beyond 2^27 whose decays are those of ordinary ones, on inputs as small as the steps are large."""
    x, dt, Bm, Cm, A_log, dt_bias, D, x0 = inputs(1, 150, 4, 64, 1, 128, seed=8, state="fp32")
    dt[:] = (size * torch.rand(1, 150, 4, generator=torch.Generator().manual_seed(1))).to(bf16).cuda()
    A_log = torch.log(torch.tensor([0.01, 1.0, 2.0, 4.5], dtype=torch.float64) / size).float().cuda()      # (whole 32-token blocks lose 2^-0.2 to 2^-104)
    x = (x.float() / size).to(bf16)
    want, mass, last, lmass = R.ssm(x, dt, Bm, Cm, A_log, dt_bias, D, x0, None)
    out, fin = torch.full_like(x, float("nan")), torch.full_like(x0, float("nan"))
    F.ssm_fwd(x, dt, Bm, Cm, out, A_log, dt_bias, D, initial_state=x0, final_state=fin)
    check(out, fin, want, mass, last, lmass, 150, None, False, exponent_slack(A_log, dt, dt_bias, None))


@pytest.mark.parametrize("T,B,H,P,Ns,lens", [
    (40, 1, 4, 64, 128, None), (128, 2, 3, 64, 64, None), (300, 1, 4, 128, 128, None), (200, 2, 2, 128, 64, None), (1500, 1, 2, 64, 128, None), (3000, 1, 2, 128, 64, None), (1, 1, 5, 64, 128, [17, 130, 260, 5]),
    (1, 1, 2, 64, 64, [3000])])
def test_fp32_states_are_as_exact_as_fp32(T, B, H, P, Ns, lens):
    """The last tokens, 61 apart, are there alone (x = 0 elsewhere) with a decay that is all but 1: few terms w x B, each of which has to be there with all its bits.

    In units of 2^-24: delta of arguments up to 10 in size, 32 (the sum with the bias 4, its product with log2 e and that constant 10, the exponential 4, the division 4, sums and
    products of the logarithm 10); w = delta times two powers of all but 0, 10; its product with x taken in three parts of eight bits 4; the products of
    these with B are exact, and their three sums, each rounded towards zero, 6, and that again for every term that is added behind it; decays of up to three blocks or a run, a power and a product each, 15."""
    n = T if lens is None else sum(lens)
    x, dt, Bm, Cm, A_log, dt_bias, D, _ = inputs(B, n, H, P, 1, Ns, seed=T + n)
    A_log.fill_(-14.0)
    keep = torch.zeros(n, dtype=torch.bool)
    cu = None if lens is None else torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), device="cuda")
    ends = [n] if lens is None else cu.tolist()[1:]
    first = [0] if lens is None else cu.tolist()[:-1]
    terms = 0
    for a, e in zip(first, ends):
        at = [t for t in range(e - 1, a - 1, -61)][:4]
        keep[at] = True
        terms = max(terms, len(at))
    x[:, ~keep] = 0.0
    N = B if lens is None else len(lens)
    want, mass, last, lmass = R.ssm(x, dt, Bm, Cm, A_log, dt_bias, D, None, None if cu is None else cu.cpu())
    out, fin = torch.empty_like(x), torch.full((N, H, P, Ns), float("nan"), device="cuda")
    F.ssm_fwd(x, dt, Bm, Cm, out, A_log, dt_bias, D, final_state=fin, cu_seqlens=cu)
    steps = 32 + 10 + 4 + 6 * terms + 15
    assert R.off(fin, last, steps * R.FP32 * lmass + 1e-30) <= 1


@pytest.mark.parametrize("T", [300, 3000])
@pytest.mark.parametrize("P,Ns", [(64, 128), (128, 64)])
def test_out_does_not_depend_on_the_state_that_is_asked_for(T, P, Ns):
    """An fp32 state is kept with more bits than one in bf16 or none: `out` is the same within the roundings of its operands."""
    x, dt, Bm, Cm, A_log, dt_bias, D, _ = inputs(1, T, 4, P, 2, Ns, seed=T)
    outs, fins = [], []
    for state in (fp32, bf16, None):
        outs.append(torch.full_like(x, float("nan")))
        fins.append(None if state is None else torch.empty(1, 4, P, Ns, dtype=state, device="cuda"))
        F.ssm_fwd(x, dt, Bm, Cm, outs[-1], A_log, dt_bias, D, final_state=fins[-1])
    assert torch.equal(outs[1], outs[2])
    # what differs is 2^-16 of what goes into the states: a few operands and results are rounded the other way
    assert ((outs[0].double() - outs[1].double()).norm() / outs[0].double().norm()).item() <= R.BF16
    assert ((fins[0].double() - fins[1].double()).norm() / fins[0].double().norm()).item() <= R.BF16


@pytest.mark.parametrize("B,T,H,P,G,Ns,state", [(2, 500, 4, 64, 1, 128, "fp32"), (1, 700, 2, 128, 2, 64, "bf16"), (1, 2000, 1, 64, 1, 64, "fp32")])
def test_out_as_a_whole(B, T, H, P, G, Ns, state):
    """Three roundings to bf16 - M, the state's copy, out - each off by 2^-7 / sqrt(12) of a value between 1 and 2 in the mean square; on random inputs, where neither they nor the terms
    of a sum go together, at most sqrt(3) of that, 2^-8, over all of `out`."""
    args = inputs(B, T, H, P, G, Ns, seed=T + 1, state=state)
    x, dt, Bm, Cm, A_log, dt_bias, D, x0 = args
    want = R.ssm(*args, None)[0]
    out = torch.full_like(x, float("nan"))
    F.ssm_fwd(x, dt, Bm, Cm, out, A_log, dt_bias, D, initial_state=x0, final_state=torch.empty_like(x0))
    assert ((out.double().cpu() - want).norm() / want.norm()).item() <= 2.0 ** -8
