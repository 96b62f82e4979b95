"""GPU: batches of the operators round the recurrence at the edges of their planning - many packed sequences, cu_seqlens that are not in order - and waits
of the scan that run out."""
import ctypes

import pytest
import torch

import flashkda_b200 as F
import layer_ref as R
from flashkda_b200 import _binding, _layer
from test_gpu_conv_norm import randn
from test_gpu_ssm import check, exponent_slack, inputs

pytestmark = pytest.mark.gpu
bf16, fp32 = torch.bfloat16, torch.float32


def ssm_many(x, dt, Bm, Cm, A_log, dt_bias, D, x0, lens):
    """As R.ssm for a packed batch with one group, all sequences a token at a time."""
    x, dt, Bm, Cm = (t[0].double() for t in (x, dt, Bm, Cm))
    lens = torch.tensor(lens, device="cuda")
    first, A = lens.cumsum(0) - lens, torch.exp(A_log.double())
    S, out = x0.double(), torch.zeros_like(x)
    M, mass = S.abs(), torch.zeros_like(x)
    for t in range(int(lens.max())):
        n = (lens > t).nonzero()[:, 0]
        at = first[n] + t
        delta = R.softplus(dt[at] + dt_bias.double())
        decay = torch.exp(-A * delta)[..., None, None]
        add = (delta[..., None] * x[at])[..., None] * Bm[at][:, :, None]
        S[n], M[n] = decay * S[n] + add, decay * M[n] + add.abs()
        out[at] = (S[n] @ Cm[at][..., None])[..., 0] + D.double()[:, None] * x[at]
        mass[at] = (M[n] @ Cm[at].abs()[..., None])[..., 0] + (D.double()[:, None] * x[at]).abs()
    return out[None].cpu(), mass[None].cpu(), S.cpu(), M.cpu()


@pytest.mark.parametrize("n,lo,hi,longer,H", [(600, 17, 20, [300, 1500], 1), (600, 1, 40, [], 2), (2100, 17, 20, [1300], 1), (2100, 1, 20, [200, 3], 1)])
def test_many_sequences(n, lo, hi, longer, H):
    """More than the plan's threads, and more than it sorts; a longer one among them."""
    gen = torch.Generator().manual_seed(n + lo)
    lens = torch.randint(lo, hi + 1, (n,), generator=gen).tolist()
    lens = lens[:n // 3] + longer + lens[n // 3:]
    cu = torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), device="cuda")
    x, dt, Bm, Cm, A_log, dt_bias, D, x0 = inputs(1, sum(lens), H, 64, 1, 64, seed=n, state="fp32", N=len(lens))
    want, mass, last, lmass = ssm_many(x, dt, Bm, Cm, A_log, dt_bias, D, x0, lens)
    out, fin = torch.full_like(x, float("nan")), torch.full_like(x0, float("nan"))
    args = (x, dt, Bm, Cm, out, A_log, dt_bias, D, x0, fin, cu)
    ws = torch.empty(F.ssm_workspace_size(*args), dtype=torch.uint8, device="cuda")
    F.ssm_fwd(*args, workspace=ws)
    assert F.read_status(ws) == 0
    check(out, fin, want, mass, last, lmass, max(lens), None, False, exponent_slack(A_log, dt, dt_bias, None))


def guarded(nbytes):
    buf = torch.full((8192 + nbytes,), 0x5A, dtype=torch.uint8, device="cuda")
    return buf, buf[4096:4096 + nbytes]


BAD = [[-3, 400, 380], [0, 200, 1000, 300], [0, 100, 90, 1 << 40, 400], [-(1 << 40), -5, 400, 100], [500, 600, 700], [0, 400, 0, 400, 100], [399, 17, 401, 2], [20, -20, 20, 420]]


@pytest.mark.parametrize("bad", BAD)
@pytest.mark.parametrize("T", [400, 12])
def test_bad_cu_seqlens_of_a_scan_stay_in_bounds(bad, T):
    x, dt, Bm, Cm, A_log, dt_bias, D, x0 = inputs(1, T, 2, 64, 1, 128, state="fp32", N=len(bad) - 1)
    buf_o, o = guarded(x.numel() * 2)
    buf_f, f = guarded(x0.numel() * 4)
    args = [x, dt, Bm, Cm, o.view(bf16).view(x.shape), A_log, dt_bias, D, x0, f.view(fp32).view(x0.shape), torch.tensor(bad, device="cuda")]
    need = F.ssm_workspace_size(*args)
    buf_w, ws = guarded(max(need, 256))
    F.ssm_fwd(*args, workspace=ws)
    with pytest.raises(RuntimeError, match="not monotone"):
        F.read_status(ws)
    for buf, n in ((buf_o, o.numel()), (buf_f, f.numel()), (buf_w, ws.numel())):
        assert bool((buf[:4096] == 0x5A).all()) and bool((buf[4096 + n:] == 0x5A).all())


@pytest.mark.parametrize("bad", BAD)
@pytest.mark.parametrize("T,W", [(400, 4), (12, 2)])
def test_bad_cu_seqlens_of_a_convolution_stay_in_bounds(bad, T, W):
    x, w, x0 = randn(1, T, 72, seed=1), randn(72, W, seed=2), randn(len(bad) - 1, W - 1, 72, seed=3)
    buf_o, o = guarded(x.numel() * 2)
    buf_f, f = guarded(x0.numel() * 2)
    F.short_conv(x, w, o.view(bf16).view(x.shape), initial_state=x0, final_state=f.view(bf16).view(x0.shape), cu_seqlens=torch.tensor(bad, device="cuda"))
    torch.cuda.synchronize()
    for buf, n in ((buf_o, o.numel()), (buf_f, f.numel())):
        assert bool((buf[:4096] == 0x5A).all()) and bool((buf[4096 + n:] == 0x5A).all())


@pytest.mark.parametrize("B,T,H,P,lens,stop", [(8, 300, 64, 64, None, 1), (1, 900, 64, 64, None, 1), (1, 900, 4, 64, [300, 5, 280, 315], 1)])
def test_a_wait_that_runs_out_with_states_in_bf16(B, T, H, P, lens, stop):
    """As with states in fp32, which the scan keeps in another form: the status says so, and the next call is as the one before."""
    N = B if lens is None else len(lens)
    cu = None if lens is None else torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), device="cuda")
    x, dt, Bm, Cm, A_log, dt_bias, D, x0 = inputs(B, T, H, P, 1, 128, state="bf16", N=N)
    before, fin = torch.empty_like(x), torch.empty_like(x0)
    F.ssm_fwd(x, dt, Bm, Cm, before, A_log, dt_bias, D, x0, fin, cu)
    out, fin2 = torch.empty_like(x), torch.empty_like(x0)
    args = (x, dt, Bm, Cm, out, A_log, dt_bias, D, x0, fin2, cu)
    ws = torch.zeros(F.ssm_workspace_size(*args), dtype=torch.uint8, device="cuda")
    p = _layer._ssm_params(*args)
    p.workspace, p.workspace_bytes = ws.data_ptr(), ws.numel()
    give_up = _layer._lib().fkda_debug_ssm_giveup
    give_up.argtypes, give_up.restype = [ctypes.POINTER(_layer.SsmParams), ctypes.c_int, ctypes.c_int, ctypes.c_void_p], ctypes.c_int
    assert give_up(ctypes.byref(p), stop, 3000, _binding._stream(x)) == 0
    with pytest.raises(RuntimeError, match="gave up"):
        F.read_status(ws)
    F.ssm_fwd(*args, workspace=ws)
    assert F.read_status(ws) == 0
    assert torch.equal(out, before) and torch.equal(fin, fin2)


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("state", ["bf16", None])
@pytest.mark.parametrize("T,P,lens", [(1500, 64, None), (700, 128, None), (20, 64, None), (1, 64, [700, 3, 900, 17])])
def test_inputs_and_states_in_bf16_that_the_kernel_before_wrote(T, P, lens, state, captured):
    """The scan's launches overlap: inputs written, a scan, another over the same buffers, again and again, give what each gives alone."""
    n = T if lens is None else sum(lens)
    cu = None if lens is None else torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), device="cuda")
    sets = [inputs(1, n, 2, P, 1, 128, seed=s, state=state, N=1 if lens is None else len(lens)) for s in (1, 2)]
    x, dt, Bm, Cm, A_log, dt_bias, D, x0 = [t.clone() if t is not None else None for t in sets[0]]
    out = torch.empty_like(x)

    def run():
        F.ssm_fwd(x, dt, Bm, Cm, out, A_log, dt_bias, D, initial_state=x0, final_state=x0, cu_seqlens=cu)
        x.copy_(out.clamp(-4, 4))
        F.ssm_fwd(x, dt, Bm, Cm, out, A_log, dt_bias, D, initial_state=x0, final_state=x0, cu_seqlens=cu)

    def load(s):
        for to, t in zip((x, dt, Bm, Cm, A_log, dt_bias, D, x0), s):
            if t is not None:
                to.copy_(t)

    want = []
    for s in sets:
        load(s)
        torch.cuda.synchronize()
        run()
        torch.cuda.synchronize()
        want.append((out.clone(), x0.clone() if x0 is not None else out))
    if captured:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            run()
    got = []
    for i in range(10):
        load(sets[i & 1])
        graph.replay() if captured else run()
        got.append((out.clone(), x0.clone() if x0 is not None else want[i & 1][1]))
    for i, (o, f) in enumerate(got):
        assert torch.equal(o, want[i & 1][0]) and torch.equal(f, want[i & 1][1])
