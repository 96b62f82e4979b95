"""GPU: the operators round the recurrence as a layer uses them - one after the other, captured and replayed, on other streams - and
what they must not do: write past their tensors, answer calls that are not in order, hang when a wait gives up."""
import ctypes

import pytest
import torch

import flash_kda
import flashkda_b200 as F
import layer_ref as R
import oracle
from flashkda_b200 import _binding, _layer
from helpers import OUT_MAX_ABS, max_abs
from test_gpu_conv_norm import conv_bound, norm_bound
from test_gpu_ssm import check, exponent_slack, inputs

pytestmark = pytest.mark.gpu
bf16, fp32 = torch.bfloat16, torch.float32


def randn(*shape, dtype=bf16, seed=0, std=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype).cuda()


class ScanLayer:
    """projections' output -> convolution -> selective scan -> gated norm -> residual norm, with the states of every sequence"""

    def __init__(self, N, H=4, P=64, G=1, Ns=128, seed=0):
        self.H, self.P, self.G, self.Ns, self.C = H, P, G, Ns, H * P + 2 * G * Ns
        _, _, _, _, self.A_log, self.dt_bias, self.D, _ = inputs(1, 1, H, P, G, Ns, seed=seed)
        self.w, self.b = randn(self.C, 4, seed=seed + 1, std=0.5), randn(self.C, seed=seed + 2, std=0.1)
        self.norm, self.norm2 = randn(H * P, dtype=fp32, seed=seed + 3), randn(H * P, seed=seed + 4)
        self.conv_state = torch.zeros(N, 3, self.C, dtype=bf16, device="cuda")
        self.ssm_state = torch.zeros(N, H, P, Ns, device="cuda")

    def width(self):
        return self.H * self.P + self.C + 8                     # z | x B C | dt

    def buffers(self, B, T):
        return dict(xbc=torch.empty(B, T, self.C, dtype=bf16, device="cuda"), y=torch.empty(B, T, self.H, self.P, dtype=bf16, device="cuda"),
                    n=torch.empty(B, T, 1, self.H * self.P, dtype=bf16, device="cuda"), out=torch.empty(B, T, self.H * self.P, dtype=bf16, device="cuda"))

    def views(self, proj, buf):
        inner = self.H * self.P
        z, xbc, dt = proj[..., :inner].unflatten(-1, (1, inner)), proj[..., inner:inner + self.C], proj[..., inner + self.C:inner + self.C + self.H]
        x, Bm, Cm = (t.unflatten(-1, s) for t, s in zip(buf["xbc"].split([inner, self.G * self.Ns, self.G * self.Ns], -1), ((self.H, self.P), (self.G, self.Ns), (self.G, self.Ns))))
        return z, xbc, dt, x, Bm, Cm

    def __call__(self, proj, residual, buf, cu=None):
        z, xbc, dt, x, Bm, Cm = self.views(proj, buf)
        F.short_conv(xbc, self.w, buf["xbc"], self.b, initial_state=self.conv_state, final_state=self.conv_state, cu_seqlens=cu)
        F.ssm_fwd(x, dt, Bm, Cm, buf["y"], self.A_log, self.dt_bias, self.D, initial_state=self.ssm_state, final_state=self.ssm_state, cu_seqlens=cu)
        F.gated_norm(buf["y"].flatten(2).unsqueeze(2), z, self.norm, buf["n"], eps=1e-5, act="silu", gate_first=True)
        F.add_norm(buf["n"].squeeze(2), residual, self.norm2, buf["out"], residual, eps=1e-5)


def verify(layer, proj, residual0, residual, buf, cu, conv0, ssm0, lens):
    """Every operator of the run against its 64-bit form on what the operator before it left."""
    z, xbc, dt, x, Bm, Cm = layer.views(proj, buf)
    want, mass, last = R.conv(xbc, layer.w, layer.b, conv0, cu, True)
    assert R.off(buf["xbc"], want, conv_bound(want, mass, True)) <= 1 and torch.equal(layer.conv_state.cpu().double(), last)
    want, mass, last, lmass = R.ssm(x, dt, Bm, Cm, layer.A_log, layer.dt_bias, layer.D, ssm0, cu)
    check(buf["y"], layer.ssm_state, want, mass, last, lmass, max(lens), None, False, exponent_slack(None, None, None, None))
    want = R.gated(buf["y"].flatten(2).unsqueeze(2), z, layer.norm, 1e-5, "silu", True)
    assert R.off(buf["n"], want, norm_bound(want)) <= 1
    want, h = R.add(buf["n"].squeeze(2), residual0, layer.norm2, 1.0, 1e-5)
    slack = 3 * R.FP32 * (residual0.double().cpu().abs() + buf["n"].squeeze(2).double().cpu().abs())
    assert R.off(residual, h, R.FP32 * h.abs() + slack + 1e-30) <= 1
    assert R.off(buf["out"], want, norm_bound(want) + 2 * slack / torch.sqrt(h.square().mean(-1, keepdim=True) + 1e-5) * layer.norm2.double().cpu().abs()) <= 1


def test_a_run_of_them_prompts_then_single_tokens():
    lens = [150, 3, 40, 1, 260]
    layer = ScanLayer(len(lens))
    steps = [torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), device="cuda"), None, None]      # a packed batch, then two tokens of every sequence
    for i, cu in enumerate(steps):
        B, T = (1, sum(lens)) if cu is not None else (len(lens), 1)
        proj, residual = randn(B, T, layer.width(), seed=20 + i), randn(B, T, layer.H * layer.P, dtype=fp32, seed=30 + i, std=3.0)
        conv0, ssm0, residual0, buf = layer.conv_state.clone(), layer.ssm_state.clone(), residual.clone(), layer.buffers(B, T)
        layer(proj, residual, buf, cu)
        verify(layer, proj, residual0, residual, buf, None if cu is None else cu.cpu(), conv0, ssm0, lens if cu is not None else [1])


def test_a_kda_layer():
    """q, k, v through their convolution, `flash_kda.fwd`, the output norm with its sigmoid gate, the residual norm."""
    H, T, B = 2, 100, 2
    qkv, w = randn(B, T, 3 * H * 128, seed=1), randn(3 * H * 128, 4, seed=2, std=0.5)
    g, beta, gate, residual = randn(B, T, H, 128, seed=3), randn(B, T, H, seed=4), randn(B, T, H, 128, seed=5), randn(B, T, H * 128, seed=6)
    A_log, dt_bias, norm, norm2 = randn(H, dtype=fp32, seed=7), randn(H, 128, dtype=fp32, seed=8), randn(128, dtype=fp32, seed=9), randn(H * 128, seed=10)
    parts = [torch.empty(B, T, H, 128, dtype=bf16, device="cuda") for _ in range(3)]
    for i, t in enumerate(parts):                               # columns of one projection to three contiguous tensors
        c = slice(i * H * 128, (i + 1) * H * 128)
        F.short_conv(qkv[..., c], w[c], t.flatten(2))
        want, mass, _ = R.conv(qkv[..., c], w[c], None, None, None, True)
        assert R.off(t.flatten(2), want, conv_bound(want, mass, True)) <= 1
    o, n, out, res = torch.empty_like(gate), torch.empty_like(gate), torch.empty_like(residual), torch.empty_like(residual)
    flash_kda.fwd(*parts, g, beta, 128 ** -0.5, o, A_log, dt_bias, -5.0)
    o64, _ = oracle.recurrence_f64(*(t.cpu() for t in parts), g.cpu(), beta.cpu(), 128 ** -0.5, A_log.cpu(), dt_bias.cpu(), -5.0)
    assert max_abs(o.cpu(), o64) <= OUT_MAX_ABS
    F.gated_norm(o, gate, norm, n)
    want = R.gated(o, gate, norm, 1e-6, "sigmoid", False)
    assert R.off(n, want, norm_bound(want)) <= 1
    F.add_norm(n.flatten(2), residual, norm2, out, res)
    want, h = R.add(n.flatten(2), residual, norm2, 1.0, 1e-6)
    assert R.off(res, h, (R.BF16 + 3 * R.FP32) * h.abs() + 3 * R.FP32 * residual.double().cpu().abs() + 1e-30) <= 1


@pytest.mark.parametrize("lens", [None, [200, 1, 7, 300]])
def test_captured_and_replayed_on_new_inputs(lens):
    """States go round in place: three replays equal three ordinary calls, bit for bit; two graphs of the same layer share a memory pool."""
    N = 3 if lens is None else len(lens)
    B, T = (N, 70) if lens is None else (1, sum(lens))
    cu = None if lens is None else torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), device="cuda")
    projs = [randn(B, T, ScanLayer(N).width(), seed=40 + i) for i in range(3)]
    results = []
    for captured in (False, True):
        layer = ScanLayer(N)
        proj, residual, buf = projs[0].clone(), torch.zeros(B, T, layer.H * layer.P, device="cuda"), layer.buffers(B, T)
        if captured:
            layer(proj, residual, buf, cu)                      # (first use: outside of the capture)
            graphs = []
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            for _ in range(2):
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, pool=graphs[0].pool() if graphs else None, stream=side):
                    layer(proj, residual, buf, cu)
                graphs.append(graph)
            layer.conv_state.zero_()
            layer.ssm_state.zero_()
            residual.zero_()
        got = []
        for i, p in enumerate(projs):
            proj.copy_(p)
            if captured:
                graphs[i & 1].replay()
            else:
                layer(proj, residual, buf, cu)
            got += [buf["out"].clone(), residual.clone(), layer.conv_state.clone(), layer.ssm_state.clone()]
        results.append(got)
    for a, b in zip(*results):
        assert torch.equal(a, b)


def test_two_streams_at_once():
    """Calls on two streams, many in flight: each equals the call alone."""
    cases = []
    for s in range(2):
        T = 700 + 128 * s
        x, dt, Bm, Cm, A_log, dt_bias, D, x0 = inputs(1, T, 4, 64, 1, 128, seed=s, state="fp32")
        alone, fin = torch.empty_like(x), torch.empty_like(x0)
        F.ssm_fwd(x, dt, Bm, Cm, alone, A_log, dt_bias, D, initial_state=x0, final_state=fin)
        cases.append((x, dt, Bm, Cm, A_log, dt_bias, D, x0, alone, fin))
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in cases], [[], []]
    for _ in range(10):
        for s, (x, dt, Bm, Cm, A_log, dt_bias, D, x0, _, _) in enumerate(cases):
            with torch.cuda.stream(streams[s]):
                out, fin = torch.empty_like(x), torch.empty_like(x0)
                F.ssm_fwd(x, dt, Bm, Cm, out, A_log, dt_bias, D, initial_state=x0, final_state=fin)
                outs[s].append((out, fin))
    torch.cuda.synchronize()
    for s, case in enumerate(cases):
        assert all(torch.equal(o, case[8]) and torch.equal(f, case[9]) for o, f in outs[s])


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("T,P", [(1500, 64), (700, 128), (20, 64)])
def test_inputs_that_the_kernel_before_wrote(T, P, captured):
    """Launches of a scan that is cut into runs overlap: none may read an input before the kernel that writes it, or leave an output to the one behind it too early."""
    layer = ScanLayer(1, H=2, P=P, seed=T)
    projs = [randn(1, T, layer.width(), seed=11 + i) for i in range(2)]
    proj, buf, residual = torch.empty_like(projs[0]), layer.buffers(1, T), torch.empty(1, T, layer.H * P, device="cuda")

    def run():
        layer.conv_state.zero_()
        layer.ssm_state.zero_()
        residual.zero_()
        layer(proj, residual, buf)

    want = []
    for q in projs:
        proj.copy_(q)
        torch.cuda.synchronize()
        run()
        torch.cuda.synchronize()
        want.append([buf["out"].clone(), residual.clone(), layer.conv_state.clone(), layer.ssm_state.clone()])
    if captured:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            run()
    got = []
    for i in range(12):
        proj.copy_(projs[i & 1])
        graph.replay() if captured else run()
        got.append([buf["out"].clone(), residual.clone(), layer.conv_state.clone(), layer.ssm_state.clone()])
    for i, result in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(result, want[i & 1]))


def test_the_python_checks_launch_the_same_calls(monkeypatch):
    layer = ScanLayer(2)
    proj, buf = randn(2, 40, layer.width(), seed=3), layer.buffers(2, 40)
    got = []
    for fast in (None, {}):
        monkeypatch.setattr(_layer, "_fast", fast)
        layer.conv_state.zero_(), layer.ssm_state.zero_()
        residual = torch.zeros(2, 40, layer.H * layer.P, device="cuda")
        layer(proj, residual, buf)
        got.append([buf["out"].clone(), residual, layer.conv_state.clone(), layer.ssm_state.clone()])
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_refusals_leave_the_outputs_alone():
    x, w = randn(2, 8, 64, seed=1), randn(64, 4, seed=2)
    out = torch.full_like(x, 5.0)
    bad = [lambda: F.short_conv(x.float(), w, out), lambda: F.short_conv(x, w[:32], out), lambda: F.short_conv(x, w, out[:, :4]), lambda: F.short_conv(x, randn(64, 5), out),
           lambda: F.short_conv(x, w, out, randn(64, dtype=fp32)), lambda: F.short_conv(x, w, out, initial_state=torch.zeros(2, 2, 64, dtype=bf16, device="cuda")),
           lambda: F.short_conv(x, w, out, cu_seqlens=torch.tensor([0, 8], device="cuda")), lambda: F.short_conv(x, w, out.transpose(1, 2).contiguous().transpose(1, 2)), lambda: F.short_conv(x, w, x),
           lambda: F.short_conv(x, w, out.cpu()), lambda: F.short_conv(x[:1], w, out[:1], cu_seqlens=torch.tensor([0, 8], device="cuda", dtype=torch.int32)),
           lambda: F.gated_norm(x.unsqueeze(2), x.unsqueeze(2), w[:, 0].contiguous(), out.unsqueeze(2), act="relu"), lambda: F.gated_norm(x.unsqueeze(2), x.unsqueeze(2), w, out.unsqueeze(2)),
           lambda: F.add_norm(x, x.clone(), w[:, 0].contiguous(), out, out), lambda: F.add_norm(x, x.half(), w[:, 0].contiguous(), out, out.clone())]
    for call in bad:
        with pytest.raises(RuntimeError):
            call()
    x, dt, Bm, Cm, A_log, dt_bias, D, x0 = inputs(2, 20, 4, 64, 1, 128, state="fp32")
    o = torch.full_like(x, 5.0)
    good = dict(x=x, dt=dt, B=Bm, C=Cm, out=o, A_log=A_log, dt_bias=dt_bias, D=D, initial_state=x0, final_state=None)
    for more in (dict(dt=dt.float()), dict(B=Bm[..., :96]), dict(A_log=A_log.to(bf16)), dict(final_state=x0.to(bf16)), dict(initial_state=x0[:1]), dict(D=D[:2]), dict(out=x), dict(x=x[..., :32]),
                 dict(C=Cm.repeat(1, 1, 3, 1)), dict(workspace=torch.empty(16, device="cuda")), dict(workspace=torch.empty(0, dtype=torch.uint8, device="cuda"))):
        with pytest.raises(RuntimeError):
            F.ssm_fwd(**{**good, **more})
    torch.cuda.synchronize()
    assert bool((out == 5.0).all()) and bool((o == 5.0).all())


@pytest.mark.parametrize("lens,T,state", [(None, 300, fp32), (None, 1, bf16), ([130, 9, 128, 4, 200], 530, bf16), (None, 1500, fp32)])
def test_nothing_outside_is_written(lens, T, state):
    """out, final_state and the workspace inside patterned buffers, the workspace no larger than asked for."""
    N, B = (2, 2) if lens is None else (len(lens), 1)
    cu = None if lens is None else torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), device="cuda")
    x, dt, Bm, Cm, A_log, dt_bias, D, x0 = inputs(B, T, 3, 64, 1, 128, seed=5, state="fp32" if state == fp32 else "bf16", N=N)

    def guarded(nbytes):
        buf = torch.full((8192 + nbytes,), 0x5A, dtype=torch.uint8, device="cuda")
        return buf, buf[4096:4096 + nbytes]
    buf_o, o = guarded(x.numel() * 2)
    buf_f, f = guarded(x0.numel() * x0.element_size())
    out, fin = o.view(bf16).view(x.shape), f.view(state).view(x0.shape)
    args = (x, dt, Bm, Cm, out, A_log, dt_bias, D, x0, fin, cu)
    need = F.ssm_workspace_size(*args)
    assert (need == 0) == (T <= 16)
    buf_w, ws = guarded(need)
    F.ssm_fwd(*args, workspace=ws if need else None)
    torch.cuda.synchronize()
    if need:
        assert F.read_status(ws) == 0
    for buf, n in ((buf_o, o.numel()), (buf_f, f.numel()), (buf_w, need)):
        assert bool((buf[:4096] == 0x5A).all()) and bool((buf[4096 + n:] == 0x5A).all())
    plain, fin2 = torch.empty_like(x), torch.empty_like(fin)
    F.ssm_fwd(x, dt, Bm, Cm, plain, A_log, dt_bias, D, x0, fin2, cu)
    n = T if lens is None else sum(lens)
    assert torch.equal(plain[:, :n], out[:, :n]) and torch.equal(fin, fin2)
    if lens is not None:
        assert bool((out[:, n:].contiguous().view(torch.uint8) == 0x5A).all())


def test_bad_cu_seqlens_is_reported_and_stays_in_bounds():
    x, dt, Bm, Cm, A_log, dt_bias, D, _ = inputs(1, 400, 2, 64, 1, 128)
    cu = torch.tensor([0, 400, 0, 400, 100], device="cuda")
    args = (x, dt, Bm, Cm, torch.empty_like(x), A_log, dt_bias, D, None, None, cu)
    ws = torch.empty(F.ssm_workspace_size(*args), dtype=torch.uint8, device="cuda")
    F.ssm_fwd(*args, workspace=ws)
    with pytest.raises(RuntimeError, match="not monotone"):
        F.read_status(ws)


@pytest.mark.parametrize("B,T,H,P,lens,stop", [
    (8, 300, 64, 64, None, 1), (8, 300, 32, 128, None, 2),          # whole sequences of three blocks, a CTA each
    (1, 900, 64, 64, None, 1),                                      # runs of two blocks, both passes
    (1, 900, 4, 64, [300, 5, 280, 315], 1)])                        # walks from the queue of a packed batch
def test_a_wait_that_runs_out_ends_the_call_with_a_status(B, T, H, P, lens, stop):
    """Loads that stop after a block or two of every walk: its waits give up, the status says so, and the next call is as the one before."""
    N = B if lens is None else len(lens)
    cu = None if lens is None else torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), device="cuda")
    x, dt, Bm, Cm, A_log, dt_bias, D, x0 = inputs(B, T, H, P, 1, 128, state="fp32", N=N)
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


def test_offsets_past_32_bits():
    """Tensors of more than 2^31 elements.  With states that are gone within a few tokens the end of a long sequence is the end of a short one."""
    H, P, T, tail = 64, 128, 270000, 700
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(1, T, H, P, generator=gen, device="cuda", dtype=bf16)
    dt, Bm, Cm = (torch.randn(1, T, *s, generator=gen, device="cuda", dtype=bf16) for s in ((H,), (1, 128), (1, 128)))
    A_log, dt_bias = torch.full((H,), 2.0, device="cuda"), torch.full((H,), 3.0, device="cuda")
    out = torch.empty_like(x)
    F.ssm_fwd(x, dt, Bm, Cm, out, A_log, dt_bias)
    short = torch.empty(1, tail, H, P, dtype=bf16, device="cuda")
    F.ssm_fwd(x[:, -tail:], dt[:, -tail:], Bm[:, -tail:], Cm[:, -tail:], short, A_log, dt_bias)
    a, b = out[:, -400:].double(), short[:, -400:].double()
    assert ((a - b).norm() / b.norm()).item() <= 4 * R.BF16          # two evaluations, each at most 2 roundings' worth off
    w = randn(H * P, 4, seed=3)
    F.short_conv(x.flatten(2), w, out.flatten(2))
    want, mass, _ = R.conv(x[:, -64:].flatten(2), w, None, None, None, True)
    assert R.off(out[:, -61:].flatten(2), want[:, 3:], conv_bound(want, mass, True)[:, 3:]) <= 1
    F.gated_norm(x, x, randn(P, dtype=fp32, seed=4), out)
    want = R.gated(x[:, -5:], x[:, -5:], randn(P, dtype=fp32, seed=4), 1e-6, "sigmoid", False)
    assert R.off(out[:, -5:], want, norm_bound(want)) <= 1


@pytest.mark.parametrize("seed", range(24))
def test_random_calls_of_the_scan(seed):
    gen = torch.Generator().manual_seed(1000 + seed)
    pick = lambda *a: a[int(torch.randint(len(a), (1,), generator=gen))]
    G = pick(1, 1, 2, 3)
    H, P, Ns = G * pick(1, 2, 3), pick(64, 128), pick(64, 128)
    state, regime = pick("fp32", "bf16", None), pick("usual", "usual", "wide", "keeps", "forgets")
    if seed % 2:
        lens = torch.randint(0, pick(12, 140, 900), (pick(1, 3, 9),), generator=gen).tolist()
        cu, B, T, N = torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), device="cuda"), 1, max(1, sum(lens)), len(lens)
    else:
        B, T = pick(1, 2, 5), int(torch.randint(1, pick(20, 300, 1300), (1,), generator=gen))
        lens, cu, N = [T], None, B
    x, dt, Bm, Cm, A_log, dt_bias, D, x0 = inputs(B, T, H, P, G, Ns, seed=seed, regime=regime, state=state, N=N, skip=seed % 3 > 0)
    want, mass, last, lmass = R.ssm(x, dt, Bm, Cm, A_log, dt_bias, D, x0, None if cu is None else cu.cpu())
    out, fin = torch.full_like(x, 7.0), torch.empty_like(x0) if state else None
    F.ssm_fwd(x, dt, Bm, Cm, out, A_log, dt_bias, D, x0, fin, cu)
    n = T if cu is None else sum(lens)
    check(out[:, :n], fin, want[:, :n], mass[:, :n], last, lmass, max(lens), None, state == "bf16", exponent_slack(A_log, dt, dt_bias, None))


@pytest.mark.parametrize("lens", [[5000, 5, 2300], [3000], [1, 4000, 200, 9, 130, 0]])
def test_packed_sequences_that_are_cut_into_runs(lens):
    cu = torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), device="cuda")
    x, dt, Bm, Cm, A_log, dt_bias, D, x0 = inputs(1, sum(lens), 2, 64, 1, 64, seed=len(lens), state="fp32", N=len(lens))
    want, mass, last, lmass = R.ssm(x, dt, Bm, Cm, A_log, dt_bias, D, x0, cu.cpu())
    out, fin = torch.empty_like(x), torch.empty_like(x0)
    F.ssm_fwd(x, dt, Bm, Cm, out, A_log, dt_bias, D, x0, fin, cu)
    check(out, fin, want, mass, last, lmass, max(lens), None, False, exponent_slack(A_log, dt, dt_bias, None))
    again = torch.empty_like(x)
    F.ssm_fwd(x, dt, Bm, Cm, again, A_log, dt_bias, D, x0, x0, cu)
    assert torch.equal(again, out) and torch.equal(x0, fin)
