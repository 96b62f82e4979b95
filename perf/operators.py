"""The operators round the recurrence, over the range a user calls them: `short_conv`, `ssm_fwd`, `gated_norm`, `add_norm`.

A case is one call.  Inputs are laid out as a layer has them: the channels of the convolution are columns of a wider projection, and x, B
and C of the selective scan are columns of one convolution's output, dt columns of the projection.  With `own` false `run` computes the
operator from elementary torch operations in 32 bits, with `own` true it calls the framework.  `exact` is the definition in 64 bits:
the scan token by token, the convolution sequence by sequence.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
MOST_TOKEN_COLUMNS = 120206 * 2048      # tokens x heads x channels of the largest listed scan; a drawn one has no more
MOST_CHAINS = 8192                      # states of a batch: up to 64 KB each
MOST_ELEMENTS = 4 * 8192 * 4352         # of the largest listed convolution
MOST_NORM = 4 * 8192 * 4096             # elements of the largest listed norm


def _conv(C, B=1, T=0, W=4, n_seqs=0, lo=0, hi=0, len_seed=0, state_in=False, state_out=False, bias=False, silu=True, weight="bf16"):
    return dict(op="conv", C=C, B=B, T=T, W=W, n_seqs=n_seqs, lo=lo, hi=hi, len_seed=len_seed, state_in=state_in, state_out=state_out,
                bias=bias, silu=silu, weight=weight)


def _ssm(H, P, N, G=1, B=1, T=0, n_seqs=0, n_single=0, lo=0, hi=0, len_seed=0, state_in=None, state_out=None, skip=True):
    return dict(op="ssm", H=H, P=P, N=N, G=G, B=B, T=T, n_seqs=n_seqs, n_single=n_single, lo=lo, hi=hi, len_seed=len_seed,
                state_in=state_in, state_out=state_out, skip=skip)


def _gated(H, D, B=1, T=1, act="sigmoid", gate_first=False, per_head=False, weight="fp32"):
    return dict(op="gated", H=H, D=D, B=B, T=T, act=act, gate_first=gate_first, per_head=per_head, weight=weight)


def _add(D, B=1, T=1, residual="bf16", scale=1.0, weight="bf16"):
    return dict(op="add", D=D, B=B, T=T, residual=residual, scale=scale, weight=weight)


def _lengths(case):
    """Sequence lengths of a packed batch (`n_single` sequences of one token, then `n_seqs` of lo..hi), or None for equal lengths."""
    if case.get("n_seqs", 0) == 0:
        return None
    gen = torch.Generator().manual_seed(case["len_seed"])
    return [1] * case.get("n_single", 0) + torch.randint(case["lo"], case["hi"] + 1, (case["n_seqs"],), generator=gen).tolist()


def _sizes(case):
    """(tokens in all, sequences)"""
    lens = _lengths(case)
    return (case["B"] * case["T"], case["B"]) if lens is None else (sum(lens), len(lens))


def listed():
    return [
        # a decode step of one request: q, k and v of 32 heads in one convolution; nothing but latency
        dict(_conv(12288, B=1, T=1, state_in=True, state_out=True), name="conv_decode_b1"),
        # many short ragged sequences in one packed batch
        dict(_conv(2048, n_seqs=200, lo=1, hi=300, len_seed=5, state_in=True, state_out=True, bias=True), name="conv_packed_n200"),
        # the prefill of the benchmark, channels of the selective scan: x of 32 heads, B and C
        dict(_conv(4352, B=4, T=8192, state_out=True, bias=True, weight="fp32"), name="conv_prefill_b4_t8192"),
        # a decode step of a serving batch: the stream over the states
        dict(_ssm(32, 64, 128, B=256, T=1, state_in="fp32", state_out="fp32"), name="ssm_step_b256"),
        # an ordinary prompt of odd length
        dict(_ssm(32, 64, 128, B=1, T=777, state_out="bf16"), name="ssm_prompt_t777"),
        # the prefill of the benchmark: four prompts, wide heads
        dict(_ssm(32, 128, 128, B=4, T=8192, state_in="fp32", state_out="fp32"), name="ssm_prefill_b4_t8192"),
        # the benchmark's packed prefill, lengths U[256, 16384]
        dict(_ssm(32, 64, 128, n_seqs=16, lo=256, hi=16384, state_in="bf16", state_out="bf16"), name="ssm_packed_n16"),
        # few heads, one very long sequence
        dict(_ssm(8, 64, 128, B=1, T=131072, state_in="fp32", state_out="fp32"), name="ssm_long_t131072_h8"),
        # output norm of a decode batch, a row per head
        dict(_gated(32, 128, B=64, T=1), name="gated_step_b64"),
        # output norm of the benchmark's prefill
        dict(_gated(32, 128, B=4, T=8192), name="gated_prefill_b4_t8192"),
        # residual norm of a decode batch
        dict(_add(4096, B=64, T=1), name="add_step_b64"),
        # residual norm of a prefill, the stream kept in fp32
        dict(_add(4096, B=4, T=8192, residual="fp32", scale=0.5), name="add_prefill_b4_t8192"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi)))))))


def draw(rng: random.Random):
    """One more call: convolutions and scans as steps, prompts and packed batches, both norms; sizes log-uniform, odd ones included."""
    kind = rng.choice(["conv_step", "conv", "conv_packed", "ssm_step", "ssm_prompt", "ssm_prompt", "ssm_packed", "ssm_mixed", "ssm_long", "gated", "add"])
    seed = rng.randrange(1 << 20)
    if kind.startswith("conv"):
        C = 8 * _log_int(rng, 8, 1536)
        more = dict(W=rng.choice([2, 3, 4, 4]), state_in=rng.random() < 0.5, state_out=rng.random() < 0.7, bias=rng.random() < 0.5,
                    silu=rng.random() < 0.8, weight=rng.choice(["bf16", "fp32"]))
        if kind == "conv_step":
            more.update(state_in=True, state_out=True)
            return _conv(C, B=_log_int(rng, 1, 512), T=rng.choice([1, 1, 2, 5]), **more)
        tokens = MOST_ELEMENTS // C
        if kind == "conv":
            T = _log_int(rng, 6, min(32768, tokens))
            return _conv(C, B=_log_int(rng, 1, min(64, tokens // T)), T=T, **more)
        hi = _log_int(rng, 4, min(8192, tokens))
        return _conv(C, n_seqs=_log_int(rng, 1, max(1, min(512, tokens // hi))), lo=1, hi=hi, len_seed=seed, **more)
    if kind.startswith("ssm"):
        H, P, N = rng.choice([1, 2, 3, 5, 8, 12, 16, 32, 64]), rng.choice([64, 64, 128]), rng.choice([64, 128, 128])
        G = rng.choice([1, 1, 2 if H % 2 == 0 else 1, 4 if H % 4 == 0 else H])
        state = rng.choice([(None, None), (None, "fp32"), (None, "bf16"), ("fp32", "fp32"), ("bf16", "bf16")])
        more = dict(G=G, state_in=state[0], state_out=state[1], skip=rng.random() < 0.8)
        tokens = MOST_TOKEN_COLUMNS // (2 * H * P)
        if kind == "ssm_step":
            kept = rng.choice(["fp32", "bf16"])
            more.update(state_in=kept, state_out=kept)
            return _ssm(H, P, N, B=_log_int(rng, 1, min(512, MOST_CHAINS // H)), T=rng.choice([1, 1, 1, 2, 4, 7]), **more)
        if kind == "ssm_prompt":
            T = _log_int(rng, 8, min(16384, tokens))
            return _ssm(H, P, N, B=_log_int(rng, 1, max(1, min(32, tokens // T))), T=T, **more)
        if kind == "ssm_long":
            H = rng.choice([1, 2, 4, 8])
            more.update(G=1)
            return _ssm(H, 64, N, B=1, T=_log_int(rng, 16384, 131072), **more)
        if kind == "ssm_packed":
            hi = _log_int(rng, 32, min(16384, tokens // 2))
            return _ssm(H, P, N, n_seqs=_log_int(rng, 2, max(2, min(256, tokens // hi, MOST_CHAINS // H))), lo=1, hi=hi, len_seed=seed, **more)
        hi = _log_int(rng, 64, min(4096, tokens))
        single = _log_int(rng, 4, max(4, min(128, tokens // hi, MOST_CHAINS // H)))
        return _ssm(H, P, N, n_seqs=rng.randint(1, max(1, min(8, tokens // hi))), n_single=single, lo=hi // 8, hi=hi, len_seed=seed, **more)
    if kind == "gated":
        D, H = 8 * _log_int(rng, 8, 512), rng.choice([1, 1, 2, 5, 8, 16, 32])
        rows = max(1, MOST_NORM // (D * H))
        B = _log_int(rng, 1, min(64, rows))
        return _gated(H, D, B=B, T=rng.choice([1, _log_int(rng, 1, min(8192, max(1, rows // B)))]), act=rng.choice(["sigmoid", "silu"]),
                      gate_first=rng.random() < 0.5, per_head=rng.random() < 0.5, weight=rng.choice(["bf16", "fp32"]))
    D = 8 * _log_int(rng, 8, 1024)
    rows = MOST_NORM // D
    B = _log_int(rng, 1, 64)
    return _add(D, B=B, T=rng.choice([1, _log_int(rng, 1, min(8192, max(1, rows // B)))]), residual=rng.choice(["bf16", "fp32"]),
                scale=rng.choice([1.0, 0.5, 0.22]), weight=rng.choice(["bf16", "fp32"]))


def prepare(case, seed):
    """The inputs of one call and the tensors its results go to."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    bf = torch.bfloat16

    def randn(*shape, dtype=bf, std=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * std).to(dtype)

    s = dict(case)
    lens = _lengths(case)
    tokens, n = _sizes(case)
    B, T = (1, tokens) if lens is not None else (case["B"], case["T"])
    s["longest"] = max(lens) if lens is not None else T
    s["cu"] = None if lens is None else torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), device="cuda")
    s["x0"] = s["fin"] = None
    if case["op"] == "conv":
        C, W = case["C"], case["W"]
        s["x"] = randn(B, T, C + 64)[..., 64:]
        s["w"] = randn(C, W, dtype=DTYPES[case["weight"]], std=W ** -0.5)
        s["b"] = randn(C, dtype=DTYPES[case["weight"]], std=0.1) if case["bias"] else None
        s["x0"] = randn(n, W - 1, C) if case["state_in"] else None
        s["fin"] = torch.empty(n, W - 1, C, dtype=bf, device="cuda") if case["state_out"] else None
        s["out"] = torch.empty(B, T, C, dtype=bf, device="cuda")
    elif case["op"] == "ssm":
        H, P, N, G = case["H"], case["P"], case["N"], case["G"]
        xbc = randn(B, T, H * P + 2 * G * N)
        s["x"] = xbc[..., :H * P].unflatten(-1, (H, P))
        s["Bm"] = xbc[..., H * P:H * P + G * N].unflatten(-1, (G, N))
        s["Cm"] = xbc[..., H * P + G * N:].unflatten(-1, (G, N))
        s["dt"] = randn(B, T, H + 8, std=0.5)[..., :H]
        # step sizes of 0.001 to 0.1 and decay rates of 1 to 16, as these layers start from
        step = torch.exp(torch.empty(H, device="cuda").uniform_(math.log(1e-3), math.log(1e-1), generator=gen))
        s["dt_bias"] = step + torch.log(-torch.expm1(-step))
        s["A_log"] = torch.log(torch.empty(H, device="cuda").uniform_(1.0, 16.0, generator=gen))
        s["D"] = randn(H, dtype=torch.float32) if case["skip"] else None
        s["x0"] = randn(n, H, P, N, dtype=DTYPES[case["state_in"]], std=0.5) if case["state_in"] else None
        s["fin"] = torch.empty(n, H, P, N, dtype=DTYPES[case["state_out"]], device="cuda") if case["state_out"] else None
        s["out"] = torch.empty(B, T, H, P, dtype=bf, device="cuda")
    elif case["op"] == "gated":
        H, D = case["H"], case["D"]
        s["x"] = randn(B, T, H, D)
        s["gate"] = randn(B, T, H * D + 128)[..., 128:].unflatten(-1, (H, D))
        s["w"] = 1 + randn(*((H, D) if case["per_head"] else (D,)), dtype=torch.float32, std=0.1)
        s["w"] = s["w"].to(DTYPES[case["weight"]])
        s["out"] = torch.empty(B, T, H, D, dtype=bf, device="cuda")
    else:
        D = case["D"]
        s["x"] = randn(B, T, D)
        s["res"] = randn(B, T, D, dtype=DTYPES[case["residual"]], std=3.0)
        s["w"] = (1 + randn(D, dtype=torch.float32, std=0.1)).to(DTYPES[case["weight"]])
        s["out"] = torch.empty(B, T, D, dtype=bf, device="cuda")
        s["res_out"] = torch.empty_like(s["res"])
    return s


def run(s):
    if own:
        return _framework(s)
    return {"conv": _plain_conv, "ssm": _plain_ssm, "gated": _plain_gated, "add": _plain_add}[s["op"]](s)


def _framework(s):
    import flashkda_b200 as F
    if s["op"] == "conv":
        F.short_conv(s["x"], s["w"], s["out"], s["b"], initial_state=s["x0"], final_state=s["fin"], cu_seqlens=s["cu"], silu=s["silu"])
        return {"out": s["out"], "final_state": s["fin"]}
    if s["op"] == "ssm":
        F.ssm_fwd(s["x"], s["dt"], s["Bm"], s["Cm"], s["out"], s["A_log"], s["dt_bias"], s["D"], initial_state=s["x0"],
                  final_state=s["fin"], cu_seqlens=s["cu"])
        return {"out": s["out"], "final_state": s["fin"]}
    if s["op"] == "gated":
        F.gated_norm(s["x"], s["gate"], s["w"], s["out"], eps=1e-5, act=s["act"], gate_first=s["gate_first"])
        return {"out": s["out"]}
    F.add_norm(s["x"], s["res"], s["w"], s["out"], s["res_out"], scale=s["scale"], eps=1e-5)
    return {"out": s["out"], "residual": s["res_out"]}


def _bounds(s):
    """First token and end of every sequence in the flattened batch."""
    if s["cu"] is not None:
        return s["cu"][:-1], s["cu"][1:]
    first = torch.arange(s["B"], device="cuda") * s["T"]
    return first, first + s["T"]


def _sigmoid(x):
    return 1 / (1 + torch.exp(-x))


def _plain_conv(s):
    C, W = s["C"], s["W"]
    shape = s["out"].shape
    x = s["x"].reshape(-1, C)
    first, end = _bounds(s)
    n, total = first.numel(), x.shape[0]
    # rows behind the tokens: the states, then one of zeros
    rows = torch.cat([x] + ([s["x0"].reshape(-1, C)] if s["x0"] is not None else []) + [x.new_zeros(1, C)]).float()

    def row_of(pos, seq):
        old = total + seq * (W - 1) + (W - 1) + pos - first[seq] if s["x0"] is not None else torch.full_like(pos, rows.shape[0] - 1)
        return torch.where(pos >= first[seq], pos, old)

    t = torch.arange(total, device="cuda")
    seq = torch.searchsorted(end, t, right=True)
    w = s["w"].float()
    y = sum(rows[row_of(t - (W - 1) + k, seq)] * w[:, k] for k in range(W))
    if s["b"] is not None:
        y = y + s["b"].float()
    if s["silu"]:
        y = y * _sigmoid(y)
    fin = None
    if s["fin"] is not None:
        pos = end[:, None] + torch.arange(-(W - 1), 0, device="cuda")
        fin = rows[row_of(pos, torch.arange(n, device="cuda")[:, None].expand_as(pos))].to(torch.bfloat16)
    return {"out": y.to(torch.bfloat16).view(shape), "final_state": fin}


def _plain_ssm(s):
    """In chunks of 64 tokens: within a chunk by a masked product, across chunks by a product with the decay between them."""
    H, P, N, G, Q = s["H"], s["P"], s["N"], s["G"], 64
    first, end = _bounds(s)
    n = first.numel()
    chunks = -(-s["longest"] // Q)
    pos = torch.arange(chunks * Q, device="cuda")
    there = pos < (end - first)[:, None]                                          # [n, chunks * Q]
    idx = torch.where(there, first[:, None] + pos, 0)

    def padded(t, *dims):
        t = t.reshape(-1, *dims)[idx].float()
        return torch.where(there.view(*there.shape, *[1] * len(dims)), t, 0.0).unflatten(1, (chunks, Q))

    x = padded(s["x"], H, P)
    Bm = padded(s["Bm"], G, N).repeat_interleave(H // G, 3)
    Cm = padded(s["Cm"], G, N).repeat_interleave(H // G, 3)
    z = padded(s["dt"], H) + s["dt_bias"]
    delta = torch.where(there.view(n, chunks, Q, 1), torch.log1p(torch.exp(-z.abs())) + z.clamp(min=0), 0.0)
    a = (-torch.exp(s["A_log"].double()) * delta.double())                        # log decay of every token
    L = a.cumsum(2).permute(0, 1, 3, 2)                                           # [n, chunks, H, Q]
    causal = torch.ones(Q, Q, dtype=torch.bool, device="cuda").tril()
    decay = torch.where(causal, L[..., :, None] - L[..., None, :], -torch.inf).float().exp()
    xd = x * delta[..., None]
    scores = torch.einsum("bcihn,bcjhn->bchij", Cm, Bm) * decay
    y = torch.einsum("bchij,bcjhp->bcihp", scores, xd)
    to_end = (L[..., -1:] - L).float().exp().permute(0, 1, 3, 2)
    added = torch.einsum("bcjhp,bcjhn->bchpn", xd * to_end[..., None], Bm)
    # the state before chunk c: the states that the chunks before it added, and the first one, decayed up to there
    before = torch.zeros(n, H, 1, P, N, device="cuda") if s["x0"] is None else s["x0"].float()[:, :, None]
    added = torch.cat([before, added.permute(0, 2, 1, 3, 4)], 2)                  # [n, H, chunks + 1, P, N]
    total = torch.cat([torch.zeros(n, H, 1, dtype=torch.float64, device="cuda"), L[..., -1].permute(0, 2, 1)], 2).cumsum(2)
    causal = torch.ones(chunks + 1, chunks + 1, dtype=torch.bool, device="cuda").tril()
    decay = torch.where(causal, total[..., :, None] - total[..., None, :], -torch.inf).float().exp()
    states = torch.matmul(decay, added.flatten(3)).view(n, H, chunks + 1, P, N)
    y = y + torch.einsum("bcihn,bhcpn->bcihp", Cm, states[:, :, :-1]) * L.float().exp().permute(0, 1, 3, 2)[..., None]
    if s["D"] is not None:
        y = y + x * s["D"][:, None]
    out = y.flatten(1, 2)[there].to(torch.bfloat16).view(s["out"].shape)
    return {"out": out, "final_state": None if s["fin"] is None else states[:, :, -1].to(s["fin"].dtype)}


def _plain_gated(s):
    x, g, w = s["x"].float(), s["gate"].float(), s["w"].float()
    g = _sigmoid(g) * (g if s["act"] == "silu" else 1)
    if s["gate_first"]:
        x = x * g
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-5) * w
    return {"out": (y if s["gate_first"] else y * g).to(torch.bfloat16)}


def _plain_add(s):
    h = s["res"].float() + s["scale"] * s["x"].float()
    y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + 1e-5) * s["w"].float()
    return {"out": y.to(torch.bfloat16), "residual": h.to(s["res"].dtype)}


def work(case):
    """Bytes: every input read once, every output written once.  Operations: a multiply and an add per tap; of the scan, per state
    element, the decay, the update and the product with C; a handful per element of a norm."""
    tokens, n = _sizes(case)
    if case["op"] == "conv":
        C, W, wide = case["C"], case["W"], 4 if case["weight"] == "fp32" else 2
        states = n * (W - 1) * C * 2 * (case["state_in"] + case["state_out"])
        return {"bytes": 4 * tokens * C + states + C * (W + case["bias"]) * wide, "flops": 2 * W * tokens * C}
    if case["op"] == "ssm":
        H, P, N, G = case["H"], case["P"], case["N"], case["G"]
        size = {None: 0, "bf16": 2, "fp32": 4}
        states = n * H * P * N * (size[case["state_in"]] + size[case["state_out"]])
        return {"bytes": tokens * (4 * H * P + 2 * H + 4 * G * N) + states, "flops": 5 * P * N * tokens * H}
    if case["op"] == "gated":
        return {"bytes": 6 * tokens * case["H"] * case["D"], "flops": 10 * tokens * case["H"] * case["D"]}
    return {"bytes": tokens * case["D"] * (4 + 2 * (4 if case["residual"] == "fp32" else 2)), "flops": 7 * tokens * case["D"]}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "conv":
        return _exact_conv(s)
    if case["op"] == "ssm":
        return _exact_ssm(s)
    x, w = s["x"].double(), s["w"].double()
    if case["op"] == "gated":
        g = s["gate"].double()
        g = torch.sigmoid(g) * (g if case["act"] == "silu" else 1.0)
        u = x * g if case["gate_first"] else x
        u = u / torch.sqrt(u.square().sum(-1, keepdim=True) / case["D"] + 1e-5) * w
        return {"out": u if case["gate_first"] else u * g}
    h = s["res"].double() + case["scale"] * x
    return {"out": h / torch.sqrt(h.square().sum(-1, keepdim=True) / case["D"] + 1e-5) * w, "residual": h}


def _sequences(s, t):
    """The rows of every sequence, one after the other."""
    if s["cu"] is None:
        return list(t.unbind(0))
    return list(t[0].split(s["cu"].diff().tolist()))


def _exact_conv(s):
    W, w = s["W"], s["w"].double()
    outs, fins = [], []
    for i, x in enumerate(_sequences(s, s["x"])):
        past = s["x0"][i].double() if s["x0"] is not None else torch.zeros(W - 1, s["C"], dtype=torch.float64, device="cuda")
        u = torch.cat([past, x.double()])
        y = torch.zeros_like(x, dtype=torch.float64)
        for k in range(W):
            y += u[k:k + x.shape[0]] * w[:, k]
        if s["b"] is not None:
            y += s["b"].double()
        outs.append(y * torch.sigmoid(y) if s["silu"] else y)
        fins.append(u[u.shape[0] - (W - 1):])
    return {"out": torch.cat(outs).view(s["out"].shape), "final_state": torch.stack(fins) if s["fin"] is not None else None}


def _exact_ssm(s):
    """Token by token, all sequences at once; the shorter ones rest once they have ended."""
    H, P, N, G = s["H"], s["P"], s["N"], s["G"]
    n = s["B"] if s["cu"] is None else s["cu"].numel() - 1
    lens = [s["T"]] * n if s["cu"] is None else s["cu"].diff().tolist()
    order = sorted(range(n), key=lambda i: -lens[i])
    first = s["cu"][:-1] if s["cu"] is not None else torch.arange(n, device="cuda") * s["T"]
    first = first[order]
    A, bias = torch.exp(s["A_log"].double()), s["dt_bias"].double()
    state = torch.zeros(n, H, P, N, dtype=torch.float64, device="cuda") if s["x0"] is None else s["x0"].double()[order]
    x, dt, Bm, Cm = s["x"].reshape(-1, H, P), s["dt"].reshape(-1, H), s["Bm"].reshape(-1, G, N), s["Cm"].reshape(-1, G, N)
    y = torch.zeros(x.shape[0], H, P, dtype=torch.float64, device="cuda")
    live, ends = n, sorted(lens, reverse=True)
    for t in range(ends[0] if ends else 0):
        while ends[live - 1] <= t:
            live -= 1
        rows = first[:live] + t
        delta = torch.logaddexp(dt[rows].double() + bias, torch.zeros((), dtype=torch.float64, device="cuda"))
        b, c = Bm[rows].double()[:, :, None], Cm[rows].double()[:, :, None]           # [live, G, 1, N]
        at = x[rows].double()
        S = state[:live]
        S.mul_(torch.exp(-A * delta)[..., None, None])
        S.view(live, G, H // G, P, N).add_((delta[..., None] * at).view(live, G, H // G, P, 1) * b[:, :, :, None])
        y[rows] = torch.matmul(S.view(live, G, H // G, P, N), c.unsqueeze(-1)).view(live, H, P)
    if s["D"] is not None:
        y += s["D"].double()[:, None] * x.double()
    fin = None
    if s["fin"] is not None:
        fin = torch.empty_like(state)
        fin[order] = state
    return {"out": y.view(s["out"].shape), "final_state": fin}
