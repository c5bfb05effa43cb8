"""Performance cases of the training operators: the backward pass of the gated
delta rule, of the Local block's prologue and of its norms, and layer norm.

Each case is one pass through one operator as a training program makes it.
Head sizes are those of the model configurations (head_dim 32, 64 and 128)
with 16 heads as in the benchmark; the norms' rows are the op's outputs
(tokens x heads rows of one head) or token rows of a model's width.

A case is a dict of plain values:
  op       delta_backward | block_backward | norm_backward | layernorm
  dtype    of the activations and their gradients ("bf16" or "f32")
  delta_backward, block_backward:
    batch, seq_len    dense batch
    lengths           packed batch instead: comma-separated sequence lengths
    heads, d_k, d_v
    gate     what the caller holds: "log" (g = ln alpha) or "alpha"
    g_mean   mean of the decay logits: g = -softplus(N(g_mean, 1))
    init     "" none; "carried": the sequences continue from a state that is
             not trained (truncated backpropagation); "trained": the state's
             gradient is wanted and the final state has one
  norm_backward, layernorm: rows, dim
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
CHUNK = 64


def _delta(op, dtype, batch, seq_len, heads, d_k, d_v, *, lengths="", gate="log", g_mean=0.0, init=""):
    return dict(op=op, dtype=dtype, batch=batch, seq_len=seq_len, lengths=lengths, heads=heads, d_k=d_k, d_v=d_v,
                gate=gate, g_mean=g_mean, init=init)


def _norm(op, dtype, rows, dim):
    return dict(op=op, dtype=dtype, rows=rows, dim=dim)


def listed():
    named = {
        # a small model's training step on one short sequence: all latency
        "delta_small": _delta("delta_backward", "bf16", 1, 64, 2, 32, 32),
        # the benchmark's shape as a training batch
        "delta_batch": _delta("delta_backward", "bf16", 4, 4096, 16, 128, 128),
        # documents of different lengths packed without padding, each
        # continuing from a state that is not trained, alpha as the caller holds it
        "delta_packed": _delta("delta_backward", "bf16", 9, 0, 16, 128, 128, gate="alpha", init="carried",
                               lengths="1187,129,64,733,2048,351,1,918,1502"),
        # long context with slow decay and wide values
        "delta_long": _delta("delta_backward", "bf16", 1, 16384, 16, 128, 256, g_mean=-2.0),
        # full precision, odd length, the state's gradient wanted
        "delta_fp32": _delta("delta_backward", "f32", 2, 1003, 8, 64, 64, init="trained"),
        # the block's prologue of the same small step
        "block_small": _delta("block_backward", "bf16", 1, 64, 2, 32, 32),
        # the prologue of a training batch
        "block_batch": _delta("block_backward", "bf16", 4, 4096, 16, 128, 128),
        # full precision, packed, conv states carried with their gradients
        "block_fp32": _delta("block_backward", "f32", 5, 0, 8, 64, 64, lengths="300,77,512,1,190", init="trained"),
        # the per-head norm of the training batch's outputs
        "norm_batch": _norm("norm_backward", "bf16", 4 * 4096 * 16, 128),
        # the same of a small model at full precision
        "norm_small": _norm("norm_backward", "f32", 1003 * 8, 64),
        # token rows of the benchmark's width (16 heads of 128), forward and backward
        "layernorm_batch": _norm("layernorm", "bf16", 4 * 4096, 2048),
        # an odd width at full precision
        "layernorm_odd": _norm("layernorm", "f32", 777, 1001),
    }
    return [dict(name=n, **c) for n, c in named.items()]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    """One more case of the listed ones' ranges; tokens x heads and elements
    stay below the largest listed case's."""
    op = rng.choice(["delta_backward", "delta_backward", "delta_backward", "block_backward", "norm_backward",
                     "layernorm"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op == "norm_backward":
        dim = rng.choice([32, 64, 128, 128, 256, rng.randint(8, 300)])
        return _norm(op, dtype, _log_int(rng, 16, 30_000_000 // dim), dim)
    if op == "layernorm":
        dim = rng.choice([256, 512, 1024, 2048, 4096, rng.randint(64, 2048)])
        return _norm(op, dtype, _log_int(rng, 16, 30_000_000 // dim), dim)
    d_k = rng.choice([32, 64, 128, 128, 128])
    d_v = rng.choice([d_k, d_k, d_k, 2 * d_k])
    heads = rng.choice([2, 4, 8, 16, 16])
    gate = rng.choice(["log", "log", "alpha"]) if op == "delta_backward" else "log"
    g_mean = rng.choice([0.0, 0.0, -2.0])
    init = rng.choice(["", "", "trained" if dtype == "f32" or op == "block_backward" else "carried"])
    tokens = _log_int(rng, 64, min(16384, (64000 if dtype == "f32" else 200000) // heads))
    if rng.random() < 0.5:
        batch = _log_int(rng, 1, 8)
        return _delta(op, dtype, batch, max(1, tokens // batch), heads, d_k, d_v, gate=gate, g_mean=g_mean, init=init)
    n = rng.randint(2, 12)
    cuts = sorted(rng.randint(0, tokens) for _ in range(n - 1))
    lens = [b - a for a, b in zip([0] + cuts, cuts + [tokens])]
    return _delta(op, dtype, n, 0, heads, d_k, d_v, gate=gate, g_mean=g_mean, init=init,
                  lengths=",".join(str(x) for x in lens))


def _lengths(case):
    if case["lengths"]:
        return [int(x) for x in case["lengths"].split(",")]
    return [case["seq_len"]] * case["batch"]


def _softplus(x):
    return torch.clamp(x, min=0) + torch.log1p(torch.exp(-x.abs()))


def _unit(x):
    return x / x.norm(dim=-1, keepdim=True)


def _inputs(case, seed):
    """The tensors of the call, from the seed alone."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, mean=0.0, std=1.0):
        return torch.randn(shape, generator=gen, device="cuda") * std + mean

    if case["op"] in ("norm_backward", "layernorm"):
        rows, dim = case["rows"], case["dim"]
        s = {"x": normal(rows, dim, mean=0.3).to(dt), "dy": (normal(rows, dim) * 1e-3).to(dt),
             "scale": normal(dim, mean=1.0, std=0.1)}
        if case["op"] == "layernorm":
            s["bias"] = normal(dim, std=0.1)
        return s
    B, T, H, dk, dv = case["batch"], case["seq_len"], case["heads"], case["d_k"], case["d_v"]
    packed = bool(case["lengths"])
    lead = (sum(_lengths(case)),) if packed else (B, T)
    s = {}
    if packed:
        cu = [0]
        for n in _lengths(case):
            cu.append(cu[-1] + n)
        s["cu"] = torch.tensor(cu, dtype=torch.int32, device="cuda")
    if case["op"] == "block_backward":
        C = H * (2 * dk + dv)
        s["x"] = normal(*lead, C).to(dt)
        s["w"], s["bias"] = normal(C, 4, std=0.5), normal(C, std=0.1)
        s["beta_logit"], s["alpha_logit"] = normal(*lead, H), normal(*lead, H, mean=case["g_mean"])
        s["a_log"] = normal(H, std=0.3)
        s["dq"], s["dk"], s["dv"] = ((normal(*lead, H, d) * 1e-3).to(dt) for d in (dk, dk, dv))
        s["dbeta"], s["dg"] = ((normal(*lead, H) * 1e-3).to(dt) for _ in range(2))
        if case["init"]:
            s["conv_state"], s["dconv_state"] = normal(B, C, 3), normal(B, C, 3) * 1e-3
        return s
    s["q"] = (_unit(normal(*lead, H, dk)) * math.sqrt(dk)).to(dt)
    s["k"] = _unit(normal(*lead, H, dk)).to(dt)
    s["v"] = normal(*lead, H, dv).to(dt)
    g = -_softplus(normal(*lead, H, mean=case["g_mean"]))
    s["gate"] = g if case["gate"] == "log" else torch.exp(g)
    s["beta"] = torch.sigmoid(normal(*lead, H))
    # a loss's gradient, a mean over the batch: far below 1
    s["do"] = (normal(*lead, H, dv) * 1e-3).to(dt)
    if case["init"]:
        s["state"] = normal(B, H, dv, dk, std=0.05)
    if case["init"] == "trained":
        s["dfinal"] = normal(B, H, dv, dk, std=0.05) * 1e-3
    return s


def prepare(case, seed):
    return {"case": dict(case), **_inputs(case, seed)}


def run(state):
    s, case = state, state["case"]
    if not own:
        return _PLAIN[case["op"]](s, case)
    import rhizome_amd

    if case["op"] == "delta_backward":
        gate = {"g" if case["gate"] == "log" else "alpha": s["gate"]}
        out = rhizome_amd.prefill_backward(
            s["q"], s["k"], s["v"], beta=s["beta"], do=s["do"], dfinal_state=s.get("dfinal"), cu_seqlens=s.get("cu"),
            initial_state=s.get("state"), output_dinitial_state=case["init"] == "trained", **gate)
        return out if case["init"] == "trained" else out[:5]
    if case["op"] == "block_backward":
        out = rhizome_amd.conv_prepare_backward(
            s["x"], s["w"], s["bias"], s["beta_logit"], s["alpha_logit"], s["a_log"], s["dq"], s["dk"], s["dv"],
            s["dbeta"], s["dg"], heads=case["heads"], d_k=case["d_k"], d_v=case["d_v"], cu_seqlens=s.get("cu"),
            initial_state=s.get("conv_state"), dfinal_state=s.get("dconv_state"))
        return out if case["init"] else out[:6]
    if case["op"] == "norm_backward":
        return rhizome_amd.rmsnorm_heads_backward(s["dy"], s["x"], s["scale"])
    y = rhizome_amd.layernorm(s["x"], s["scale"], s["bias"])
    return (y, *rhizome_amd.layernorm_backward(s["dy"], s["x"], s["scale"]))


# ------------------------------------------------------------- plain forms
def _rows_norm_backward(s, case):
    x, dy = s["x"].float(), s["dy"].float()
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
    xh, t = x * r, dy * s["scale"]
    dx = r * (t - xh * (t * xh).mean(-1, keepdim=True))
    return dx.to(s["x"].dtype), (dy * xh).sum(0, dtype=torch.float64).float()


def _layernorm(s, case):
    x, dy = s["x"].float(), s["dy"].float()
    xc = x - x.mean(-1, keepdim=True)
    r = torch.rsqrt((xc * xc).mean(-1, keepdim=True) + 1e-5)
    xh, t = xc * r, dy * s["scale"]
    dx = r * (t - t.mean(-1, keepdim=True) - xh * (t * xh).mean(-1, keepdim=True))
    dt = s["x"].dtype
    return ((xh * s["scale"] + s["bias"]).to(dt), dx.to(dt), (dy * xh).sum(0, dtype=torch.float64).float(),
            dy.sum(0, dtype=torch.float64).float())


def _places(case, device):
    """Of every token of the pack: its sequence and its place in it; the first token of each sequence."""
    lens = torch.tensor(_lengths(case), device=device)
    seq = torch.repeat_interleave(torch.arange(len(lens), device=device), lens)
    start = torch.cumsum(lens, 0) - lens
    return seq, torch.arange(int(lens.sum()), device=device) - start[seq], start, lens


def _block_backward(s, case):
    """The prologue's adjoint over the pack's tokens: the convolution again,
    the adjoint of the row norms on it, then the taps' adjoints."""
    H, dk, dv = case["heads"], case["d_k"], case["d_v"]
    C, dt = H * (2 * dk + dv), s["x"].dtype
    x = s["x"].reshape(-1, C).float()
    n_tok, w = x.shape[0], s["w"]
    seq, pos, start, lens = _places(case, x.device)
    init = s.get("conv_state")
    at = torch.arange(n_tok, device=x.device)

    def back(j):
        """x_{t-j} of every token: before a sequence's start its carried state."""
        if j == 0:
            return x
        v = torch.where((pos >= j)[:, None], x[(at - j).clamp(min=0)], torch.zeros((), device=x.device))
        if init is not None:
            old = init[seq, :, (3 - j + pos).clamp(max=2)]
            v = torch.where((pos >= j)[:, None], v, old)
        return v

    taps = [back(3 - j) for j in range(4)]
    y = s["bias"] + sum(w[:, j] * taps[j] for j in range(4))
    dq, dk_, dv_ = (s[n].float().reshape(n_tok, H, -1) for n in ("dq", "dk", "dv"))

    def unit_backward(y, d, scale):
        f = scale * torch.rsqrt((y * y).sum(-1, keepdim=True).clamp(min=1e-24))
        return f * d - y * ((f * d * y).sum(-1, keepdim=True) / (y * y).sum(-1, keepdim=True).clamp(min=1e-24))

    yq, yk = y[:, :H * dk].reshape(n_tok, H, dk), y[:, H * dk:2 * H * dk].reshape(n_tok, H, dk)
    dy = torch.cat([unit_backward(yq, dq, math.sqrt(dk)).reshape(n_tok, -1),
                    unit_backward(yk, dk_, 1.0).reshape(n_tok, -1), dv_.reshape(n_tok, -1)], 1)
    dw = torch.stack([(dy * taps[j]).sum(0, dtype=torch.float64) for j in range(4)], 1).float()
    db = dy.sum(0, dtype=torch.float64).float()
    left = lens[seq] - 1 - pos  # tokens of the sequence after this one
    dx = torch.zeros_like(x)
    for j in range(4):
        ahead = dy[(at + j).clamp(max=n_tok - 1)] * w[:, 3 - j]
        dx = dx + torch.where((left >= j)[:, None], ahead, torch.zeros((), device=x.device))
    dinit = None
    if init is not None:
        dfin = s["dconv_state"]
        dx = dx + torch.where((left < 3)[:, None], dfin[seq, :, (2 - left).clamp(min=0)],
                              torch.zeros((), device=x.device))
        # carried sample m meets tap m - t of tokens t <= m, and stays in the
        # state of a sequence of m tokens or fewer
        dinit = torch.zeros_like(init)
        for m in range(3):
            for t in range(m + 1):
                got = dy[(start + t).clamp(max=n_tok - 1)] * w[:, m - t]
                dinit[:, :, m] += torch.where((lens > t)[:, None], got, torch.zeros((), device=x.device))
            stays = (m - lens).clamp(min=0)
            old = torch.gather(dfin, 2, stays[:, None, None].expand(-1, C, 1))[:, :, 0]
            dinit[:, :, m] += torch.where((lens <= m)[:, None], old, torch.zeros((), device=x.device))
    bl, al, a = s["beta_logit"].reshape(-1, H), s["alpha_logit"].reshape(-1, H), s["a_log"]
    dbeta, dg = s["dbeta"].float().reshape(-1, H), s["dg"].float().reshape(-1, H)
    sg = torch.sigmoid(bl)
    dbl = dbeta * sg * (1 - sg)
    dal = -dg * _softplus(a) * torch.sigmoid(al)
    da = (-dg * torch.sigmoid(a) * _softplus(al)).sum(0, dtype=torch.float64).float()
    lead = s["beta_logit"].shape
    out = (dx.to(dt).reshape(s["x"].shape), dw, db, dbl.reshape(lead), dal.reshape(lead), da)
    return out if dinit is None else (*out, dinit)


def _pad_index(case, device, multiple):
    """[N, T] token index of the padded layout (0 where padded), whether it is a token, and T."""
    lens = torch.tensor(_lengths(case), device=device)
    T = -(-max(1, max(_lengths(case))) // multiple) * multiple
    start = torch.cumsum(lens, 0) - lens
    t = torch.arange(T, device=device)
    there = t[None] < lens[:, None]
    return torch.where(there, start[:, None] + t[None], 0), there, T


def _delta_backward(s, case):
    """The chunked adjoint in 32 bits: sequences padded to whole chunks by
    positions that leave the state alone, everything within a chunk at once
    over all chunks, and a loop over chunks for the state and its gradient."""
    H, dk, dv, dt, dev = case["heads"], case["d_k"], case["d_v"], s["q"].dtype, s["q"].device
    idx, there, T = _pad_index(case, dev, CHUNK)
    N, nc, c = idx.shape[0], T // CHUNK, CHUNK

    def chunks(x, fill=0.0, to=torch.float32):
        x = x.to(to)[idx]  # [tokens, H, ...] to [N, T, H, ...]
        m = there.reshape(N, T, *([1] * (x.dim() - 2)))
        x = torch.where(m, x, torch.full((), fill, dtype=to, device=dev))
        return x.reshape(N, nc, c, H, *x.shape[3:]).movedim(3, 1)  # [N, H, nc, c, ...]

    flat = {n: s[n].reshape(-1, *s[n].shape[-2:]) for n in ("q", "k", "v", "do")}
    gate, beta = s["gate"].reshape(-1, H), s["beta"].reshape(-1, H)
    q, k, v, do = (chunks(flat[n]) for n in ("q", "k", "v", "do"))
    b = chunks(beta)
    ln = gate.double() if case["gate"] == "log" else torch.log(gate.double())
    G = torch.cumsum(chunks(ln.clamp(min=-1000.0), 0.0, torch.float64), -1)
    Gc = G[..., -1:]
    gamma, tail, gc = torch.exp(G).float(), torch.exp(Gc - G).float(), torch.exp(Gc).float()
    low = torch.ones(c, c, device=dev, dtype=torch.bool).tril()
    D = torch.where(low, torch.exp(torch.where(low, G[..., :, None] - G[..., None, :], 0.0)).float(), 0.0)
    kk, qk = k @ k.mT, q @ k.mT
    L = (D * kk).tril(-1)
    # the inverse of I + L diag(beta), a unit triangle of 64: the product of
    # I + (-A)^(2^j), j < 6
    eye = torch.eye(c, device=dev)
    A = -L * b[..., None, :]
    Tm = eye + A
    for _ in range(5):
        A = A @ A
        Tm = Tm + Tm @ A
    P = D * qk
    Wt, Wk = Tm @ v, Tm @ (gamma[..., None] * k)
    Tb = Tm.mT * b[..., None, :]
    dXt, Kd = Tb @ (P.mT @ do), Tb @ (tail[..., None] * k)
    write = (b * tail)[..., None] * k
    S = s["state"] if "state" in s else torch.zeros(N, H, dv, dk, device=dev)
    S0, W = torch.empty(N, H, nc, dv, dk, device=dev), torch.empty_like(v)
    for n in range(nc):
        S0[:, :, n] = S
        W[:, :, n] = Wt[:, :, n] - Wk[:, :, n] @ S.mT
        S = gc[:, :, n, :, None] * S + W[:, :, n].mT @ write[:, :, n]
    dS = s["dfinal"] if "dfinal" in s else torch.zeros(N, H, dv, dk, device=dev)
    dS1, dX = torch.empty_like(S0), torch.empty_like(v)
    gq, gk = gamma[..., None] * q, gamma[..., None] * k
    for n in reversed(range(nc)):
        dS1[:, :, n] = dS
        dX[:, :, n] = dXt[:, :, n] + Kd[:, :, n] @ dS.mT
        dS = gc[:, :, n, :, None] * dS + do[:, :, n].mT @ gq[:, :, n] - dX[:, :, n].mT @ gk[:, :, n]
    E1, E2 = do @ W.mT, dX @ W.mT
    N1, N2 = E1 * D * b[..., None, :], (E2 * D * b[..., None, :]).tril(-1)
    Zq, Zk, Zw = do @ S0, dX @ S0, W @ dS1
    dq = gamma[..., None] * Zq + N1 @ k
    dkk = (b * tail)[..., None] * Zw - gamma[..., None] * Zk + N1.mT @ q - N2 @ k - N2.mT @ k
    kw = tail * (k * Zw).sum(-1)
    dbeta = kw + (P * E1 - L * E2).sum(-2)
    a = gamma * ((q * Zq).sum(-1) - (k * Zk).sum(-1))
    M = (N1 * qk - N2 * kk).tril(-1)
    before = torch.cumsum(M, -1) - M  # over s < t
    dg = torch.where(low, before, 0.0).sum(-2)
    dg = dg + a.flip(-1).cumsum(-1).flip(-1) + torch.cumsum(b * kw, -1) - b * kw + gc * (dS1 * S0).sum((-1, -2))[..., None]

    def tokens(x, like):
        x = x.movedim(1, 3).reshape(N, T, *x.shape[1:2], *x.shape[4:])
        return x[there].to(dt).reshape(like.shape)

    if case["gate"] == "alpha":
        dg = dg / chunks(gate, 1.0)
    out = (tokens(dq, s["q"]), tokens(dkk, s["k"]), tokens(dX, s["v"]), tokens(dg, s["gate"]), tokens(dbeta, s["beta"]))
    return (*out, dS) if case["init"] == "trained" else out


_PLAIN = {"delta_backward": _delta_backward, "block_backward": _block_backward, "norm_backward": _rows_norm_backward,
          "layernorm": _layernorm}


# ------------------------------------------------------------------- exact
def _exact_delta(s, case):
    """Token by token in 64 bits: states kept every 128 positions on the way
    forward, each stretch again on the way back."""
    H, dk, dv, dev = case["heads"], case["d_k"], case["d_v"], s["q"].device
    idx, there, T = _pad_index(case, dev, 1)
    N = idx.shape[0]

    def pad(x, fill):
        x = x.double()[idx]
        return torch.where(there.reshape(N, T, *([1] * (x.dim() - 2))), x, torch.tensor(fill, dtype=torch.float64, device=dev))

    q, k, v, do = (pad(s[n].reshape(-1, *s[n].shape[-2:]), 0.0) for n in ("q", "k", "v", "do"))
    gate = s["gate"].reshape(-1, H).double()
    al, be = pad(gate.exp() if case["gate"] == "log" else gate, 1.0), pad(s["beta"].reshape(-1, H), 0.0)

    def mv(S, x):
        return (S @ x[..., None])[..., 0]

    def step(S, t):
        a, b = al[:, t, :, None], be[:, t, :, None]
        u = b * (v[:, t] - a * mv(S, k[:, t]))
        return a[..., None] * S + u[..., None] * k[:, t, :, None, :], u

    S = s["state"].double() if "state" in s else torch.zeros(N, H, dv, dk, dtype=torch.float64, device=dev)
    span, kept = 128, []
    for t in range(T):
        if t % span == 0:
            kept.append(S)
        S, _ = step(S, t)
    dS = s["dfinal"].double() if "dfinal" in s else torch.zeros_like(S)
    dq, dk_, dv_, dal, dbe = (torch.empty_like(x) for x in (q, k, v, al, be))
    for t0 in reversed(range(0, T, span)):
        Ss = [kept.pop()]
        for t in range(t0, min(t0 + span, T)):
            Ss.append(step(Ss[-1], t)[0])
        for t in reversed(range(t0, min(t0 + span, T))):
            S1, S = Ss.pop(), Ss[-1]
            a, b, kt = al[:, t, :, None], be[:, t, :, None], k[:, t]
            dS = dS + do[:, t, :, :, None] * q[:, t, :, None, :]
            dq[:, t] = mv(S1.mT, do[:, t])
            p = mv(S, kt)
            u, du = b * (v[:, t] - a * p), mv(dS, kt)
            dv_[:, t] = b * du
            dbe[:, t] = (du * (v[:, t] - a * p)).sum(-1)
            dp = -a * b * du
            dal[:, t] = (dS * S).sum((-1, -2)) - (b * du * p).sum(-1)
            dk_[:, t] = mv(dS.mT, u) + mv(S.mT, dp)
            dS = a[..., None] * dS + dp[..., None] * kt[..., None, :]
    if case["gate"] == "log":
        dal = dal * al
    out = tuple(x[there].reshape(y.shape) for x, y in ((dq, s["q"]), (dk_, s["k"]), (dv_, s["v"]), (dal, s["gate"]),
                                                       (dbe, s["beta"])))
    return (*out, dS) if case["init"] == "trained" else out


def _exact_block(s, case):
    """Sequence by sequence in 64 bits, the derivative by torch's own of the
    forward formulas."""
    H, dk, dv = case["heads"], case["d_k"], case["d_v"]
    C = H * (2 * dk + dv)
    x, w, bias, bl, al, a = (s[n].double().reshape(sh).requires_grad_(True) for n, sh in (
        ("x", (-1, C)), ("w", (C, 4)), ("bias", (C,)), ("beta_logit", (-1, H)), ("alpha_logit", (-1, H)),
        ("a_log", (H,))))
    init = s["conv_state"].double().requires_grad_(True) if "conv_state" in s else None
    loss, at = 0.0, 0
    for i, n in enumerate(_lengths(case)):
        head = init[i].T if init is not None else torch.zeros(3, C, dtype=torch.float64, device=x.device)
        xx = torch.cat([head, x[at:at + n]])
        if init is not None:
            loss = loss + (xx[n:].T * s["dconv_state"][i].double()).sum()
        y = bias + w[:, 0] * xx[:n] + w[:, 1] * xx[1:n + 1] + w[:, 2] * xx[2:n + 2] + w[:, 3] * xx[3:]
        d = {m: s[m].double().reshape(-1, H * e)[at:at + n] for m, e in (("dq", dk), ("dk", dk), ("dv", dv))}
        for part, scale, m in ((y[:, :H * dk], math.sqrt(dk), "dq"), (y[:, H * dk:2 * H * dk], 1.0, "dk")):
            r = part.reshape(n, H, dk)
            r = r / (r * r).sum(-1, keepdim=True).sqrt() * scale
            loss = loss + (r.reshape(n, H * dk) * d[m]).sum()
        loss = loss + (y[:, 2 * H * dk:] * d["dv"]).sum()
        at += n
    g = -_softplus(a) * _softplus(al)
    loss = loss + (torch.sigmoid(bl) * s["dbeta"].double().reshape(-1, H)).sum()
    loss = loss + (g * s["dg"].double().reshape(-1, H)).sum()
    leaves = [x, w, bias, bl, al, a] + ([init] if init is not None else [])
    d = torch.autograd.grad(loss, leaves)
    lead = s["beta_logit"].shape
    return (d[0].reshape(s["x"].shape), d[1], d[2], d[3].reshape(lead), d[4].reshape(lead), *d[5:])


def _exact_norm(s, case):
    centre = case["op"] == "layernorm"
    x, dy, w = s["x"].double(), s["dy"].double(), s["scale"].double()
    mu = x.sum(-1, keepdim=True) / x.shape[-1] if centre else 0.0
    sd = (((x - mu) ** 2).sum(-1, keepdim=True) / x.shape[-1] + (1e-5 if centre else 1e-6)).sqrt()
    xh = (x - mu) / sd
    gx = dy * w
    proj = xh * ((gx * xh).sum(-1, keepdim=True) / x.shape[-1])
    if not centre:
        return (gx - proj) / sd, (dy * xh).sum(0)
    dx = (gx - gx.sum(-1, keepdim=True) / x.shape[-1] - proj) / sd
    return xh * w + s["bias"].double(), dx, (dy * xh).sum(0), dy.sum(0)


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "delta_backward":
        return _exact_delta(s, case)
    if case["op"] == "block_backward":
        return _exact_block(s, case)
    return _exact_norm(s, case)


def work(case):
    """Bytes: every input and output once.  Flops of the delta rule's
    backward: the chunked form's, per (chunk of c <= 64 tokens, head)
    12 c^2 d_k + 8 c^2 d_v + 16 c d_k d_v; of the others a few per element."""
    e = 2 if case["dtype"] == "bf16" else 4
    if case["op"] in ("norm_backward", "layernorm"):
        n = case["rows"] * case["dim"]
        passes = 3 if case["op"] == "norm_backward" else 4  # x, dy and dx; layer norm's y too
        return {"bytes": passes * n * e + 4.0 * case["dim"] * 4, "flops": 16.0 * n}
    H, dk, dv = case["heads"], case["d_k"], case["d_v"]
    lens = _lengths(case)
    unit = sum(lens) * H
    if case["op"] == "block_backward":
        C = H * (2 * dk + dv)
        states = len(lens) * C * 3 * 4 * (3 if case["init"] else 0)
        return {"bytes": unit * (3 * (2 * dk + dv) * e + 4 * 4 + 2 * e) + C * 36.0 + states,
                "flops": unit * (2 * dk + dv) * 32.0}
    flops = 0.0
    for n in lens:
        for c, times in ((CHUNK, n // CHUNK), (n % CHUNK, 1)):
            flops += H * times * (12.0 * c * c * dk + 8.0 * c * c * dv + 16.0 * c * dk * dv)
    states = len(lens) * H * dk * dv * 4 * {"": 0, "carried": 1, "trained": 3}[case["init"]]
    return {"bytes": unit * ((4 * dk + 3 * dv) * e + 8 + 2 * e) + states, "flops": flops}
