"""Backward pass of the Local block's prologue against torch's derivative of
its formulas in 64 bits on the CPU, and the whole training pass of a block's
mixer: layer norm, prologue, delta rule, per-head norm, and back.

Tolerances of the 2-norm, set before the first run: fp32 outputs 3e-6 (some 40
operations of half a step, 2^-24, on a value); a bf16 dx half a step, 2^-8,
more; sums over tokens are held against the norm of the sums of magnitudes.
"""
import math

import pytest
import torch

import rhizome_amd

pytestmark = pytest.mark.gpu
F32_TOL, BF16_TOL = 3e-6, 2.0 ** -8 + 3e-6
NAMES = ("dx", "dweight", "dbias", "dbeta_logit", "dalpha_logit", "da_log", "dinitial_state")
DTYPES = [torch.float32, torch.bfloat16]


def make(lengths, H, dk, dv, dtype, seed=0, state=True):
    gen = torch.Generator().manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen)

    n, C = sum(lengths), H * (2 * dk + dv)
    s = dict(x=normal(n, C).to(dtype), weight=normal(C, 4) * 0.5, bias=normal(C) * 0.1, beta_logit=normal(n, H),
             alpha_logit=normal(n, H) * 2, a_log=normal(H), dq=normal(n, H, dk).to(dtype), dk=normal(n, H, dk).to(dtype),
             dv=normal(n, H, dv).to(dtype), dbeta=normal(n, H).to(dtype), dg=normal(n, H).to(dtype))
    if state:
        s["initial_state"], s["dfinal_state"] = normal(len(lengths), C, 3), normal(len(lengths), C, 3)
    return s


def softplus(x):
    return torch.where(x > 30, x, torch.log1p(torch.exp(x)))


def prologue(x, weight, bias, beta_logit, alpha_logit, a_log, state, lengths, H, dk, dv, q_scale):
    """Outputs of the forward pass by formula, and the final conv states."""
    ys, finals, at = [], [], 0
    for i, n in enumerate(lengths):
        xx = torch.cat([state[i].T, x[at:at + n]])
        ys.append(bias + sum(weight[:, j] * xx[j:j + n] for j in range(4)))
        finals.append(xx[n:].T)
        at += n
    y = torch.cat(ys)
    q, k, v = (t.reshape(-1, H, d) for t, d in zip(y.split([H * dk, H * dk, H * dv], 1), (dk, dk, dv)))
    norm = lambda t: t / t.norm(dim=-1, keepdim=True).clamp(min=1e-12)  # noqa: E731
    return norm(q) * q_scale, norm(k), v, torch.sigmoid(beta_logit), -softplus(a_log) * softplus(alpha_logit), \
        torch.stack(finals)


def reference(s, lengths, H, dk, dv, q_scale):
    """Gradients, and for each the magnitudes that its terms have."""
    names = ("x", "weight", "bias", "beta_logit", "alpha_logit", "a_log")
    leaf = [s[n].double().requires_grad_(True) for n in names]
    C = leaf[0].shape[1]
    state = (s["initial_state"].double() if "initial_state" in s
             else torch.zeros(len(lengths), C, 3, dtype=torch.float64)).requires_grad_(True)
    out = prologue(*leaf, state, lengths, H, dk, dv, q_scale)
    grads = [s[n].double() for n in ("dq", "dk", "dv", "dbeta", "dg")]
    loss = sum((o * g).sum() for o, g in zip(out, grads))
    if "dfinal_state" in s:
        loss = loss + (out[5] * s["dfinal_state"].double()).sum()
    return torch.autograd.grad(loss, leaf + [state])


def call(s, lengths, H, dk, dv, device, dense=False, q_scale=None, **kw):
    a = {n: t.to(device) for n, t in s.items()}
    if dense:
        B, T = len(lengths), lengths[0]
        per_token = ("x", "beta_logit", "alpha_logit", "dq", "dk", "dv", "dbeta", "dg")
        a = {n: t.reshape(B, T, *t.shape[1:]) if n in per_token else t for n, t in a.items()}
    else:
        a["cu_seqlens"] = torch.tensor([0] + list(torch.tensor(lengths).cumsum(0)), dtype=torch.int32, device=device)
    out = rhizome_amd.conv_prepare_backward(**a, heads=H, d_k=dk, d_v=dv, q_scale=q_scale, **kw)
    torch.cuda.synchronize()
    flat = lambda n, t: t.reshape(-1, t.shape[-1]) if n in ("dx", "dbeta_logit", "dalpha_logit") else t  # noqa: E731
    return [None if t is None else flat(n, t).cpu() for n, t in zip(NAMES, out)]


def check(got, want, s, dtype):
    n = max(1, s["x"].shape[0])
    for name, x, y in zip(NAMES, got, want):
        if x is None:
            continue
        assert x.shape == y.shape and bool(torch.isfinite(x).all()), name
        tol = BF16_TOL if name == "dx" and dtype == torch.bfloat16 else F32_TOL
        # sums of n terms of random sign are about sqrt(n) below their magnitudes' sum
        room = math.sqrt(n) if name in ("dweight", "dbias", "da_log") else 1.0
        err, norm = float((x.double() - y).norm()), float(y.norm())
        assert err <= tol * norm * room + 1e-30, f"{name}: {err / max(norm, 1e-300):.3g}, tolerance {tol * room:.3g}"


SHAPES = [
    # lengths, H, d_k, d_v
    ([1], 1, 32, 32), ([2, 2], 2, 16, 8), ([3], 1, 8, 16), ([4, 1, 2, 3, 0, 5], 2, 32, 32), ([16], 1, 64, 64), ([17], 3, 32, 40),
    ([64, 64], 2, 128, 128), ([0, 0, 33, 0, 100, 1, 0], 2, 64, 32), ([300], 2, 256, 64), ([515], 16, 32, 32),
]


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("state", [True, False], ids=["state", "zeros"])
@pytest.mark.parametrize("lengths,H,dk,dv", SHAPES)
def test_shapes(device, dtype, state, lengths, H, dk, dv):
    s = make(lengths, H, dk, dv, dtype, seed=dk + len(lengths), state=state)
    want = reference(s, lengths, H, dk, dv, math.sqrt(dk))
    check(call(s, lengths, H, dk, dv, device), want, s, dtype)
    if len(set(lengths)) == 1:
        check(call(s, lengths, H, dk, dv, device, dense=True), want, s, dtype)


def test_more_tokens_than_spans(device):
    """Spans longer than the shortest, crossing sequences; a scale of its own."""
    lengths = [3000, 1, 2, 2900, 0, 3000]
    s = make(lengths, 2, 32, 32, torch.float32, seed=3)
    check(call(s, lengths, 2, 32, 32, device, q_scale=0.7), reference(s, lengths, 2, 32, 32, 0.7), s, torch.float32)


def test_zero_rows_and_large_logits(device):
    """A convolved row of zeros (the norm's floor), saturated gates."""
    s = make([40], 2, 32, 32, torch.float32, seed=4, state=False)
    s["bias"][:64], s["x"][10:20] = 0.0, 0.0
    s["alpha_logit"][:5], s["alpha_logit"][5:9], s["beta_logit"][:4], s["beta_logit"][4:8] = 80.0, -80.0, 90.0, -90.0
    s["a_log"][1] = 50.0
    s["dq"][13:20], s["dk"][13:20] = 0.0, 0.0  # the rows of zeros: their gradient is 1e12 times the one that comes in
    got, want = call(s, [40], 2, 32, 32, device), reference(s, [40], 2, 32, 32, math.sqrt(32))
    want = [torch.nan_to_num(t) for t in want]  # log1p(exp(80)) is not taken, but its derivative is formed
    check(got, want, s, torch.float32)


def test_without_bias_and_rows_outside(device):
    s = make([60], 2, 32, 32, torch.bfloat16, seed=5, state=False)
    s["bias"] = torch.zeros_like(s["bias"])
    want = call(s, [60], 2, 32, 32, device)
    a = {n: t.to(device) for n, t in s.items() if n != "bias"}
    got = rhizome_amd.conv_prepare_backward(**a, bias=None, heads=2, d_k=32, d_v=32,
                                            cu_seqlens=torch.tensor([0, 60], dtype=torch.int32, device=device))
    assert got[2] is None and got[6] is None and torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])
    # the pack's first 7 and last 11 rows belong to no sequence
    per_token = ("x", "beta_logit", "alpha_logit", "dq", "dk", "dv", "dbeta", "dg")
    inner = {n: t[7:49] if n in per_token else t for n, t in s.items()}
    want = call(inner, [20, 22], 2, 32, 32, device)
    a = {n: t.to(device) for n, t in s.items()}
    marked = rhizome_amd.train._empty
    rhizome_amd.train._empty = lambda like, shape, dtype=None: marked(like, shape, dtype).fill_(77)
    try:
        got = rhizome_amd.conv_prepare_backward(**a, heads=2, d_k=32, d_v=32,
                                                cu_seqlens=torch.tensor([7, 27, 49], dtype=torch.int32, device=device))
    finally:
        rhizome_amd.train._empty = marked
    for i in (0, 3, 4):
        x = got[i].cpu()
        assert torch.equal(x[7:49], want[i]) and bool((x[:7] == 77).all()) and bool((x[49:] == 77).all())
    for i in (1, 2, 5):
        assert float((got[i].cpu() - want[i]).norm()) <= F32_TOL * math.sqrt(42) * float(want[i].norm())


@pytest.mark.parametrize("offsets", [[0, 50, 20, 64], [-3, 900, 10, 10]])
def test_bad_offsets_stay_inside(device, offsets):
    s = make([64], 2, 32, 32, torch.bfloat16, seed=6, state=False)
    a = {n: t.to(device) for n, t in s.items()}
    rhizome_amd.conv_prepare_backward(**a, heads=2, d_k=32, d_v=32,
                                      cu_seqlens=torch.tensor(offsets, dtype=torch.int32, device=device))
    torch.cuda.synchronize()


def test_differences(device):
    """Along a direction, against central differences of the formulas in 64 bits (step 1e-5)."""
    lengths, H, dk, dv = [30, 2], 2, 16, 16
    s = make(lengths, H, dk, dv, torch.float32, seed=7)
    got = call(s, lengths, H, dk, dv, device)
    gen = torch.Generator().manual_seed(8)
    names = ("x", "weight", "bias", "beta_logit", "alpha_logit", "a_log", "initial_state")
    base = {n: t.double() for n, t in s.items()}
    for i, name in enumerate(names):
        way = torch.randn(base[name].shape, generator=gen, dtype=torch.float64)
        ends = []
        for step in (1e-5, -1e-5):
            b = {**base, name: base[name] + step * way}
            out = prologue(*(b[n] for n in names), lengths, H, dk, dv, math.sqrt(dk))
            given = [b[n] for n in ("dq", "dk", "dv", "dbeta", "dg", "dfinal_state")]
            ends.append(float(sum((o * g).sum() for o, g in zip(out, given))))
        slope, mine = (ends[0] - ends[1]) / 2e-5, float((got[i].double() * way).sum())
        assert abs(slope - mine) <= 1e-5 * float(got[i].double().norm() * way.norm()), name


def test_stream_graph_and_same_bits(device):
    s = make([70, 70], 2, 64, 64, torch.bfloat16, seed=9)
    want = call(s, [70, 70], 2, 64, 64, device, dense=True)
    got = call(s, [70, 70], 2, 64, 64, device, dense=True, stream=torch.cuda.Stream())
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    per_token = ("x", "beta_logit", "alpha_logit", "dq", "dk", "dv", "dbeta", "dg")
    a = {n: (t.reshape(2, 70, *t.shape[1:]) if n in per_token else t).to(device) for n, t in s.items()}
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rhizome_amd.conv_prepare_backward(**a, heads=2, d_k=64, d_v=64)
    for f in (1.0, 0.5, 2.0):
        a["dv"].copy_(a["dv"] * f)
        s["dv"] = s["dv"] * f
        graph.replay()
        torch.cuda.synchronize()
        want = call(s, [70, 70], 2, 64, 64, device, dense=True)
        assert torch.equal(out[0].cpu().reshape(want[0].shape), want[0]) and torch.equal(out[1].cpu(), want[1])


def test_refusals(device):
    a = {n: t.to(device) for n, t in make([10], 2, 32, 32, torch.bfloat16).items()}
    a["cu_seqlens"] = torch.tensor([0, 10], dtype=torch.int32, device=device)
    kw = dict(heads=2, d_k=32, d_v=32)
    for over in (dict(dq=a["dq"].float()), dict(dg=a["dg"][:5]), dict(weight=a["weight"][:, :3].contiguous()),
                 dict(x=a["x"].half()), dict(initial_state=a["initial_state"][:, :, :2].contiguous()), dict(heads=3),
                 dict(cu_seqlens=a["cu_seqlens"].long()), dict(a_log=None)):
        with pytest.raises((ValueError, AttributeError)):
            rhizome_amd.conv_prepare_backward(**{**a, **kw, **over})
    odd = {n: t.to(device) for n, t in make([10], 2, 24, 32, torch.bfloat16).items()}
    with pytest.raises(rhizome_amd.gdr.GdrError):
        rhizome_amd.conv_prepare_backward(**odd, cu_seqlens=a["cu_seqlens"], heads=2, d_k=24, d_v=32)
    with pytest.raises(rhizome_amd.gdr.GdrError):
        rhizome_amd.conv_prepare_backward(**a, **kw, q_scale=math.inf)


# ---------------------------------------------------------------- together
@pytest.mark.parametrize("dtype,tol", [(torch.float32, 2e-5), (torch.bfloat16, 4e-2)], ids=["f32", "bf16"])
def test_a_block_forward_and_back(device, dtype, tol):
    """The mixer of a Local block as it trains: layer norm, projection, prologue,
    delta rule, per-head norm, against torch in 64 bits over two packed
    sequences.  fp32: three operators of 3e-6 and two products of 2e-6 deep.
    bf16: nine tensors on the way are rounded to 2^-8 each, on the way there
    and back: 9 * 2^-8 = 3.5e-2."""
    lengths, H, dk, dv, width = [90, 47], 2, 32, 32, 96
    n, C = sum(lengths), H * (2 * dk + dv)
    gen = torch.Generator().manual_seed(10)

    def normal(*shape, std=1.0):
        return torch.randn(shape, generator=gen, dtype=torch.float64) * std

    h, dout = normal(n, width).to(dtype), normal(n, H, dv).to(dtype)
    nw, nb, proj = normal(width, std=0.1) + 1, normal(width, std=0.1), normal(width, C, std=width ** -0.5).to(dtype)
    weight, bias, a_log, scale = normal(C, 4, std=0.5), normal(C, std=0.1), normal(H), normal(dv, std=0.1) + 1
    bl, al = normal(n, H).float(), normal(n, H).float()
    nw, nb, weight, bias, a_log, scale = (t.float() for t in (nw, nb, weight, bias, a_log, scale))

    leaf = [t.double().requires_grad_(True) for t in (h, nw, nb, proj, weight, bias, bl, al, a_log, scale)]
    lh, lnw, lnb, lproj, lw, lb, lbl, lal, la, ls = leaf
    hc = lh - lh.mean(-1, keepdim=True)
    x = (hc / torch.sqrt((hc * hc).mean(-1, keepdim=True) + 1e-5) * lnw + lnb) @ lproj
    zero = torch.zeros(2, C, 3, dtype=torch.float64)
    q, k, v, beta, g, _ = prologue(x, lw, lb, lbl, lal, la, zero, lengths, H, dk, dv, math.sqrt(dk))
    outs, at = [], 0
    for length in lengths:
        S = torch.zeros(H, dv, dk, dtype=torch.float64)
        for t in range(at, at + length):
            a, b = g[t].exp(), beta[t]
            u = b[:, None] * (v[t] - a[:, None] * (S @ k[t][..., None])[..., 0])
            S = a[:, None, None] * S + u[..., None] * k[t][:, None, :]
            outs.append((S @ q[t][..., None])[..., 0])
        at += length
    o = torch.stack(outs)
    y = o / torch.sqrt((o * o).mean(-1, keepdim=True) + 1e-6) * ls
    want = torch.autograd.grad((y * dout.double()).sum(), leaf)

    dev = lambda *ts: [t.to(device) for t in ts]  # noqa: E731
    h, dout, nw, nb, proj, weight, bias, a_log, scale, bl, al = dev(h, dout, nw, nb, proj, weight, bias, a_log, scale, bl,
                                                                     al)
    cu = torch.tensor([0, 90, 137], dtype=torch.int32, device=device)
    kw = dict(heads=H, d_k=dk, d_v=dv, cu_seqlens=cu)
    hn = rhizome_amd.layernorm(h, nw, nb)
    x = hn @ proj
    q, k, v, beta, g, _ = rhizome_amd.conv_prepare(x, weight, bias, bl, al, a_log, **kw)
    o, _ = rhizome_amd.prefill(q, k, v, g, beta, cu_seqlens=cu)
    do, dscale = rhizome_amd.rmsnorm_heads_backward(dout, o, scale)
    dq, dk_, dv_, dg, dbeta, _ = rhizome_amd.prefill_backward(q, k, v, g, beta, do, cu_seqlens=cu)
    dx, dw, db, dbl, dal, da, _ = rhizome_amd.conv_prepare_backward(x, weight, bias, bl, al, a_log, dq, dk_, dv_, dbeta,
                                                                   dg, **kw)
    dproj = hn.T.contiguous() @ dx
    dh, dnw, dnb = rhizome_amd.layernorm_backward(dx @ proj.T.contiguous(), h, nw)
    got = (dh, dnw, dnb, dproj, dw, db, dbl, dal, da, dscale)
    names = ("h", "norm weight", "norm bias", "projection", "conv weight", "conv bias", "beta logit", "alpha logit",
             "a_log", "scale")
    for name, a, b in zip(names, got, want):
        err = float((a.double().cpu() - b).norm()) / float(b.norm())
        assert err <= tol, f"{name}: {err:.3g}"
