"""Latent attention in 64 bits on the CPU, with bounds of what the kernels may be off by.

Bounds are first-order sums of roundings, taken where the kernels round: u =
eps / 2 of the tensors' type (2^-8 in bf16: results, and weights before they
meet the values; 2^-24 in fp32) and w = 2^-24 for every fp32 sum, whose terms
each take part in at most as many additions as there are terms.  A score's error
d_s is that of its product; a weight's, relative, at most that of its own score
and of the sum's (2 d_s), of the exponent's argument, which is rounded at
magnitude log2 of the weight and a maximum of scores (m), and of the exponential.
"""
import math

import torch

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
W = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def visible(n, m, causal):
    if not causal:
        return torch.ones(n, m, dtype=torch.bool)
    return torch.arange(m) <= torch.arange(n)[:, None] + (m - n)


def scores(q, k, r, scale):
    """[H, n, m] scores and, of the same shape, the sums of their terms' magnitudes."""
    q = q.double().transpose(0, 1)
    keys = k.double().transpose(0, 1)
    if r is not None:
        keys = torch.cat([keys, r.double().expand(keys.shape[0], -1, -1)], -1)
    return scale * q @ keys.mT, scale * q.abs() @ keys.abs().mT, keys


def weights(s, size, seen, terms):
    """Softmax over what is seen, its logarithm of sums, and the relative error that fp32 may leave in a weight."""
    s = s.masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    e = torch.exp(s - top)
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total == 0, torch.ones_like(total), total)
    lse = (torch.log(total) + top)[..., 0]
    size = torch.where(seen, size, torch.zeros_like(size))
    d_s = (terms + 4) * W * size.amax(-1, keepdim=True)  # the products, scale and its logarithm's base
    m = torch.where(seen, s.abs(), torch.zeros_like(s)).amax(-1, keepdim=True)
    rel = 2 * d_s + 8 * W * (m + 1) + (s.shape[-1] + 8) * W
    return p, lse, rel


def attend(q, k, v, r, scale, causal, dtype):
    """One sequence: o [n, H, d_v], lse [n, H] and the bounds of both."""
    n, m = q.shape[0], k.shape[0]
    if m == 0:
        o = torch.zeros(n, q.shape[1], v.shape[-1], dtype=torch.float64)
        return o, torch.full((n, q.shape[1]), -math.inf, dtype=torch.float64), o, torch.zeros(n, q.shape[1])
    s, size, _ = scores(q, k, r, scale)
    p, lse, rel = weights(s, size, visible(n, m, causal), q.shape[-1])
    v = v.double().transpose(0, 1)
    o, around = p @ v, p @ v.abs()
    u = half_step(dtype)
    rounded = u if dtype == torch.bfloat16 else 0.0
    tol = u * o.abs() + (rel + rounded + (m + 8) * W) * around * (1 + 2 * u) + 1e-37
    lse_tol = rel[..., 0] + 4 * W * lse.abs().masked_fill(torch.isinf(lse), 0.0)
    return o.transpose(0, 1), lse.T, tol.transpose(0, 1), lse_tol.T


def attend_backward(q, k, v, r, do, dlse, scale, causal, dtype):
    """One sequence: (dq, dk, dv, dr) and their bounds, where o and lse are the
    forward kernel's: o rounded, lse off by what `weights` says."""
    n, m, H = q.shape[0], k.shape[0], q.shape[1]
    d_n = k.shape[-1]
    seen = visible(n, m, causal)
    s, size, keys = scores(q, k, r, scale)
    p, lse, rel = weights(s, size, seen, q.shape[-1])
    qd, vd, dod = (t.double().transpose(0, 1) for t in (q, v, do))
    o = p @ vd
    dp, dp_size = dod @ vd.mT, dod.abs() @ vd.abs().mT
    delta = (dod * o).sum(-1, keepdim=True)
    d_size = (dod * o).abs().sum(-1, keepdim=True)
    if dlse is not None:
        delta = delta - dlse.double().T[..., None]
        d_size = d_size + dlse.double().abs().T[..., None]
    ds = p * (dp - delta)
    u = half_step(dtype)
    rounded = u if dtype == torch.bfloat16 else 0.0
    rel = rel * 2  # lse's error beside the weight's own
    o_size = (dod.abs() * (p @ vd.abs())).sum(-1, keepdim=True)  # what o's own error is relative to
    d_delta = u * d_size + (rel + rounded + 2 * v.shape[-1] * W + (m + 8) * W) * (d_size + o_size)
    e_p = (rel + rounded) * p
    e_ds = rel * ds.abs() + p * (d_delta + (v.shape[-1] + 4) * W * dp_size) + rounded * ds.abs() + 4 * W * p * (dp_size + d_size)

    def out(x, tol, terms, around):
        return x, u * x.abs() + tol * (1 + 2 * u) + (terms + 8) * W * around + 1e-37

    dq, dq_t = out(scale * ds @ keys, scale * e_ds @ keys.abs(), m, scale * ds.abs() @ keys.abs())
    dk, dk_t = out(scale * ds.mT @ qd, scale * e_ds.mT @ qd.abs(), n, scale * ds.abs().mT @ qd.abs())
    dv, dv_t = out(p.mT @ dod, e_p.mT @ dod.abs(), n, p.mT @ dod.abs())
    res = {"dq": (dq, dq_t), "dk": (dk[..., :d_n], dk_t[..., :d_n]), "dv": (dv, dv_t)}
    res = {name: (a.transpose(0, 1), b.transpose(0, 1)) for name, (a, b) in res.items()}
    if r is not None:
        dr, tail = dk[..., d_n:].sum(0), dk_t[..., d_n:].sum(0)
        res["dr"] = (dr, tail + u * dr.abs() + H * W * dk[..., d_n:].abs().sum(0))
    return res


def near(got, want, tol, what=""):
    got = got.double().cpu()
    assert got.shape == want.shape, f"{what}: {tuple(got.shape)} is not {tuple(want.shape)}"
    same = got == want  # infinities
    off = torch.where(same, torch.zeros_like(want), (got - want).abs())
    bad = ~(off <= tol)
    worst = float((off / tol.clamp(min=1e-300)).max()) if off.numel() else 0.0
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} outside, {worst:.3g} of the bound"


def normal(shape, gen, dtype, std=1.0):
    return (torch.randn(shape, generator=gen) * std).to(dtype)


def make(lens, keys, H, d_n, d_r, d_v, dtype, seed=0, sharp=1.0):
    """Packed inputs of sequences of `lens` queries and `keys` keys; k and v are halves of one tensor."""
    gen = torch.Generator().manual_seed(seed)
    nq, nk = sum(lens), sum(keys)
    q = normal((nq, H, d_n + d_r), gen, dtype, sharp)
    kv = normal((nk, H, d_n + d_v), gen, dtype)
    r = normal((nk, d_r), gen, dtype) if d_r else None
    do = normal((nq, H, d_v), gen, dtype)
    return q, kv, r, do


def starts(lens):
    return torch.tensor([0, *torch.tensor(lens).cumsum(0).tolist()], dtype=torch.int32)
