"""Latent attention over expanded keys and values, and its backward pass,
against the formulas in 64 bits; bounds as attn_cases.py derives them."""
import math

import pytest
import torch

import rhizome_amd
from attn_cases import DTYPES, attend, attend_backward, make, near, starts

pytestmark = pytest.mark.gpu


def check(lens, keys, H, d_n, d_r, d_v, dtype, device, causal=True, dense=False, seed=0, sharp=1.0, scale=None, dlse=False,
          backward=True):
    scale = (d_n + d_r) ** -0.5 if scale is None else scale
    q, kv, r, do = make(lens, keys, H, d_n, d_r, d_v, dtype, seed, sharp)
    dl = torch.randn(sum(lens), H, generator=torch.Generator().manual_seed(seed + 1)) if dlse else None
    if dense:
        shape = lambda t, n: t if t is None else t.reshape(len(n), n[0], *t.shape[1:])
        cu = cu_k = None
    else:
        shape = lambda t, n: t
        cu = starts(lens).to(device)
        cu_k = starts(keys).to(device) if keys != lens else None
    dq, dkv, dr = shape(q, lens).to(device), shape(kv, keys).to(device), shape(r, keys)
    dr = dr.to(device) if r is not None else None
    args = (dq, dkv[..., :d_n], dkv[..., d_n:], dr)
    kw = dict(scale=scale, causal=causal, cu_seqlens=cu, cu_seqlens_k=cu_k)
    o, lse = rhizome_amd.latent_prefill(*args, **kw)
    ddo = shape(do, lens).to(device)
    ddl = shape(dl, lens).to(device) if dlse else None
    got = rhizome_amd.latent_prefill_backward(*args, o, lse, ddo, dlse=ddl, **kw) if backward else None
    torch.cuda.synchronize()
    flat = lambda t: t.reshape(-1, *t.shape[2:]) if dense else t
    o, lse = flat(o), flat(lse)
    if backward:
        got = dict(zip(("dq", "dk", "dv", "dr"), (flat(t) if t is not None else None for t in got)))
    q0 = k0 = 0
    for n, m in zip(lens, keys):
        qs, ks = slice(q0, q0 + n), slice(k0, k0 + m)
        one = (q[qs], kv[ks, :, :d_n], kv[ks, :, d_n:], r[ks] if r is not None else None)
        want_o, want_l, tol_o, tol_l = attend(*one, scale, causal, dtype)
        near(o[qs], want_o, tol_o, "o")
        near(lse[qs], want_l, tol_l, "lse")
        if backward and m:
            want = attend_backward(*one, do[qs], dl[qs] if dlse else None, scale, causal, dtype)
            for name, (x, tol) in want.items():
                near(got[name][qs if name == "dq" else ks], x, tol, name)
        elif backward:
            assert not bool(got["dq"][qs].any())
        q0, k0 = q0 + n, k0 + m


@pytest.mark.parametrize("dtype", DTYPES.values(), ids=DTYPES.keys())
@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 300])
def test_lengths(device, dtype, n):
    """Around the sizes of a wave's rows, a tile and a workgroup's rows."""
    check([n], [n], 2, 32, 16, 32, dtype, device, dense=True, seed=n)


@pytest.mark.parametrize("dtype", DTYPES.values(), ids=DTYPES.keys())
@pytest.mark.parametrize("d_n,d_r,d_v", [(64, 32, 64), (128, 0, 128), (128, 64, 128), (64, 64, 128), (96, 0, 96), (128, 16, 64),
                                         (8, 8, 8), (1, 0, 1), (5, 3, 7), (33, 30, 65), (127, 64, 128), (128, 64, 127),
                                         (40, 24, 48), (16, 176, 128), (12, 4, 20)])
def test_widths(device, dtype, d_n, d_r, d_v):
    """Every pair of padded widths, panels that two tensors share, and widths that are no whole chunks."""
    check([150], [150], 2, d_n, d_r, d_v, dtype, device, dense=True, seed=d_n)


@pytest.mark.parametrize("dtype", DTYPES.values(), ids=DTYPES.keys())
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "full"])
@pytest.mark.parametrize("lens,keys", [
    ([5, 0, 130, 1, 64], [5, 0, 130, 1, 64]),
    ([1, 1, 1], [200, 1, 64]),
    ([70, 3, 0, 128], [133, 300, 40, 128]),
    ([100, 10], [37, 0]),  # queries that see no key
    ([0, 0], [3, 0]),
    ([17], [1024]),
])
def test_packs(device, dtype, causal, lens, keys):
    check(lens, keys, 3, 64, 32, 64, dtype, device, causal=causal, seed=len(lens), dlse=True)


@pytest.mark.parametrize("dtype", DTYPES.values(), ids=DTYPES.keys())
@pytest.mark.parametrize("lens,keys", [
    ([300, 0, 700, 1, 129, 128, 513], [300, 5, 900, 400, 129, 100, 513]),
    ([128, 256, 384], [128, 256, 384]),
    ([700, 20], [100, 650]),  # most of its queries see nothing, few see much
    ([1, 600], [600, 1]),
])
def test_packs_of_many_tiles(device, dtype, lens, keys):
    """Whose tiles are worked on by the length of their way, over all sequences."""
    check(lens, keys, 2, 64, 16, 64, dtype, device, seed=len(lens))


@pytest.mark.parametrize("dtype", DTYPES.values(), ids=DTYPES.keys())
@pytest.mark.parametrize("count", [2, 63, 64, 65])
def test_numbers_of_sequences(device, dtype, count):
    lens = [int(x) for x in torch.randint(0, 200, (count,), generator=torch.Generator().manual_seed(count))]
    check(lens, lens, 2, 32, 0, 32, dtype, device, seed=4)


@pytest.mark.parametrize("dtype", DTYPES.values(), ids=DTYPES.keys())
def test_many_sequences(device, dtype):
    """More sequences than a wave has lanes, empty ones among them."""
    lens = [int(x) for x in torch.randint(0, 9, (150,), generator=torch.Generator().manual_seed(2))]
    check(lens, lens, 2, 32, 16, 32, dtype, device, seed=3)


@pytest.mark.parametrize("dtype", DTYPES.values(), ids=DTYPES.keys())
@pytest.mark.parametrize("n,m", [(100, 40), (40, 100), (130, 129), (1, 500), (3, 0), (0, 5)])
def test_dense_rectangles(device, dtype, n, m):
    for causal in (True, False):
        check([n] * 2, [m] * 2, 2, 64, 0, 64, dtype, device, causal=causal, dense=True, seed=n)


@pytest.mark.parametrize("dtype", DTYPES.values(), ids=DTYPES.keys())
def test_sharp_and_flat_weights(device, dtype):
    """Scores of tens, where a row's maximum grows tile after tile, and of next to nothing."""
    check([260], [260], 2, 128, 64, 128, dtype, device, dense=True, sharp=8.0, seed=5)
    check([260], [260], 2, 128, 64, 128, dtype, device, dense=True, scale=1e-6, seed=6)


def test_rows_growing_along_the_keys(device):
    """Keys whose scores rise by less than the 2^8 at which the maximum is raised, and by more."""
    for step in (0.02, 0.3):
        n, d = 400, 32
        q = torch.ones(1, n, 1, d, device=device)
        k = (torch.arange(n, device=device) * step / d).view(1, n, 1, 1).expand(1, n, 1, d).contiguous()
        v = torch.randn(1, n, 1, d, generator=torch.Generator().manual_seed(1)).to(device)
        o, lse = rhizome_amd.latent_prefill(q, k, v, scale=1.0)
        want_o, want_l, tol_o, tol_l = attend(q[0].cpu(), k[0].cpu(), v[0].cpu(), None, 1.0, True, torch.float32)
        near(o[0], want_o, tol_o, "o")
        near(lse[0], want_l, tol_l, "lse")


@pytest.mark.parametrize("dtype", DTYPES.values(), ids=DTYPES.keys())
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf], ids=["nan", "inf", "-inf"])
def test_what_is_not_seen_has_no_part(device, dtype, value):
    """A padded batch: what follows a sequence's real tokens holds anything, and
    the real tokens' results are those of the sequence alone."""
    H, d_n, d_r, d_v, n, real = 2, 64, 32, 64, 150, (70, 129)
    q, kv, r, do = make([n, n], [n, n], H, d_n, d_r, d_v, dtype, seed=9)
    for b, m in enumerate(real):
        for t in (q, kv, r):
            t.view(2, n, *t.shape[1:])[b, m:] = value
    dev = [t.view(2, n, *t.shape[1:]).to(device) for t in (q, kv, r, do)]
    args = (dev[0], dev[1][..., :d_n], dev[1][..., d_n:], dev[2])
    o, lse = rhizome_amd.latent_prefill(*args)
    # the padding's own rows are not the loss's
    o, lse, dod = o.clone(), lse.clone(), dev[3].clone()
    got = rhizome_amd.latent_prefill_backward(*args, o, lse, dod)
    for b, m in enumerate(real):
        cut = (dev[0][b:b + 1, :m], dev[1][b:b + 1, :m, :, :d_n], dev[1][b:b + 1, :m, :, d_n:], dev[2][b:b + 1, :m])
        cut = [t.contiguous() for t in cut]
        o1, l1 = rhizome_amd.latent_prefill(*cut)
        want = rhizome_amd.latent_prefill_backward(*cut, o1, l1, dod[b:b + 1, :m].contiguous())
        one = (q.view(2, n, H, -1)[b, :m], kv.view(2, n, H, -1)[b, :m, :, :d_n], kv.view(2, n, H, -1)[b, :m, :, d_n:],
               r.view(2, n, -1)[b, :m])
        wo, wl, to, tl = attend(*one, (d_n + d_r) ** -0.5, True, dtype)
        near(o[b, :m], wo, to, "o")
        near(lse[b, :m], wl, tl, "lse")
        exact = attend_backward(*one, do.view(2, n, H, -1)[b, :m], None, (d_n + d_r) ** -0.5, True, dtype)
        near(got[0][b, :m], *exact["dq"], "dq")
        for t in (o1, l1, *want):
            assert bool(torch.isfinite(t).all())


@pytest.mark.parametrize("dtype", DTYPES.values(), ids=DTYPES.keys())
def test_leading_padding(device, dtype):
    """Queries in front of a sequence hold anything: dk and dv of the keys behind them do not."""
    H, d, n, pad = 2, 64, 140, 40
    q, kv, _, do = make([n], [n], H, d, 0, d, dtype, seed=11)
    q[:pad], do[:pad] = math.nan, math.inf
    args = (q[None].to(device), kv[None, ..., :d].to(device), kv[None, ..., d:].to(device), None)
    o, lse = rhizome_amd.latent_prefill(*args)
    got = rhizome_amd.latent_prefill_backward(*args, o, lse, do[None].to(device))
    # keys from `pad` on are seen by the real queries alone
    q2, do2 = q.clone(), do.clone()
    q2[:pad], do2[:pad] = 0.0, 0.0
    want = attend_backward(q2, kv[..., :d], kv[..., d:], None, do2, None, d ** -0.5, True, dtype)
    for name, t in (("dk", got[1]), ("dv", got[2])):
        near(t[0, pad:], want[name][0][pad:], want[name][1][pad:], name)
    near(got[0][0, pad:], want["dq"][0][pad:], want["dq"][1][pad:], "dq")


def test_what_is_seen_is_seen(device):
    """An infinity or NaN that a row does see reaches it, and only it and those behind."""
    n, d = 100, 32
    q, kv, _, do = make([n], [n], 1, d, 0, d, torch.float32, seed=12)
    kv[60, 0, d + 3] = math.inf
    args = (q[None].to(device), kv[None, ..., :d].to(device), kv[None, ..., d:].to(device), None)
    o, _ = rhizome_amd.latent_prefill(*args)
    assert bool(torch.isfinite(o[0, :60]).all()) and bool((o[0, 60:, 0, 3] == math.inf).all())
    assert bool(torch.isfinite(o[0, :, 0, :3]).all())
    kv[60, 0, d + 3], kv[60, 0, 2] = 0.0, math.nan
    o, lse = rhizome_amd.latent_prefill(q[None].to(device), kv[None, ..., :d].to(device), kv[None, ..., d:].to(device))
    assert bool(torch.isfinite(o[0, :60]).all()) and bool(torch.isnan(o[0, 60:]).all()) and bool(torch.isnan(lse[0, 60:]).all())


@pytest.mark.parametrize("dtype", DTYPES.values(), ids=DTYPES.keys())
def test_strides_and_alignment(device, dtype):
    """Views: heads before tokens, every other token, a slice of wider heads at an odd place."""
    H, d_n, d_r, d_v, n = 3, 64, 16, 32, 130
    q, kv, r, do = make([n], [n], H, d_n, d_r, d_v, dtype, seed=13)
    plain = (q[None].to(device), kv[None, ..., :d_n].contiguous().to(device), kv[None, ..., d_n:].contiguous().to(device),
             r[None].to(device))
    want = rhizome_amd.latent_prefill(*plain)
    grads = rhizome_amd.latent_prefill_backward(*plain, *want, do[None].to(device))

    def by_head(t):
        return t.transpose(1, 2).contiguous().transpose(1, 2)

    def spaced(t):
        wide = torch.full((t.shape[0], 2 * t.shape[1], *t.shape[2:]), 7.0, dtype=t.dtype, device=device)
        wide[:, ::2] = t
        return wide[:, ::2]

    def odd(t):
        wide = torch.full((*t.shape[:-1], t.shape[-1] + 5), 7.0, dtype=t.dtype, device=device)
        wide[..., 3:-2] = t
        return wide[..., 3:-2]

    for view in (by_head, spaced):
        got = rhizome_amd.latent_prefill(*[view(t) if t.dim() == 4 else t for t in plain])
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        again = rhizome_amd.latent_prefill_backward(*[view(t) if t.dim() == 4 else t for t in plain], *want, do[None].to(device))
        assert all(torch.equal(a, b) for a, b in zip(again, grads))
    got = rhizome_amd.latent_prefill(*[odd(t) for t in plain])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    again = rhizome_amd.latent_prefill_backward(*[odd(t) for t in plain], *want, do[None].to(device))
    assert all(torch.equal(a, b) for a, b in zip(again, grads))


@pytest.mark.parametrize("dtype", DTYPES.values(), ids=DTYPES.keys())
def test_expanded_inputs(device, dtype):
    """One head's keys and values for all heads, one token's for all tokens: strides of zero."""
    n, H, d = 150, 4, 64
    q, kv, _, do = (t[None].to(device) if t is not None else None for t in make([n], [n], H, d, 0, d, dtype, seed=21))
    for whole in (kv[:, :, :1], kv[:, :1]):
        k, v = (t.expand(1, n, H, d) for t in (whole[..., :d], whole[..., d:]))
        o, lse = rhizome_amd.latent_prefill(q, k, v)
        got = o, lse, *rhizome_amd.latent_prefill_backward(q, k, v, None, o, lse, do)[:3]
        k, v = k.contiguous(), v.contiguous()
        o, lse = rhizome_amd.latent_prefill(q, k, v)
        want = o, lse, *rhizome_amd.latent_prefill_backward(q, k, v, None, o, lse, do)[:3]
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", DTYPES.values(), ids=DTYPES.keys())
def test_one_token_of_a_long_tensor(device, dtype):
    """Its batch of one is 2^23 elements long, which no token's distance from the next is."""
    H, d, m = 2, 64, 50
    q, kv, _, _ = make([1], [m], H, d, 0, d, dtype, seed=18)
    long = torch.zeros(1, (1 << 23) // (H * d), H, d, dtype=dtype, device=device)
    long[:, 5:6] = q.to(device)
    k, v = (t[None].to(device) for t in (kv[..., :d], kv[..., d:]))
    got = rhizome_amd.latent_prefill(long[:, 5:6], k, v)
    want = rhizome_amd.latent_prefill(q[None].to(device), k, v)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype", DTYPES.values(), ids=DTYPES.keys())
def test_one_packed_token_far_from_a_next_one(device, dtype):
    """A sequence of one query, 2^23 elements from where the next would be, and of one key."""
    H, d = 2, 64
    q, kv, _, do = make([1], [1], H, d, 0, d, dtype, seed=19)
    long = torch.zeros(2, (1 << 23) // (H * d), H, d, dtype=dtype, device=device)
    long[1, 5] = q[0].to(device)
    far = long[1:, 5]
    assert far.shape == q.shape and far.stride(0) == 1 << 23
    k, v, cu = kv[..., :d].to(device), kv[..., d:].to(device), starts([1]).to(device)
    got = rhizome_amd.latent_prefill(far, k, v, cu_seqlens=cu)
    want = rhizome_amd.latent_prefill(q.to(device), k, v, cu_seqlens=cu)
    grads = [rhizome_amd.latent_prefill_backward(x, k, v, None, *want, do.to(device), cu_seqlens=cu) for x in (far, q.to(device))]
    turned = [rhizome_amd.rope(x, cu[:1], torch.ones(8, dtype=torch.float64, device=device)) for x in (far, q.to(device))]
    assert all(torch.equal(a, b) for a, b in zip((*got, *grads[0][:3], turned[0]), (*want, *grads[1][:3], turned[1])))



@pytest.mark.parametrize("dtype", DTYPES.values(), ids=DTYPES.keys())
def test_a_sequence_alone_and_in_a_pack(device, dtype):
    """Batch-invariance, bit for bit; rows outside every sequence are left as they were."""
    lens, H, d = [37, 150, 64], 2, 64
    q, kv, r, do = make(lens, lens, H, d, 32, d, dtype, seed=14)
    total, front = sum(lens), 10
    pad = lambda t: torch.cat([torch.full((front, *t.shape[1:]), math.nan, dtype=t.dtype), t,
                               torch.full((7, *t.shape[1:]), math.nan, dtype=t.dtype)]).to(device)
    cu = (starts(lens) + front).to(device)
    q2, kv2, r2, do2 = (pad(t) for t in (q, kv, r, do))
    args = (q2, kv2[..., :d], kv2[..., d:], r2)
    out = torch.full((front + total + 7, H, d), 5.0, dtype=dtype, device=device)
    o, lse = rhizome_amd.latent_prefill(*args, cu_seqlens=cu, out=out)
    grads = rhizome_amd.latent_prefill_backward(*args, o, lse, do2, cu_seqlens=cu)
    assert bool((o[:front] == 5.0).all()) and bool((o[front + total:] == 5.0).all())
    at = 0
    for n in lens:
        s = slice(at, at + n)
        one = [t.to(device)[None] for t in (q[s], kv[s, :, :d], kv[s, :, d:], r[s])]
        o1, l1 = rhizome_amd.latent_prefill(*one)
        g1 = rhizome_amd.latent_prefill_backward(*one, o1, l1, do[s].to(device)[None])
        there = slice(front + at, front + at + n)
        assert torch.equal(o[there], o1[0]) and torch.equal(lse[there], l1[0])
        for a, b in zip(grads, g1):
            assert torch.equal(a[there], b[0])
        at += n


def test_gradients_against_differences(device):
    """fp32, by central differences of a scalar of o and lse in 64 bits."""
    lens, H, d_n, d_r, d_v = [9, 5], 2, 8, 4, 8
    q, kv, r, do = make(lens, lens, H, d_n, d_r, d_v, torch.float32, seed=15)
    dl = torch.randn(sum(lens), H, generator=torch.Generator().manual_seed(4))
    dev = [t.to(device) for t in (q, kv, r, do, dl)]
    cu = starts(lens).to(device)
    args = (dev[0], dev[1][..., :d_n], dev[1][..., d_n:], dev[2])
    o, lse = rhizome_amd.latent_prefill(*args, cu_seqlens=cu, scale=0.4)
    dq, dk, dv, dr = rhizome_amd.latent_prefill_backward(*args, o, lse, dev[3], dlse=dev[4], cu_seqlens=cu, scale=0.4)

    def loss(q, kv, r):
        total, at = 0.0, 0
        for n in lens:
            s = slice(at, at + n)
            o, lse, _, _ = attend(q[s], kv[s, :, :d_n], kv[s, :, d_n:], r[s], 0.4, True, torch.float32)
            total += float((o * do[s].double()).sum() + (lse * dl[s].double()).sum())
            at += n
        return total

    leaves = [t.double() for t in (q, kv, r)]
    grads = (dq, torch.cat([dk, dv], -1), dr)
    gen = torch.Generator().manual_seed(6)
    for i, g in enumerate(grads):
        for at in torch.randint(0, leaves[i].numel(), (12,), generator=gen).tolist():
            h, save = 1e-5, leaves[i].view(-1)[at].item()
            leaves[i].view(-1)[at] = save + h
            up = loss(*leaves)
            leaves[i].view(-1)[at] = save - h
            down = loss(*leaves)
            leaves[i].view(-1)[at] = save
            diff = (up - down) / (2 * h)
            # differences: h^2 of a third derivative of order 1, rounding 1e-15 / h; fp32: a few dozen roundings of terms of order 1
            assert abs(float(g.reshape(-1)[at]) - diff) < 2e-5 * (1 + abs(diff)), (i, at)


@pytest.mark.parametrize("dtype", DTYPES.values(), ids=DTYPES.keys())
def test_graph_replays(device, dtype):
    """Forward and backward in one graph, replayed with other inputs and eager work between."""
    n, H, d = 200, 2, 64
    q, kv, r, do = (t[None].to(device) for t in make([n], [n], H, d, 32, d, dtype, seed=16))
    args = (q, kv[..., :d], kv[..., d:], r)
    o, lse = rhizome_amd.latent_prefill(*args)
    rhizome_amd.latent_prefill_backward(*args, o, lse, do)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, lse = rhizome_amd.latent_prefill(*args)
        grads = rhizome_amd.latent_prefill_backward(*args, o, lse, do)
    for i in range(3):
        new = make([n], [n], H, d, 32, d, dtype, seed=20 + i)
        for t, x in zip((q, kv, r, do), new):
            t.copy_(x[None])
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (o, lse, *grads)]
        eager = rhizome_amd.latent_prefill(*args)
        eager = (*eager, *rhizome_amd.latent_prefill_backward(*args, *eager, do))
        assert all(torch.equal(a, b) for a, b in zip(got, eager)), f"replay {i}"


def test_long_rows(device):
    """A few thousand keys, against 64 bits at some of the rows."""
    n, H, dtype = 3500, 1, torch.bfloat16
    q, kv, r, do = make([n], [n], H, 128, 64, 128, dtype, seed=17)
    args = [t[None].to(device) for t in (q, kv[..., :128], kv[..., 128:], r)]
    o, lse = rhizome_amd.latent_prefill(*args)
    want_o, want_l, tol_o, tol_l = attend(q, kv[..., :128], kv[..., 128:], r, 192 ** -0.5, True, dtype)
    near(o[0], want_o, tol_o, "o")
    near(lse[0], want_l, tol_l, "lse")
    got = rhizome_amd.latent_prefill_backward(*args, o, lse, do[None].to(device))
    want = attend_backward(q, kv[..., :128], kv[..., 128:], r, do, None, 192 ** -0.5, True, dtype)
    for name, t in zip(("dq", "dk", "dv", "dr"), got):
        near(t[0], *want[name], name)
