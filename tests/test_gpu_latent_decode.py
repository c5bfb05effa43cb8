"""The paged latents' decode against the formulas in 64 bits (bounds as
attn_cases.py derives them), and a run of rope, append and decode against the
expanded prefill."""
import math
from ctypes import byref, c_size_t

import pytest
import torch

import rhizome_amd
from rhizome_amd import _abi
from attn_cases import DTYPES, W, half_step, near, normal, scores, weights

pytestmark = pytest.mark.gpu


def pages(lens, page, gen, spare=3):
    need = [-(-max(n, 0) // page) for n in lens]
    order = torch.randperm(sum(need) + spare, generator=gen).tolist()
    table, at = torch.full((len(lens), max(max(need), 1)), -7, dtype=torch.int32), 0
    for i, n in enumerate(need):
        table[i, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    return table, sum(need) + spare


def make(lens, steps, H, d_c, d_r, page, dtype, seed=0, std=1.0):
    gen = torch.Generator().manual_seed(seed)
    table, n = pages(lens, page, gen)
    cache = normal((n, page, d_c + d_r), gen, dtype)
    return normal((len(lens), steps, H, d_c + d_r), gen, dtype, std), cache, table, torch.tensor(lens, dtype=torch.int32)


def exact(q, cache, table, lens, d_c, scale, dtype, page):
    """o, lse and their bounds of every sequence."""
    B, steps, H, D = q.shape
    out = [torch.zeros(B, steps, H, d_c, dtype=torch.float64), torch.full((B, steps, H), -math.inf, dtype=torch.float64)]
    tol = [torch.zeros_like(out[0]), torch.zeros(B, steps, H, dtype=torch.float64)]
    u = half_step(dtype)
    for b, n in enumerate(lens.tolist()):
        at = torch.arange(min(max(n, 0), table.shape[1] * page))
        page_of = table[b][at // page].long()
        ok = (page_of >= 0) & (page_of < cache.shape[0])
        rows = cache.view(-1, D)[(page_of.clamp(0, cache.shape[0] - 1) * page + at % page)]
        if len(at) == 0:
            continue
        keys = rows.unsqueeze(1).expand(-1, H, -1)
        s, size, k = scores(q[b], keys, None, scale)
        seen = (at[None] <= n - steps + torch.arange(steps)[:, None]) & ok[None]
        s, size = (torch.where(seen, t, torch.zeros_like(t)) for t in (s, size))
        p, lse, rel = weights(s, size, seen, D)
        v = torch.where(ok[:, None], rows[:, :d_c].double(), 0.0)
        v = torch.where(seen.any(0)[:, None], v, 0.0)  # rows that nobody sees may hold anything
        o, around = p @ v, p @ v.abs()
        out[0][b], out[1][b] = o.transpose(0, 1), lse.T
        rounded = u if dtype == torch.bfloat16 else 0.0
        t = u * o.abs() + (rel + rounded + (len(at) + 140) * W) * around * (1 + 2 * u) + 1e-37
        tol[0][b] = t.transpose(0, 1)
        tol[1][b] = (rel[..., 0] + 4 * W * lse.abs().masked_fill(torch.isinf(lse), 0.0)).T
    return out, tol


def run(q, cache, table, lens, d_c, scale, device, **kw):
    o, lse = rhizome_amd.latent_decode(*(t.to(device) for t in (q, cache, table, lens)), d_c=d_c, scale=scale, **kw)
    torch.cuda.synchronize()
    return o, lse


def check(lens, steps, H, d_c, d_r, page, dtype, device, seed=0, scale=None, std=1.0):
    scale = (d_c + d_r) ** -0.5 if scale is None else scale
    args = make(lens, steps, H, d_c, d_r, page, dtype, seed, std)
    got = run(*args, d_c, scale, device)
    want, tol = exact(*args, d_c, scale, dtype, page)
    near(got[0], want[0], tol[0], "o")
    near(got[1], want[1], tol[1], "lse")


both = pytest.mark.parametrize("dtype", DTYPES.values(), ids=DTYPES.keys())


@both
@pytest.mark.parametrize("n", [0, 1, 2, 31, 32, 33, 63, 64, 65, 95, 255, 256, 257, 300, 513, 1000])
def test_lengths(device, dtype, n):
    """None, one, and around tiles and splits."""
    check([n], 1, 2, 128, 16, 16, dtype, device, seed=n)


@both
@pytest.mark.parametrize("steps,H", [(1, 1), (1, 16), (2, 16), (1, 33), (4, 16), (5, 13), (1, 64), (3, 43), (7, 20), (64, 2),
                                     (1, 128), (64, 5)])
def test_rows(device, dtype, steps, H):
    """Numbers of rows around 32, 64, 128 and more, and rows of different reach."""
    check([300, 3, 70], steps, H, 128, 32, 64, dtype, device, seed=H)


@both
@pytest.mark.parametrize("d_c,d_r", [(512, 64), (256, 32), (512, 0), (384, 64), (136, 8), (64, 64), (1, 0), (7, 3), (130, 5),
                                     (511, 63), (256, 1), (200, 40)])
def test_widths(device, dtype, d_c, d_r):
    for steps, H in ((1, 8), (2, 40)):
        check([130, 300], steps, H, d_c, d_r, 64, dtype, device, seed=d_c)


@both
@pytest.mark.parametrize("d_c,d_r", [(130, 6), (100, 28), (1, 7), (497, 15), (251, 5), (12, 4)])
def test_rows_of_whole_chunks_with_latents_that_are_not(device, dtype, d_c, d_r):
    for steps, H in ((1, 8), (2, 16), (3, 16), (2, 40)):
        check([130, 300], steps, H, d_c, d_r, 64, dtype, device, seed=d_c)


@both
@pytest.mark.parametrize("page", [1, 3, 16, 31, 100, 1000])
def test_pages(device, dtype, page):
    """Pages that end inside a tile, of one row, and longer than a split."""
    check([257, 64, 1, 600], 2, 4, 128, 16, page, dtype, device, seed=page)


@both
@pytest.mark.parametrize("H", [2, 20])
def test_empty_sequences_and_pages_of_one_row(device, dtype, H):
    """The first table entry of all has nothing before it to be looked up."""
    check([0, 3, 0], 1, H, 128, 16, 1, dtype, device)


@both
def test_long_contexts(device, dtype):
    """More than 128 splits' worth of rows, and a table of rows refilled on the way."""
    check([40000, 2500], 1, 2, 64, 0, 64, dtype, device, seed=1)
    check([140000], 1, 1, 32, 0, 128, dtype, device, seed=2)


@both
def test_sharp_weights(device, dtype):
    check([700, 90], 3, 16, 256, 64, 32, dtype, device, std=8.0, seed=3)


@both
def test_batch_invariance(device, dtype):
    lens = [700, 33, 0, 2049, 5]
    q, cache, table, n = make(lens, 2, 8, 256, 64, 16, dtype, seed=4)
    o, lse = run(q, cache, table, n, 256, 0.05, device)
    for b in range(len(lens)):
        wide = torch.zeros(1, table.shape[1] + 3000, dtype=torch.int32)  # a longer table, as another batch may have
        wide[0, :table.shape[1]] = table[b]
        one = run(q[b:b + 1], cache, wide, n[b:b + 1], 256, 0.05, device)
        assert torch.equal(one[0][0], o[b]) and torch.equal(one[1][0], lse[b])


@both
def test_pages_outside_the_cache(device, dtype):
    """Hold no keys, and nothing is read there."""
    lens, page = [200, 90, 64], 16
    q, cache, table, n = make(lens, 2, 8, 128, 16, page, dtype, seed=5)
    table[0, 2], table[0, 7], table[1, 0], table[1, 5] = -1, cache.shape[0], 2 ** 31 - 1, -2 ** 31
    table[2, :4] = -1  # none of its keys is there
    got = run(q, cache, table, n, 128, 0.1, device)
    want, tol = exact(q, cache, table, n, 128, 0.1, dtype, page)
    near(got[0], want[0], tol[0], "o")
    near(got[1], want[1], tol[1], "lse")
    assert not bool(got[0][2].any()) and bool((got[1][2] == -math.inf).all())


@both
def test_lengths_beyond_the_table(device, dtype):
    """Positions beyond the table hold no keys; negative lengths are none."""
    q, cache, table, _ = make([64, 64, 64], 3, 4, 128, 16, 16, dtype, seed=6)
    n = torch.tensor([1000, -5, 2 ** 31 - 1], dtype=torch.int32)
    got = run(q, cache, table, n, 128, 0.1, device)
    want, tol = exact(q, cache, table, n, 128, 0.1, dtype, 16)
    near(got[0], want[0], tol[0], "o")
    near(got[1], want[1], tol[1], "lse")
    assert not bool(got[0][1].any())


@both
@pytest.mark.parametrize("value", [math.nan, math.inf], ids=["nan", "inf"])
def test_what_is_not_seen_has_no_part(device, dtype, value):
    """Rows of the cache behind the length, rows that only later steps see, other pages, row 0."""
    lens, steps, page = [45, 300], 4, 32
    q, cache, table, n = make(lens, steps, 8, 256, 64, page, dtype, seed=7)
    used = set(table[0, :2].tolist()) | set(table[1, :10].tolist())
    for i in range(cache.shape[0]):
        if i not in used:
            cache[i] = value
    cache[table[0, 1], 45 - 32:] = value
    cache[table[1, 9], 300 - 288:] = value
    clean = [t.clone() for t in (q, cache, table, n)]
    got = run(q, cache, table, n, 256, 0.06, device)
    zero = torch.where(torch.isfinite(cache), cache, torch.zeros_like(cache))
    want, tol = exact(q, zero, table, n, 256, 0.06, dtype, page)
    near(got[0], want[0], tol[0], "o")
    near(got[1], want[1], tol[1], "lse")
    # the last position's row: the last step alone sees it
    clean[1][table[0, 1], 44 - 32, 5] = value
    got = run(*clean, 256, 0.06, device)
    near(got[0][0, :3], want[0][0, :3], tol[0][0, :3], "o of the earlier steps")
    assert not bool(torch.isfinite(got[1][0, 3]).any()) or value == math.inf
    assert not bool(torch.isfinite(got[0][0, 3, :, 5]).any())
    # and pages outside the cache while row 0 holds anything
    bad = [t.clone() for t in (q, zero, table, n)]
    bad[1][0] = torch.where(torch.tensor(0 in used), bad[1][0], torch.full_like(bad[1][0], value))
    bad[2][1, 3] = -1
    got = run(*bad, 256, 0.06, device)
    if 0 not in used:
        want, tol = exact(q, zero, bad[2], n, 256, 0.06, dtype, page)
        near(got[0], want[0], tol[0], "o beside a page that is not there")


@both
def test_caller_owned_buffers_and_replays(device, dtype):
    """One workspace and output kept by the caller, in a graph whose lengths and tables change between replays."""
    lens = [500, 20, 1000]
    q, cache, table, n = (t.to(device) for t in make(lens, 1, 16, 256, 64, 64, dtype, seed=8))
    out = torch.empty(3, 1, 16, 256, dtype=dtype, device=device)
    size, args = c_size_t(), _abi.LatentDecodeArgs()
    args.batch, args.steps, args.heads, args.d_c, args.d_r, args.scale = 3, 1, 16, 256, 64, 0.06
    args.page_size, args.num_pages, args.max_pages, args.dtype = 64, cache.shape[0], table.shape[1], _abi.F32
    _abi.check(_abi.lib().rhz_latent_decode_workspace_size(byref(args), byref(size)))
    ws = torch.empty(size.value, dtype=torch.uint8, device=device)
    rhizome_amd.latent_decode(q, cache, table, n, d_c=256, scale=0.06, out=out, workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, lse = rhizome_amd.latent_decode(q, cache, table, n, d_c=256, scale=0.06, out=out, workspace=ws)
    for i, new in enumerate(([500, 20, 1000], [1, 0, 700], [513, 256, 64])):
        n.copy_(torch.tensor(new, dtype=torch.int32))
        q.copy_(normal(q.shape, torch.Generator().manual_seed(i), dtype))
        out.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone(), lse.clone()
        want = rhizome_amd.latent_decode(q, cache, table, n, d_c=256, scale=0.06)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), f"replay {i}"


def test_cache_beyond_32_bits(device):
    """Rows of a cache of 9 GB, at its end."""
    page, D = 64, 576
    pages_n = (9 << 30) // (page * D * 2)
    cache = torch.empty(pages_n, page, D, dtype=torch.bfloat16, device=device)
    at = [pages_n - 1, 3, pages_n // 2]
    gen = torch.Generator().manual_seed(9)
    rows = normal((3, page, D), gen, torch.bfloat16)
    for i, p in enumerate(at):
        cache[p] = rows[i].to(device)
    q = normal((1, 1, 16, D), gen, torch.bfloat16)
    table, n = torch.tensor([at], dtype=torch.int32), torch.tensor([180], dtype=torch.int32)
    got = rhizome_amd.latent_decode(q.to(device), cache, table.to(device), n.to(device), d_c=512, scale=0.05)
    want, tol = exact(q, rows, torch.tensor([[0, 1, 2]], dtype=torch.int32), n, 512, 0.05, torch.bfloat16, page)
    near(got[0], want[0], tol[0], "o")
    new = normal((1, 2, 512), gen, torch.bfloat16).to(device)
    key = normal((1, 2, 64), gen, torch.bfloat16).to(device)
    rhizome_amd.latent_append(new, key, cache, table.to(device), torch.tensor([64], dtype=torch.int32, device=device))
    assert torch.equal(cache[at[0], 62:, :512], new[0]) and torch.equal(cache[at[0], 62:, 512:], key[0])


@both
def test_prompt_then_steps_against_the_expanded_form(device, dtype):
    """The operators as a server runs them: a prompt's tokens enter the cache in
    two calls, queries are turned in place, and the absorbed decode of the last
    positions gives what the expanded prefill gives for them."""
    gen = torch.Generator().manual_seed(10)
    B, H, d_n, d_c, d_r, page, lens = 3, 4, 32, 128, 16, 16, [70, 33, 130]
    steps, total, width = 3, sum(lens), max(lens)
    c, r = normal((total, d_c), gen, dtype), normal((total, d_r), gen, dtype)
    q_n, q_r = normal((total, H, d_n), gen, dtype), normal((total, H, d_r), gen, dtype)
    w = (torch.randn(H, d_n, d_c, generator=gen) * d_c ** -0.5)  # keys' projection
    norm = torch.rand(d_c, generator=gen) + 0.5
    freq, mag = rhizome_amd.rope_frequencies(d_r, theta=100.0, scaling="by_parts", factor=4.0, trained_length=64, device=device)
    table, n_pages = pages(lens, page, gen)
    cache = torch.full((n_pages, page, d_c + d_r), math.nan, dtype=dtype, device=device)
    table = table.to(device)
    pos = torch.cat([torch.arange(n) for n in lens]).to(torch.int32).to(device)
    cd, rd = c.to(device), r.to(device)
    first = [n - steps for n in lens]
    begin = [sum(lens[:i]) for i in range(B)]
    prompt = torch.cat([torch.arange(b, b + n) for b, n in zip(begin, first)]).to(device)
    cu = torch.tensor([0, *torch.tensor(first).cumsum(0).tolist()], dtype=torch.int32, device=device)
    kw = dict(frequencies=freq, magnitude=mag, norm_scale=norm.to(device))
    rhizome_amd.latent_append(cd[prompt], rd[prompt], cache, table, torch.tensor(first, dtype=torch.int32, device=device),
                              cu_seqlens=cu, **kw)
    last = torch.stack([torch.arange(b + n - steps, b + n) for b, n in zip(begin, lens)]).to(device)
    lengths = torch.tensor(lens, dtype=torch.int32, device=device)
    rhizome_amd.latent_append(cd[last], rd[last], cache, table, lengths, **kw)
    qr = q_r.to(device)
    rhizome_amd.rope(qr, pos, freq, magnitude=mag, out=qr)
    q_abs = torch.einsum("bshd,hdc->bshc", q_n.to(device)[last].float(), w.to(device)).to(dtype)
    scale = (d_n + d_r) ** -0.5
    o, lse = rhizome_amd.latent_decode(torch.cat([q_abs, qr[last]], -1), cache, table, lengths, d_c=d_c, scale=scale)
    # the same positions from the cache's own rows, keys and values being the latents of 128: q absorbed, expanded form
    flat = cache.view(-1, d_c + d_r)
    at = torch.cat([table[b].long()[torch.arange(n, device=device) // page] * page + torch.arange(n, device=device) % page
                    for b, n in enumerate(lens)])
    rows = flat[at]
    assert bool(torch.isfinite(rows).all())
    keys = rows[:, None, :d_c].expand(-1, H, -1).contiguous()
    cu_q = torch.arange(0, B * steps + 1, steps, dtype=torch.int32, device=device)
    cu_k = torch.tensor([0, *torch.tensor(lens).cumsum(0).tolist()], dtype=torch.int32, device=device)
    q_all = torch.cat([q_abs, qr[last]], -1).flatten(0, 1)
    o2, lse2 = rhizome_amd.latent_prefill(q_all, keys, keys, rows[:, d_c:].contiguous(), scale=scale, cu_seqlens=cu_q,
                                          cu_seqlens_k=cu_k)
    # both have the bound of `exact`; twice it between them
    want, tol = exact(torch.cat([q_abs, qr[last]], -1).cpu(), cache.cpu().nan_to_num(0.0), table.cpu(), lengths.cpu(), d_c,
                      scale, dtype, page)
    near(o, want[0], tol[0], "decode")
    near(o2.view_as(o), want[0], tol[0], "prefill")
    near(lse, want[1], tol[1], "lse")
    near(lse2.view_as(lse), want[1], tol[1], "lse of the prefill")
    assert width == 130
