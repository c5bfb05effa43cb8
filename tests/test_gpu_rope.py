"""Rotary positions and the paged cache's writer against the formulas in 64 bits.

A turned value is a sum of two products by a cosine and a sine, each within 4
half steps (2^-24) of the true one (its argument is reduced in 64 bits and
rounded once, the function is good to 2 of them, the magnitude is one more),
with three roundings more, and one of the tensors' type.
"""
import math

import pytest
import torch

import rhizome_amd
from attn_cases import DTYPES, W, half_step, near, normal
from test_gpu_latent_decode import pages

pytestmark = pytest.mark.gpu
both = pytest.mark.parametrize("dtype", DTYPES.values(), ids=DTYPES.keys())


def turned(x, positions, freq, mag, inter, inverse=False):
    """The pairs of x's last dimension turned, and the sums of their terms' magnitudes."""
    x = x.double()
    angle = 2 * math.pi * torch.remainder(positions.double()[..., None, None] * freq, 1.0)
    if inverse:
        angle = -angle
    cos, sin = mag * torch.cos(angle), mag * torch.sin(angle)
    a, b = (x[..., 0::2], x[..., 1::2]) if inter else x.chunk(2, -1)
    y, size = (a * cos - b * sin, a * sin + b * cos), ((a * cos).abs() + (b * sin).abs(), (a * sin).abs() + (b * cos).abs())
    big = mag * (a.abs() + b.abs())  # an angle's error counts whole
    join = (lambda p: torch.stack(p, -1).flatten(-2)) if inter else (lambda p: torch.cat(p, -1))
    return join(y), join(size), join((big, big))


def bound(y, size, big, dtype):
    return half_step(dtype) * y.abs() + 8 * W * (size + big) + 1e-37


def check(shape, rot, offset, dtype, device, inter=False, inverse=False, mag=1.0, positions=None, seed=0):
    gen = torch.Generator().manual_seed(seed)
    x = normal(shape, gen, dtype)
    lead = shape[:-2]
    pos = positions if positions is not None else torch.randint(0, 5000, lead, generator=gen)
    freq, _ = rhizome_amd.rope_frequencies(rot, device=device)
    y = rhizome_amd.rope(x.to(device), pos.to(torch.int32).to(device), freq, offset=offset, interleaved=inter, magnitude=mag,
                         inverse=inverse).cpu()
    end = offset + rot
    assert torch.equal(y[..., :offset], x[..., :offset]) and torch.equal(y[..., end:], x[..., end:])
    want = turned(x[..., offset:end], pos, freq.cpu(), mag, inter, inverse)
    near(y[..., offset:end], want[0], bound(*want, dtype), "rope")


@both
@pytest.mark.parametrize("inter", [False, True], ids=["halves", "neighbours"])
@pytest.mark.parametrize("shape,rot,offset", [
    ((1, 1, 2), 2, 0), ((3, 2, 64), 64, 0), ((5, 16, 192), 64, 128), ((2, 7, 3, 96), 32, 64), ((4, 5, 40), 16, 8),
    ((300, 1, 64), 64, 0), ((33, 3, 21), 6, 7), ((2, 2, 130), 130, 0), ((3, 1, 1024), 1024, 0), ((1000, 2, 32), 16, 16),
    ((0, 2, 32), 16, 0), ((6, 40, 128), 128, 0), ((17, 2, 50), 20, 30)])
def test_shapes(device, dtype, inter, shape, rot, offset):
    for inverse in (False, True):
        check(shape, rot, offset, dtype, device, inter, inverse, mag=1.25, seed=rot)


@both
def test_far_positions(device, dtype):
    """Positions up to the largest of 32 bits and below zero."""
    pos = torch.tensor([0, 1, 131071, 10_000_019, 2 ** 31 - 1, -1, -100_003, -2 ** 31])
    check((8, 4, 64), 64, 0, dtype, device, positions=pos)
    check((8, 4, 64), 32, 16, dtype, device, inter=True, positions=pos)


@both
@pytest.mark.parametrize("inter", [False, True], ids=["halves", "neighbours"])
def test_in_place_on_views(device, dtype, inter):
    """A slice of wider heads, heads before tokens, at an odd place: what lies beside is left alone."""
    gen = torch.Generator().manual_seed(3)
    freq, mag = rhizome_amd.rope_frequencies(32, scaling="linear", factor=4.0, device=device)
    x = normal((9, 4, 80), gen, dtype).to(device)
    pos = torch.arange(9, dtype=torch.int32, device=device) * 17
    for offset in (48, 45):
        want = rhizome_amd.rope(x, pos, freq, offset=offset, interleaved=inter)
        y = x.clone()
        got = rhizome_amd.rope(y, pos, freq, offset=offset, interleaved=inter, out=y)
        assert got is y and torch.equal(y, want)
        y = x.clone()
        part = y[..., offset:offset + 32]
        rhizome_amd.rope(part, pos, freq, interleaved=inter, out=part)
        assert torch.equal(y, want)
        y = x.transpose(0, 1).contiguous().transpose(0, 1)
        rhizome_amd.rope(y, pos, freq, offset=offset, interleaved=inter, out=y)
        assert torch.equal(y, want)
        back = rhizome_amd.rope(want, pos, freq, offset=offset, interleaved=inter, inverse=True)
        near(back, x.double().cpu(), 3 * half_step(dtype) * x[..., :].double().abs().cpu().amax() + 32 * W, "back")
    # one key for all heads, and one token for all: strides of zero in the input
    row = normal((1, 1, 32), gen, dtype).to(device).expand(9, 4, 32)
    got = rhizome_amd.rope(row, pos, freq, interleaved=inter)
    assert torch.equal(got, rhizome_amd.rope(row.contiguous(), pos, freq, interleaved=inter))


def test_adjoint(device):
    """<rope(x), y> = <x, rope^T(y)>, and differences along each input."""
    gen = torch.Generator().manual_seed(4)
    x, y = (normal((6, 3, 24), gen, torch.float32) for _ in range(2))
    pos = torch.arange(6, dtype=torch.int32, device=device) * 5
    freq, _ = rhizome_amd.rope_frequencies(16, device=device)
    kw = dict(offset=4, magnitude=1.3)
    fx = rhizome_amd.rope(x.to(device), pos, freq, **kw).double().cpu()
    gy = rhizome_amd.rope(y.to(device), pos, freq, inverse=True, **kw).double().cpu()
    terms = (fx.abs() * y.double().abs()).sum() + (x.double().abs() * gy.abs()).sum()
    assert abs(float((fx * y.double()).sum() - (x.double() * gy).sum())) <= 16 * W * float(terms)
    # the operator is linear: a difference along one input is its column
    for at in (0, 5, 13, 40, 71):
        e = torch.zeros_like(x).view(-1)
        e[at] = 1.0
        column = rhizome_amd.rope(e.view_as(x).to(device), pos, freq, **kw).double().cpu()
        assert abs(float((column * y.double()).sum() - gy.view(-1)[at])) <= 16 * W * float((column.abs() * y.double().abs()).sum() + 1e-9)


@both
@pytest.mark.parametrize("d_c,d_r,page,norm,turn", [(512, 64, 64, True, True), (512, 64, 16, False, True), (128, 0, 3, True, False),
                                                    (7, 5, 1, True, False), (130, 6, 10, True, True), (1, 2, 4, False, True),
                                                    (4096, 8, 4, True, True), (256, 1024, 2, False, True), (520, 32, 7, True, True),
                                                    (3001, 0, 5, True, False)])
def test_append(device, dtype, d_c, d_r, page, norm, turn):
    """Against the formulas; rows that no token goes to stay as they were."""
    gen = torch.Generator().manual_seed(d_c)
    lens, news = [70, 5, 1, 40, 33, 0], [70, 2, 1, 0, 20, 0]
    table, n_pages = pages(lens, page, gen)
    D, total = d_c + d_r, sum(news)
    both_t = normal((total, D + 3), gen, dtype, 2.0).to(device)  # one projection's output, and more behind it
    cache = normal((n_pages, page, D), gen, dtype)
    scale = torch.rand(d_c, generator=gen) + 0.5
    freq, mag = rhizome_amd.rope_frequencies(d_r, device=device) if turn else (None, 1.0)
    mag = 1.5 if turn else 1.0
    cu = torch.tensor([0, *torch.tensor(news).cumsum(0).tolist()], dtype=torch.int32)
    for inter in (False, True):
        got = rhizome_amd.latent_append(
            both_t[:, :d_c], both_t[:, d_c:D] if d_r else None, cache.to(device), table.to(device),
            torch.tensor(lens, dtype=torch.int32, device=device), cu_seqlens=cu.to(device), frequencies=freq, magnitude=mag,
            interleaved=inter, norm_scale=scale.to(device) if norm else None).cpu()
        want, tol, at = cache.double(), torch.zeros(n_pages, page, D, dtype=torch.float64), 0
        for b, (n, k) in enumerate(zip(lens, news)):
            x = both_t[at:at + k, :d_c].double().cpu()
            at += k
            pos = torch.arange(n - k, n)
            where = (table[b].long()[pos // page], pos % page)
            t = torch.zeros_like(x)
            if norm:
                x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * scale.double()
                # the sum of squares: at most 4096 / 64 terms a lane and 6 more levels, halved by the root; four roundings
                t = (half_step(dtype) + 64 * W) * x.abs()
            want[where[0], where[1], :d_c], tol[where[0], where[1], :d_c] = x, t
            if d_r:
                r = both_t[at - k:at, d_c:D].double().cpu()
                t = torch.zeros_like(r)
                if turn:
                    y = turned(r[:, None], pos, freq.cpu(), mag, inter)
                    r, t = y[0][:, 0], bound(*y, dtype)[:, 0]
                want[where[0], where[1], d_c:], tol[where[0], where[1], d_c:] = r, t
        near(got, want, tol, "cache")


@both
def test_append_leaves_out(device, dtype):
    """Tokens without a place: negative positions, beyond the table, pages outside the cache, rows outside every sequence."""
    page, D = 4, 24
    cache = torch.full((3, page, D), 9.0, dtype=dtype, device=device)
    table = torch.tensor([[2, 0], [1, -1], [3, 7]], dtype=torch.int32, device=device)
    lens = torch.tensor([2, 7, 3], dtype=torch.int32, device=device)
    new = normal((3, 4, D), torch.Generator().manual_seed(1), dtype).to(device)
    rhizome_amd.latent_append(new[..., :16], new[..., 16:], cache, table, lens)
    want = torch.full((3, page, D), 9.0, dtype=dtype, device=device)
    want[2, 0], want[2, 1] = new[0, 2], new[0, 3]  # positions -2, -1, 0, 1
    want[1, 3] = new[1, 0]  # positions 3 .. 6: 4 and on are on page -1
    assert torch.equal(cache, want)
    lens = torch.tensor([12, 2 ** 31 - 1, -3], dtype=torch.int32, device=device)
    rhizome_amd.latent_append(new[..., :16], new[..., 16:], cache, table, lens)
    assert torch.equal(cache, want)
    cu = torch.tensor([3, 3, 5, 5], dtype=torch.int32, device=device)
    flat = new.view(12, D)
    rhizome_amd.latent_append(flat[:, :16], flat[:, 16:], cache, table, torch.tensor([1, 2, 0], dtype=torch.int32, device=device),
                              cu_seqlens=cu)
    want[1, 0], want[1, 1] = flat[3], flat[4]
    assert torch.equal(cache, want)
    rhizome_amd.latent_append(flat[:0, :16], flat[:0, 16:], cache, table, lens, cu_seqlens=torch.zeros_like(cu))
    assert torch.equal(cache, want)


def test_append_to_many_sequences(device):
    """One token each for more sequences than a wave has lanes."""
    n, page, D = 1000, 8, 40
    gen = torch.Generator().manual_seed(2)
    lens = torch.randint(1, 30, (n,), generator=gen)
    table, n_pages = pages(lens.tolist(), page, gen)
    new = normal((n, D), gen, torch.float32).to(device)
    cache = torch.zeros(n_pages, page, D, device=device)
    cu = torch.arange(n + 1, dtype=torch.int32, device=device)
    rhizome_amd.latent_append(new[:, :32], new[:, 32:], cache, table.to(device), lens.to(torch.int32).to(device), cu_seqlens=cu)
    pos = lens - 1
    assert torch.equal(cache[table[torch.arange(n), pos // page].long().to(device), (pos % page).to(device)], new)
    assert int((cache.abs().sum(-1) > 0).sum()) == n


@both
def test_expanded_tokens(device, dtype):
    """One token's heads turned to every position; an output of rows that share memory is refused."""
    n, H, d = 33, 4, 64
    freq = rhizome_amd.rope_frequencies(d, device=device)[0]
    pos = torch.arange(n, dtype=torch.int32, device=device)
    x = normal((1, H, d), torch.Generator().manual_seed(3), dtype).to(device)
    got = rhizome_amd.rope(x.expand(n, H, d), pos, freq, out=torch.empty(n, H, d, dtype=dtype, device=device))
    assert torch.equal(got, rhizome_amd.rope(x.expand(n, H, d).contiguous(), pos, freq))
    with pytest.raises(RuntimeError, match="overlap"):
        rhizome_amd.rope(got, pos, freq, out=x.clone().expand(n, H, d))
