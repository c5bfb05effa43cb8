"""Layer norm, its backward pass and RMSNorm's against torch in 64 bits on the CPU.

Tolerances of the 2-norm, set before the first run: fp32 outputs 2e-6 (a dozen
operations of half a step, 2^-24, on each value, with sums of up to 8192 terms
taken over lanes and waves: some 30 roundings); bf16 outputs half a step, 2^-8,
more than that.  A weight gradient sums over the rows, with cancellation: its
error is held against the norm of the sum of magnitudes.
"""
import pytest
import torch

import rhizome_amd

pytestmark = pytest.mark.gpu
F32_TOL, BF16_TOL = 2e-6, 2.0 ** -8 + 2e-6
DTYPES = [torch.float32, torch.bfloat16]


def make(rows, dim, dtype, seed=0, mean=0.5):
    gen = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, dim, generator=gen) + mean).to(dtype)
    dy = torch.randn(rows, dim, generator=gen).to(dtype)
    return x, dy, torch.randn(dim, generator=gen) * 0.3 + 1.0, torch.randn(dim, generator=gen)


def formulas(x, dy, w, b, eps, centre):
    """y, dx, dw, db in 64 bits, and the sums of magnitudes behind dw and db."""
    x, w, b = (t.double().requires_grad_(True) for t in (x, w, b))
    xc = x - x.mean(-1, keepdim=True) if centre else x
    xh = xc / torch.sqrt((xc * xc).mean(-1, keepdim=True) + eps)
    y = xh * w + b
    dy = dy.double()
    dx, dw, db = torch.autograd.grad((y * dy).sum(), (x, w, b))
    return y.detach(), dx, dw, db, (dy * xh).abs().sum(0).detach(), dy.abs().sum(0)


def near(got, want, tol, scale=None, what=""):
    scale = want if scale is None else scale
    assert got.shape == want.shape
    assert bool(torch.isfinite(got).all()), what
    err, norm = float((got.double().cpu() - want).norm()), float(scale.norm())
    assert err <= tol * norm + 1e-30, f"{what}: {err / max(norm, 1e-300):.3g}, tolerance {tol:.3g}"


def run(x, dy, w, b, device, centre=True, eps=1e-5):
    x, dy, w, b = (t.to(device) for t in (x, dy, w, b))
    if centre:
        out = (rhizome_amd.layernorm(x, w, b, eps), *rhizome_amd.layernorm_backward(dy, x, w, eps))
    else:
        out = (rhizome_amd.rmsnorm_heads(x, w, eps) if x.shape[-1] <= 1024 else None,
               *rhizome_amd.rmsnorm_heads_backward(dy, x, w, eps))
    torch.cuda.synchronize()
    return out


# every way of laying a row over threads: lanes of 16 bytes, a wave with 2, 4, 8
# and 16 vectors, a block; with and without whole vectors
DIMS = [1, 2, 3, 8, 31, 32, 64, 72, 128, 130, 256, 257, 384, 512, 1000, 1001, 1024, 1500, 2048, 2049, 4096, 5000, 8191,
        8192]


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("centre", [True, False], ids=["layer", "rms"])
@pytest.mark.parametrize("dim", DIMS)
def test_widths(device, dtype, centre, dim):
    if centre and dim == 1:
        pytest.skip("one value's distance from its mean is zero: see test_degenerate_rows")
    for rows in (1, 5, 67):
        x, dy, w, b = make(rows, dim, dtype, seed=dim + rows)
        y, dx, dw, db, mw, mb = formulas(x, dy, w, b, 1e-5, centre)
        got = run(x, dy, w, b, device, centre)
        tol = F32_TOL if dtype == torch.float32 else BF16_TOL
        if centre:
            near(got[0], y, tol, what="y")
            near(got[3], db, F32_TOL, mb, "db")
        # In rows of a few values dx is what is left of terms that cancel: of one
        # value, RMSNorm's dx = r t (1 - x^2 r^2) with 1 - x^2 r^2 = eps r^2, some
        # 1e-5, whose two terms of size r t are rounded by 2^-24 each: an error of
        # 2^-24 / 1e-5 = 6e-3 of dx, 2^-24 of the terms.  The error is held against
        # the terms r t there.
        spread = x.double() - x.double().mean(-1, keepdim=True) if centre else x.double()
        terms = dy.double() * w.double() / torch.sqrt((spread * spread).mean(-1, keepdim=True) + 1e-5)
        near(got[1], dx, tol, terms if dim < 8 else None, "dx")
        near(got[2], dw, F32_TOL, mw, "dw")


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,dim", [(5000, 128), (70000, 32), (3000, 2048), (1100, 8192), (2600, 1001), (0, 128)])
def test_many_rows(device, dtype, rows, dim):
    """More rows than the blocks take at once, and none."""
    for centre in (True, False):
        x, dy, w, b = make(rows, dim, dtype, seed=3)
        _, dx, dw, db, mw, mb = formulas(x, dy, w, b, 1e-5, centre)
        got = run(x, dy, w, b, device, centre)
        near(got[1], dx, F32_TOL if dtype == torch.float32 else BF16_TOL, what="dx")
        near(got[2], dw, F32_TOL, mw, "dw")
        if centre:
            near(got[3], db, F32_TOL, mb, "db")


@pytest.mark.parametrize("centre", [True, False], ids=["layer", "rms"])
def test_degenerate_rows(device, centre):
    """Constant rows and zero rows (eps holds), a large mean under a small spread, tiny and large values."""
    x, dy, w, b = make(6, 256, torch.float32, seed=4)
    x[0], x[1] = 0.0, 3.0
    x[2] = 1000.0 + x[2]
    x[3] *= 1e-15
    x[4] *= 1e15
    _, dx, dw, _, mw, _ = formulas(x, dy, w, b, 1e-5, centre)
    got = run(x, dy, w, b, device, centre)
    # the mean of row 2 is rounded to 2^-24 of itself, against a spread of 1
    row_tol = [F32_TOL, F32_TOL, 1000 * 2.0 ** -24 * 8 + F32_TOL, F32_TOL, F32_TOL, F32_TOL]
    for i in range(6):
        near(got[1][i], dx[i], row_tol[i], what=f"row {i}")
    near(got[2], dw, row_tol[2], mw, "dw")
    if centre:
        y = rhizome_amd.layernorm(torch.full((3, 1), 2.0, device=device), w[:1].to(device), b[:1].to(device))
        assert torch.equal(y.cpu(), b[:1].expand(3, 1))  # one value is its own mean


def test_a_bad_row_stays_alone(device):
    x, dy, w, b = make(40, 128, torch.bfloat16, seed=5)
    want = run(x, dy, w, b, device)
    x[7, 3], dy[11, 5] = float("nan"), float("inf")
    got = run(x, dy, w, b, device)
    keep = [i for i in range(40) if i not in (7, 11)]
    assert torch.equal(got[1][keep], want[1][keep]) and torch.equal(got[0][[i for i in range(40) if i != 7]],
                                                                   want[0][[i for i in range(40) if i != 7]])
    assert not bool(torch.isfinite(got[1][7].float()).any())


def test_eps_of_zero_adds_nothing_from_missing_rows(device):
    x, dy, w, b = make(3, 64, torch.float32, seed=6)  # three rows of a block's many
    for centre in (True, False):
        _, dx, dw, _, mw, _ = formulas(x, dy, w, b, 0.0, centre)
        got = run(x, dy, w, b, device, centre, eps=0.0)
        near(got[1], dx, F32_TOL, what="dx")
        near(got[2], dw, F32_TOL, mw, "dw")


def test_differences(device):
    """dx along a direction against central differences in 64 bits (step 1e-4: 1e-8 of third derivatives)."""
    for centre in (True, False):
        x, dy, w, b = make(20, 96, torch.float32, seed=7)
        got = run(x, dy, w, b, device, centre)
        gen = torch.Generator().manual_seed(8)
        for i, of in ((1, "x"), (2, "w")):
            way = torch.randn(x.shape if of == "x" else w.shape, generator=gen, dtype=torch.float64)
            ends = []
            for s in (1e-4, -1e-4):
                y = formulas(x.double() + s * way if of == "x" else x, dy, w.double() + s * way if of == "w" else w, b,
                             1e-5, centre)[0]
                ends.append(float((y * dy.double()).sum()))
            slope, mine = (ends[0] - ends[1]) / 2e-4, float((got[i].double().cpu() * way).sum())
            assert abs(slope - mine) <= 1e-5 * float(got[i].double().cpu().norm() * way.norm())


def test_unaligned_and_same_bits(device):
    for dtype in DTYPES:
        x, dy, w, b = make(300, 256, dtype, seed=9)
        want = run(x, dy, w, b, device)
        again = run(x, dy, w, b, device)
        assert all(torch.equal(p, q) for p, q in zip(want, again))
        room = [torch.empty(t.numel() + 1, dtype=dtype, device=device) for t in (x, dy)]
        for r, t in zip(room, (x, dy)):
            r[1:] = t.reshape(-1).to(device)
        got = rhizome_amd.layernorm_backward(room[1][1:].view(300, 256), room[0][1:].view(300, 256), w.to(device))
        near(got[0], want[1].double().cpu(), F32_TOL if dtype == torch.float32 else 2.0 ** -8, what="dx")


def test_stream_graph_and_leading_shapes(device):
    x, dy, w, b = (t.to(device) for t in make(120, 128, torch.bfloat16, seed=10))
    want = run(x, dy, w, b, device)
    got = rhizome_amd.layernorm_backward(dy.view(4, 30, 128), x.view(4, 30, 128), w)
    assert got[0].shape == (4, 30, 128) and torch.equal(got[0].view(120, 128), want[1])
    torch.cuda.synchronize()
    got = rhizome_amd.layernorm_backward(dy, x, w, stream=torch.cuda.Stream())
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want[1:]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = rhizome_amd.layernorm(x, w, b)
        got = rhizome_amd.rmsnorm_heads_backward(dy, x, w)
    for s in (1.0, 2.0, 0.5):
        x.copy_(x * s)
        graph.replay()
        torch.cuda.synchronize()
        want = run(x, dy, w, b, device)
        assert torch.equal(y, want[0])
        want = run(x, dy, w, b, device, False, 1e-6)
        assert torch.equal(got[0], want[1]) and torch.equal(got[1], want[2])


def test_in_place_and_refusals(device):
    x, dy, w, b = (t.to(device) for t in make(50, 128, torch.float32, seed=11))
    want = rhizome_amd.layernorm(x, w, b)
    z = x.clone()
    assert torch.equal(rhizome_amd.layernorm(z, w, b, out=z), want)
    near(rhizome_amd.layernorm(x, w), (want - b).double().cpu(), 1e-5, want.double().cpu())
    for f in (lambda: rhizome_amd.layernorm(x, w[:64]), lambda: rhizome_amd.layernorm(x, w, b.double()),
              lambda: rhizome_amd.layernorm(x.half(), w), lambda: rhizome_amd.layernorm_backward(dy[:9], x, w),
              lambda: rhizome_amd.layernorm_backward(dy.bfloat16(), x, w), lambda: rhizome_amd.layernorm(x.T, x[:, 0]),
              lambda: rhizome_amd.rmsnorm_heads_backward(dy, x, w.bfloat16())):
        with pytest.raises(ValueError):
            f()
    with pytest.raises(rhizome_amd.gdr.GdrError):
        rhizome_amd.layernorm(torch.zeros(1, 8193, device=device), torch.zeros(8193, device=device))
    with pytest.raises(rhizome_amd.gdr.GdrError):
        rhizome_amd.layernorm_backward(dy, x, w, workspace=torch.empty(16, device=device))
