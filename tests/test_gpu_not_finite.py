"""The latent attention where inputs that are seen are not finite: which results
that reaches, and that a pass of nothing but NaN takes about its usual time."""
import math

import pytest
import torch

import rhizome_amd
from attn_cases import DTYPES, attend, attend_backward, make, near
from test_gpu_latent_decode import exact, make as make_paged, run

pytestmark = pytest.mark.gpu
both = pytest.mark.parametrize("dtype", DTYPES.values(), ids=DTYPES.keys())


def all_nan(t):
    return bool(torch.isnan(t).all())


@both
@pytest.mark.parametrize("d_n,d_r,d_v", [(32, 16, 32), (64, 32, 64), (128, 64, 128), (33, 5, 17)])
@pytest.mark.parametrize("where", ["q", "k", "r", "v", "do"])
def test_what_a_nan_reaches(device, dtype, where, d_n, d_r, d_v):
    """Queries that see it, in every channel (a value's: in its own), and gradients of what they see."""
    n, at, scale = 300, 130, 0.1
    q, kv, r, do = make([n], [n], 2, d_n, d_r, d_v, dtype, seed=11)
    one = (q, kv[..., :d_n], kv[..., d_n:], r)
    want_o, want_l, tol_o, tol_l = attend(*one, scale, True, dtype)
    grads = attend_backward(*one, do, None, scale, True, dtype)
    bad = {"q": q, "k": kv[..., :d_n], "r": r, "v": kv[..., d_n:], "do": do}[where].clone()
    bad[at, ..., 3] = math.nan
    put = dict(q=q, k=one[1], v=one[2], r=r, do=do) | {where: bad}
    dev = {name: t.to(device)[None] for name, t in put.items()}
    args = [dev[name] for name in ("q", "k", "v", "r")]
    o, lse = rhizome_amd.latent_prefill(*args, scale=scale)
    got = rhizome_amd.latent_prefill_backward(*args, o, lse, dev["do"], scale=scale)
    torch.cuda.synchronize()
    o, lse, dq, dk, dv, dr = (t[0].cpu() for t in (o, lse, *got))
    reached = torch.zeros(n, dtype=torch.bool)
    reached[at if where == "q" else slice(at, None)] = where in ("q", "k", "r")
    if reached.any():
        assert all_nan(o[reached]) and all_nan(lse[reached])
    near(lse[~reached], want_l[~reached], tol_l[~reached], "lse")
    clean = torch.ones_like(want_o, dtype=torch.bool)
    clean[reached] = False
    if where == "v":
        assert all_nan(o[at:, :, 3])
        clean[at:, :, 3] = False
    near(o[clean], want_o[clean], tol_o[clean], "o")
    # a query's gradient is lost with its own row or with D, a key's where such a query sees it
    lost_q = reached.clone()
    lost_q[slice(at, None) if where == "v" else at] = True
    last = int(lost_q.nonzero().max())
    assert all_nan(dq[lost_q]) and all_nan(dk[:last + 1]) and all_nan(dr[:last + 1])
    near(dq[~lost_q], grads["dq"][0][~lost_q], grads["dq"][1][~lost_q], "dq")
    for name, x in (("dk", dk), ("dr", dr)):
        near(x[last + 1:], grads[name][0][last + 1:], grads[name][1][last + 1:], name)
    whole = grads["dv"][0].clone(), grads["dv"][1]
    if where in ("q", "k", "r"):
        assert all_nan(dv[:last + 1])
        dv, whole = dv[last + 1:], (whole[0][last + 1:], whole[1][last + 1:])
    elif where == "do":
        assert all_nan(dv[:at + 1, :, 3])
        dv[:at + 1, :, 3] = whole[0][:at + 1, :, 3] = 0.0
    near(dv, *whole, "dv")


@both
@pytest.mark.parametrize("steps,H,d_c,d_r", [(2, 8, 128, 16), (3, 8, 256, 64), (2, 30, 128, 16), (3, 40, 256, 0), (2, 8, 101, 7)])
@pytest.mark.parametrize("where", ["q", "row"])
def test_what_a_nan_reaches_in_the_cache(device, dtype, where, steps, H, d_c, d_r):
    lens, page = [1500, 70, 300], 16
    q, cache, table, n = make_paged(lens, steps, H, d_c, d_r, page, dtype, seed=12)
    want, tol = exact(q, cache, table, n, d_c, 0.1, dtype, page)
    lost = torch.zeros(want[1].shape, dtype=torch.bool)
    if where == "q":
        q[0, steps - 1, 3, 2] = math.nan
        lost[0, steps - 1, 3] = True
    else:  # the first sequence's 701st row, and the last of the others
        cache[table[0, 700 // page], 700 % page, 1] = math.nan
        cache[table[1, 69 // page], 69 % page, 1] = math.nan
        lost[0] = lost[1, steps - 1] = True
    o, lse = (t.cpu() for t in run(q, cache, table, n, d_c, 0.1, device))
    assert all_nan(o[lost]) and all_nan(lse[lost])
    near(o[~lost], want[0][~lost], tol[0][~lost], "o")
    near(lse[~lost], want[1][~lost], tol[1][~lost], "lse")


def took(f):
    """Milliseconds, the least of three."""
    f()
    best = math.inf
    for _ in range(3):
        a, b = torch.cuda.Event(True), torch.cuda.Event(True)
        a.record()
        f()
        b.record()
        torch.cuda.synchronize()
        best = min(best, a.elapsed_time(b))
    return best


def check_time(run_with, finite, cases):
    """Summed again pair by pair, these take hundreds of times as long as usual."""
    usual = took(lambda: run_with(finite))
    for name in cases:
        t = took(lambda: run_with({k: torch.full_like(v, math.nan) if k in name else v for k, v in finite.items()}))
        print(f"NaN in {', '.join(name)}: {t:.3f} ms, finite {usual:.3f}", flush=True)
        assert t < 20 * usual + 3.0, f"NaN in {name}: {t:.1f} ms instead of {usual:.2f}"


EVERY = ("q", "k", "v", "r", "do")


@both
@pytest.mark.parametrize("d_n,d_r,d_v", [(128, 64, 128), (64, 32, 64)])
def test_a_prompt_of_nan_takes_its_usual_time(device, dtype, d_n, d_r, d_v):
    gen = torch.Generator(device=device).manual_seed(1)
    shape = dict(q=(16, d_n + d_r), k=(16, d_n), v=(16, d_v), r=(d_r,), do=(16, d_v))
    t = {k: torch.randn(1, 4096, *s, generator=gen, device=device).to(dtype) for k, s in shape.items()}

    def forward(t):
        return rhizome_amd.latent_prefill(t["q"], t["k"], t["v"], t["r"])

    def backward(t):
        rhizome_amd.latent_prefill_backward(t["q"], t["k"], t["v"], t["r"], *forward(t), t["do"])

    check_time(forward, t, [("q",), ("k",), ("v",), EVERY])
    check_time(backward, t, [("q",), ("k",), ("do",), EVERY])


@both
@pytest.mark.parametrize("steps", [1, 4])
def test_a_cache_of_nan_takes_its_usual_time(device, dtype, steps):
    gen = torch.Generator(device=device).manual_seed(2)
    t = dict(q=torch.randn(32, steps, 16, 576, generator=gen, device=device).to(dtype),
             cache=torch.randn(32 * 64, 64, 576, generator=gen, device=device).to(dtype))
    table = torch.arange(32 * 64, device=device, dtype=torch.int32).view(32, 64)
    lengths = torch.full((32,), 4096, dtype=torch.int32, device=device)
    check_time(lambda t: rhizome_amd.latent_decode(t["q"], t["cache"], table, lengths, d_c=512, scale=0.05), t,
               [("q",), ("cache",), ("q", "cache")])
