"""The integration guide's example of the latent attention, run as it stands there."""
import os
import re

import pytest
import torch

import rhizome_amd
from attn_cases import W, attend, attend_backward, near, starts
from test_gpu_latent_decode import exact, pages

pytestmark = pytest.mark.gpu
GUIDE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "INTEGRATION.md")


def example():
    blocks = re.findall(r"```python\n(.*?)```", open(GUIDE).read(), re.S)
    return next(b for b in blocks if "latent_prefill(" in b)


def test_the_guides_example(device):
    """A prompt's scores come from the same keys whether it attends by the prefill or is read from the cache."""
    gen = torch.Generator().manual_seed(31)
    H, d_n, d_r, d_v, d_c, page, lens = 3, 32, 16, 24, 64, 16, [70, 5, 33]
    total, B, scale = sum(lens), len(lens), (d_n + d_r) ** -0.5
    randn = lambda *shape: torch.randn(shape, generator=gen).to(device)
    table, count = pages([n + 1 for n in lens], page, gen)
    lengths = torch.tensor(lens, dtype=torch.int32, device=device)
    ns = dict(rhizome_amd=rhizome_amd, H=H, d_n=d_n, d_r=d_r, d_v=d_v, d_c=d_c, q=randn(total, H, d_n + d_r), c=randn(total, d_c),
              r=randn(total, d_r), w_norm=torch.rand(d_c, generator=gen).to(device) + 0.5, w_kv=randn(d_c, H * (d_n + d_v)) / 8,
              positions=torch.cat([torch.arange(n) for n in lens]).int().to(device), cu=starts(lens).to(device),
              cache=torch.zeros(count, page, d_c + d_r, device=device), page_table=table.to(device), lengths=lengths,
              do=randn(total, H, d_v), c1=randn(B, 1, d_c), r1=randn(B, 1, d_r), lengths1=lengths + 1,
              q1=randn(B, 1, H, d_c + d_r))
    exec(example(), ns)
    torch.cuda.synchronize()
    got = {name: t.cpu() for name, t in ns.items() if isinstance(t, torch.Tensor)}
    begin = [0, *torch.tensor(lens).cumsum(0).tolist()]
    for b, n in enumerate(lens):
        at, p = slice(begin[b], begin[b + 1]), torch.arange(n)
        rows = got["cache"].view(-1, d_c + d_r)[table[b, p // page].long() * page + p % page].double()
        c_n, k_rope = got["c_n"][at].double(), got["k_rope"][at].double()
        # a norm is the square root of d_c squares' sum, a value three more products; a turned one two products of
        # factors that the magnitude 1 and the fp32 sine and cosine leave off by a few steps
        near(rows[:, :d_c], c_n, (d_c + 16) * W * c_n.abs(), "normalised latents")
        size = got["r"][at].double().abs()
        near(rows[:, d_c:], k_rope, 16 * W * (size + size.roll(d_r // 2, -1)), "turned keys")
        one = [got[name][at] for name in ("q", "k", "v", "k_rope")]
        o, lse, tol_o, tol_lse = attend(*one, scale, True, torch.float32)
        near(got["o"][at], o, tol_o, "o")
        near(got["lse"][at], lse, tol_lse, "lse")
        grads = attend_backward(*one, got["do"][at], None, scale, True, torch.float32)
        for name in ("dk", "dv"):
            near(got[name][at], *grads[name], name)
        # dq and dr are turned back, which keeps the length of every pair
        for name, x in (("dq", got["dq"][at][..., d_n:]), ("dr", got["dr"][at])):
            want, tol = grads[name]
            want, tol = want[..., -d_r:], tol[..., -d_r:]
            pair = lambda t: (t.double()[..., :d_r // 2] ** 2 + t.double()[..., d_r // 2:] ** 2).sqrt()
            near(pair(x), pair(want), pair(tol) + 16 * W * pair(want), name)
    want, tol = exact(got["q1"], got["cache"], table, got["lengths1"], d_c, scale, torch.float32, page)
    near(got["o1"], want[0], tol[0], "o of the step")
    near(got["lse1"], want[1], tol[1], "lse of the step")
