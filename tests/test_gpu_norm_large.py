"""Row norms of as many rows as 32-bit sizes name, and of more."""
import pytest
import torch

import rhizome_amd

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layer", [False, True])
def test_backward_of_the_most_rows(device, layer):
    """2^31 - 1 rows of one value: the row counter's last steps lie beyond 2^31.
    Zeros but for the first and the last rows, so that the sums are of a few
    terms.  With eps = 1, r = (x^2 + 1)^(-1/2) for RMSNorm and 1 for layer norm,
    whose centred values are 0."""
    rows, ends = (1 << 31) - 1, 9000
    x = torch.zeros((rows, 1), dtype=torch.bfloat16, device=device)
    dy = torch.zeros_like(x)
    gen = torch.Generator().manual_seed(41)
    w = torch.full((1,), 2.0, device=device)
    part = [torch.randn((ends, 1), generator=gen).bfloat16() for _ in range(4)]
    x[:ends], x[-ends:], dy[:ends], dy[-ends:] = (t.to(device) for t in part)
    if layer:
        dx, dw, db = rhizome_amd.layernorm_backward(dy, x, w, 1.0)
    else:
        dx, dw = rhizome_amd.rmsnorm_heads_backward(dy, x, w, 1.0)
    torch.cuda.synchronize()
    xs, ys = torch.cat(part[:2]).double(), torch.cat(part[2:]).double()
    r = (xs * xs + 1.0).rsqrt()
    want = torch.zeros_like(xs) if layer else 2.0 * r * ys * (1.0 - (xs * r) ** 2)
    got = torch.cat([dx[:ends], dx[-ends:]]).cpu().double()
    # dx: r and five products in fp32, then bf16's half step
    assert bool(((got - want).abs() <= 2.0 ** -8 * want.abs() + 1e-6).all())
    for at in range(ends, rows - ends, 1 << 28):
        assert not bool(dx[at:min(at + (1 << 28), rows - ends)].any())
    # sums of 18000 terms, each thread's in fp32
    if layer:
        assert float(dw) == 0.0 and abs(float(db) - float(ys.sum())) <= 2.0 ** -24 * 18000 * float(ys.abs().sum())
    else:
        terms = ys * xs * r
        assert abs(float(dw) - float(terms.sum())) <= 2.0 ** -24 * 18000 * float(terms.abs().sum())


@pytest.mark.parametrize("name", ["rmsnorm_heads", "layernorm", "rmsnorm_heads_backward", "layernorm_backward"])
def test_more_rows_than_the_sizes_hold(device, name):
    """2^32 + 5 rows are refused, not taken for five."""
    x = torch.empty(((1 << 32) + 5, 1), dtype=torch.bfloat16, device=device)
    w = torch.ones(1, device=device)
    args = (x, x, w) if "backward" in name else (x, w)
    with pytest.raises(ValueError, match="2\\^31"):
        getattr(rhizome_amd, name)(*args)
