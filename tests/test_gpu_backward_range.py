"""The bf16 backward pass of the delta-rule prefill where its fp16 operands
come near the ends of fp16's range, against the same reference and with the
same tolerances as test_gpu_backward.py.

The inputs are such that a gradient does not cancel to a small remainder of the
terms that it is summed from, whose rounding the tolerances count: keys that
repeat have beta up to 1/2, a decay beside it, and so on.
"""
import math

import pytest
import torch

from test_gpu_backward import call, check, inputs, reference

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def alike(lengths, H, dk, dv, keys, beta, decay):
    """Queries, values and output gradients near one direction.  `keys`: one key
    for all tokens, unit vectors in turn, or random ones with a mean."""
    d = inputs(BF16, lengths, H, dk, dv, seed=31, state=False)
    noise = 1.0 if keys == "random" else 0.01
    for name, x in (("q", 1.0), ("v", 1.0), ("do", 1.9)):
        d[name] = (d[name].double() * noise + (2.0 if keys == "random" else x)).to(BF16)
    n = d["k"].shape[0]
    if keys == "one":
        d["k"].fill_(dk ** -0.5)
    elif keys == "units":
        d["k"] = torch.eye(dk)[torch.arange(n) % dk][:, None].expand(n, H, dk).contiguous().to(BF16)
    else:
        d["q"], k = d["q"].double(), d["k"].double() * math.sqrt(dk) + 2.0
        d["q"] = (d["q"] / d["q"].norm(dim=-1, keepdim=True) * math.sqrt(dk)).to(BF16)
        d["k"] = (k / k.norm(dim=-1, keepdim=True)).to(BF16)
    d["beta"].fill_(beta)
    d["g"].fill_(decay)
    return d


@pytest.mark.parametrize("keys,d_v,beta,decay", [
    ("one", 1024, 0.1, -0.05), ("one", 256, 0.5, -0.5), ("one", 1024, 0.5, -0.5), ("units", 64, 1.0, 0.0),
    ("units", 256, 0.5, -0.05), ("units", 1024, 1.0, 0.0), ("random", 1024, 1.0, -0.5), ("random", 1024, 0.5, -0.05)])
def test_sums_over_channels_that_agree(device, keys, d_v, beta, decay):
    """dX.W over the value channels, all terms of one sign: up to 4e6 in units
    of its operands' exponents, where fp16 ends at 65504."""
    d = alike([200, 64], 1, 128, d_v, keys, beta, decay)
    check(call(d, [200, 64], device), reference(d, [200, 64]), BF16)


def test_a_large_state_that_channels_share(device):
    """dO.W over the value channels: W is the state's share of a value, here
    1000 times the value itself and the same in every channel."""
    d = inputs(BF16, [100, 200], 1, 128, 1024, seed=32)
    d["do"] = (d["do"].double() * 0.01 + 1.9).to(BF16)
    k = 128 ** -0.5 + 0.01 * d["k"].double() * math.sqrt(128)
    d["k"] = (k / k.norm(dim=-1, keepdim=True)).to(BF16)
    d["initial_state"] = 1000.0 + d["initial_state"] * 10.0
    d["g"].fill_(-0.05)
    check(call(d, [100, 200], device), reference(d, [100, 200]), BF16)


def test_a_value_gradient_beyond_fp16(device):
    """The first token's dX is 69 000 in units of its exponent, from operands
    that fp16 holds, and the state takes a fifth of it: nothing but dX itself
    says that the head has left fp16's range."""
    d = inputs(BF16, [64], 2, 128, 16, seed=33, state=False)
    up, across = torch.ones(128, dtype=torch.float64) / math.sqrt(128), torch.ones(128, dtype=torch.float64) / math.sqrt(128)
    across[1::2] *= -1
    d["q"][:, 0] = 15.875
    for t, side in ((0, 1), (1, -1)):
        d["k"][t, 0] = (math.cos(math.radians(50)) * up + side * math.sin(math.radians(50)) * across).to(BF16)
    d["do"][:, 0] = 1.9921875
    d["g"][:, 0], d["beta"][:, 0] = 0.0, 0.0
    d["g"][0, 0], d["beta"][:2, 0] = math.log(0.2), 1.0
    check(call(d, [64], device), reference(d, [64]), BF16)


@pytest.mark.parametrize("state", [True, False])
@pytest.mark.parametrize("beta", [1e-5, 1e-7, 1e-9, 1e-20])
def test_small_betas(device, beta, state):
    """Gates that are all but shut in every token of a head, or of a chunk of
    it: every gradient keeps its bits, however small it is."""
    d = inputs(BF16, [200, 64], 2, 128, 128, seed=34, state=state)
    d["beta"][:, 0] = beta
    d["beta"][64:128, 1] = beta
    got, want = call(d, [200, 64], device), reference(d, [200, 64])
    for h in (0, 1):  # each head against its own norms
        check([x[:, h] for x in got], [x[:, h] for x in want], BF16, f"head {h}")
    check([got[2][64:128, 1]], [want[2][64:128, 1]], BF16, "the chunk's")


@pytest.mark.parametrize("gate", ["g", "alpha"])
@pytest.mark.parametrize("g", [-12.0, -20.0, -60.0])
def test_strong_decays_keep_the_state_gradients(device, g, gate):
    """Decays of 6e-6 to 9e-27 a token.  The state's gradient is dO's and dX's
    share times the first token's decay, and as accurate for it."""
    d = inputs(BF16, [200, 64, 1], 2, 64, 64, seed=35, gate=gate)
    d[gate][:, 0] = g if gate == "g" else math.exp(g)
    d[gate][[0, 200, 264], 1] = g if gate == "g" else math.exp(g)  # the first token's alone
    got, want = call(d, [200, 64, 1], device), reference(d, [200, 64, 1])
    for h in (0, 1):
        check([x[:, h] for x in got], [x[:, h] for x in want], BF16, f"head {h}")


@pytest.mark.parametrize("g", [-25.0, -40.0, -math.inf])
@pytest.mark.parametrize("at", [64, 128])
def test_a_large_state_forgotten(device, at, g):
    """A state 1e9 times what the values make of it, up to a chunk's first
    token, which forgets it: the tokens behind keep their gradients."""
    d = inputs(BF16, [200], 2, 64, 64, seed=36)
    d["initial_state"] *= 1e10
    d["g"].fill_(-0.02)
    d["g"][at] = g
    got, want = call(d, [200], device), reference(d, [200])
    want[3] = torch.nan_to_num(want[3])  # 0 * inf in the derivative of exp at -inf, whose value is 0
    check([x[at:] for x in got[:5]], [x[at:] for x in want[:5]], BF16)
