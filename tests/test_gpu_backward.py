"""Backward pass of the gated delta-rule prefill against torch's derivative of
the recurrence in 64 bits on the CPU, token by token.

Tolerances, of the 2-norm of each gradient, set before the first run:
* fp32 calls: 1e-5.  A gradient is a sum of chains of some ten products, each
  accumulated over up to 128 terms with half a step (2^-24) of error each; with
  signs at random that is about sqrt(128) * 10 * 2^-24 = 7e-6.
* bf16 calls: half a step of the output, 2^-8, plus one of an fp16 operand,
  2^-11, for each of eight products in a chain (T, its products with K and V,
  W or dX, the state, N, and the operands they meet): 2^-8 + 8 * 2^-11 = 2^-7.
  grad_initial_state is not rounded to bf16 and gets the second part alone.
"""
import math

import pytest
import torch

import rhizome_amd

pytestmark = pytest.mark.gpu
NAMES = ("dq", "dk", "dv", "dgate", "dbeta", "dstate")
TOL = {torch.float32: 1e-5, torch.bfloat16: 2.0 ** -7}


def inputs(dtype, lengths, H, dk, dv, *, seed=0, gate="g", g_mean=0.0, state=True, dense=False, scale=1.0):
    """Rounded inputs of one call on the CPU; `dense`: the sequences have one length."""
    gen = torch.Generator().manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, dtype=torch.float64)

    n = sum(lengths)
    q, k = normal(n, H, dk), normal(n, H, dk)
    q = q / q.norm(dim=-1, keepdim=True) * math.sqrt(dk)
    k = k / k.norm(dim=-1, keepdim=True)
    g = -torch.nn.functional.softplus(normal(n, H) + g_mean)
    d = dict(q=q.to(dtype), k=k.to(dtype), v=normal(n, H, dv).to(dtype), beta=torch.sigmoid(normal(n, H)).float(),
             do=(normal(n, H, dv) * scale).to(dtype))
    d["g" if gate == "g" else "alpha"] = (g if gate == "g" else g.exp()).float()
    if state:
        d["initial_state"] = normal(len(lengths), H, dv, dk).float() * 0.1
        d["dfinal_state"] = (normal(len(lengths), H, dv, dk) * 0.1 * scale).float()
    return d


def reference(d, lengths):
    """Gradients by torch from the recurrence in 64 bits, sequence by sequence."""
    leaf = {x: t.double().requires_grad_(True) for x, t in d.items() if x not in ("do", "dfinal_state")}
    H, dk, dv = d["q"].shape[1], d["q"].shape[2], d["v"].shape[2]
    gate = "g" if "g" in d else "alpha"
    state = leaf.get("initial_state")
    if state is None:
        state = torch.zeros(len(lengths), H, dv, dk, dtype=torch.float64, requires_grad=True)
    loss, at = torch.zeros((), dtype=torch.float64), 0
    for n, length in enumerate(lengths):
        S = state[n]
        for t in range(at, at + length):
            a = leaf[gate][t].exp() if gate == "g" else leaf[gate][t]
            kt, b = leaf["k"][t], leaf["beta"][t]
            u = b[:, None] * (leaf["v"][t] - a[:, None] * (S @ kt[..., None])[..., 0])
            S = a[:, None, None] * S + u[..., None] * kt[:, None, :]
            loss = loss + ((S @ leaf["q"][t][..., None])[..., 0] * d["do"][t].double()).sum()
        if "dfinal_state" in d:
            loss = loss + (S * d["dfinal_state"][n].double()).sum()
        at += length
    wrt = [leaf["q"], leaf["k"], leaf["v"], leaf[gate], leaf["beta"], state]
    got = torch.autograd.grad(loss, wrt, allow_unused=True)
    return [torch.zeros_like(x) if y is None else y for x, y in zip(wrt, got)]


def call(d, lengths, device, dense=False, **kw):
    """The gradients on the CPU, packed; `dense`: through the dense layout."""
    a = {x: t.to(device) for x, t in d.items()}
    if dense:
        B, T = len(lengths), lengths[0]
        a = {x: t if "state" in x else t.reshape(B, T, *t.shape[1:]) for x, t in a.items()}
    else:
        a["cu_seqlens"] = torch.tensor([0] + list(torch.tensor(lengths).cumsum(0)), dtype=torch.int32, device=device)
    out = rhizome_amd.prefill_backward(**a, output_dinitial_state=True, **kw)
    torch.cuda.synchronize()
    return [x.cpu() if "state" in name else x.cpu().reshape(-1, *x.shape[1 if not dense else 2:])
            for name, x in zip(NAMES, out)]


def check(got, want, dtype, what="", only=NAMES):
    for name, x, y in zip(NAMES, got, want):
        if name not in only:
            continue
        assert x.shape == y.shape, (what, name)
        assert bool(torch.isfinite(x).all()), f"{what} {name}: not finite"
        tol = TOL[dtype] - (2.0 ** -8 if dtype == torch.bfloat16 and name == "dstate" else 0.0)
        err, norm = float((x.double() - y).norm()), float(y.norm())
        assert err <= tol * norm + 1e-30, f"{what} {name}: {err / max(norm, 1e-300):.3g} of the norm, tolerance {tol:.3g}"


DTYPES = [torch.float32, torch.bfloat16]
SHAPES = [
    # lengths, H, d_k, d_v
    ([1], 1, 32, 32), ([2], 3, 1, 1), ([63], 2, 64, 64), ([64], 2, 128, 128), ([65], 2, 128, 128), ([200], 2, 128, 256),
    ([130], 1, 20, 36), ([100], 2, 37, 51), ([70], 2, 96, 17), ([129], 1, 8, 200), ([66], 1, 33, 1024),
    ([0, 70, 1, 0, 129, 64], 2, 64, 32), ([3, 2, 1], 2, 128, 48),
]


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("lengths,H,dk,dv", SHAPES)
def test_shapes(device, dtype, lengths, H, dk, dv):
    d = inputs(dtype, lengths, H, dk, dv, seed=len(lengths) + dk)
    want = reference(d, lengths)
    check(call(d, lengths, device), want, dtype, "packed")
    if len(set(lengths)) == 1:
        check(call(d, lengths, device, dense=True), want, dtype, "dense")


@pytest.mark.parametrize("dk", [20, 64, 100, 128])
def test_more_state_tiles_than_cus(device, dk):
    """Two sequences of 16 heads and 80 value channels: 384 tiles of 16 state
    rows over both scans, which share workgroups."""
    d = inputs(torch.float32, [70, 3], 16, dk, 80, seed=dk)
    check(call(d, [70, 3], device), reference(d, [70, 3]), torch.float32)


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("gate", ["g", "alpha"])
@pytest.mark.parametrize("g_mean", [-6.0, 3.0])
def test_decays(device, dtype, gate, g_mean):
    """Decays near 1 and strong ones, as ln alpha and as alpha, without states."""
    d = inputs(dtype, [150, 150], 2, 64, 64, gate=gate, g_mean=g_mean, state=False, seed=5)
    check(call(d, [150, 150], device, dense=True), reference(d, [150, 150]), dtype)


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("gate", ["g", "alpha"])
def test_resets(device, dtype, gate):
    """alpha = 0 and tiny alphas, in a chunk's first, inner and last places and twice in a row."""
    d = inputs(dtype, [190], 2, 64, 64, gate=gate, seed=6)
    at, small = [0, 5, 6, 64, 100, 127, 189], [1e-20, 1e-30, 1e-38]
    if gate == "alpha":
        d["alpha"][at, 0] = 0.0
        d["alpha"][[20, 70, 130], 1] = torch.tensor(small)
    else:
        d["g"][at, 0] = -math.inf
        d["g"][[20, 70, 130], 1] = torch.tensor(small).log()
    want = reference(d, [190])
    if gate == "g":  # 0 * inf in the derivative of exp at -inf, whose value is 0
        want[3] = torch.nan_to_num(want[3])
    got = call(d, [190], device)
    check(got, want, dtype)
    if gate == "alpha":  # each one's own gradient, not only the norm of all
        scale = float(want[3].norm()) / math.sqrt(want[3].numel())
        for t in at:
            assert abs(float(got[3][t, 0]) - float(want[3][t, 0])) <= TOL[dtype] * (abs(float(want[3][t, 0])) + 8 * scale)


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
def test_small_alphas_keep_their_gradients(device, dtype):
    """dalpha = dg / alpha: nothing may cancel in dg where alpha is small."""
    d = inputs(dtype, [128], 1, 64, 64, gate="alpha", seed=7)
    d["alpha"][::9, 0] = 10.0 ** -torch.arange(1.0, 16.0)[:len(d["alpha"][::9, 0])]
    got, want = call(d, [128], device), reference(d, [128])
    check(got, want, dtype)
    x, y = got[3][::9, 0].double(), want[3][::9, 0]
    assert float((x - y).norm()) <= TOL[dtype] * float(y.norm())


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
def test_beta_of_zero_and_one(device, dtype):
    d = inputs(dtype, [140], 2, 64, 64, seed=8)
    d["beta"][:, 0] = (torch.arange(140) % 2).float()
    d["beta"][:, 1] = 0.0
    d["beta"][70, 1] = 1.0
    check(call(d, [140], device), reference(d, [140]), dtype)


@pytest.mark.parametrize("scale", [1e-30, 1e-9, 1e6])
def test_magnitudes_of_bf16_inputs(device, scale):
    """The gradient's, the values', the keys' and the queries' magnitudes are taken up by the tiles' exponents."""
    d = inputs(torch.bfloat16, [150], 2, 64, 64, seed=9, scale=scale)
    check(call(d, [150], device), reference(d, [150]), torch.bfloat16, "grad_o")
    d = inputs(torch.bfloat16, [150], 2, 64, 64, seed=9)
    s = max(scale, 1e-12)
    d["v"], d["initial_state"] = (d["v"].double() * s).bfloat16(), d["initial_state"] * s
    check(call(d, [150], device), reference(d, [150]), torch.bfloat16, "v")
    d["q"] = (d["q"].double() * s).bfloat16()
    check(call(d, [150], device), reference(d, [150]), torch.bfloat16, "q")


def test_magnitudes_along_a_bf16_sequence(device):
    """Late and early tokens of very different sizes, and a state far above what follows it."""
    d = inputs(torch.bfloat16, [256], 1, 64, 64, seed=10, g_mean=1.0)
    d["initial_state"] *= 1e5
    d["do"][:128] *= 2.0 ** -20
    want, got = reference(d, [256]), call(d, [256], device)
    check(got, want, torch.bfloat16)
    for part in (slice(0, 64), slice(64, 128), slice(128, 192), slice(192, 256)):  # chunk by chunk
        for i in (0, 2):
            x, y = got[i][part].double(), want[i][part]
            assert float((x - y).norm()) <= TOL[torch.bfloat16] * float(y.norm()), (part, NAMES[i])


@pytest.mark.parametrize("size", [0.0, 1e-2, 1e-4, 2e-5, 1e-6, 1e-12])
def test_small_keys_in_bf16(device, size):
    """Keys of a chunk that are zero or small: what they multiply keeps its
    size, and so do the gradients that do not pass through them."""
    d = inputs(torch.bfloat16, [200, 64], 2, 64, 64, seed=9)
    d["k"][64:128] = (d["k"][64:128].double() * size).to(torch.bfloat16)
    d["k"][200:, 1] = (d["k"][200:, 1].double() * size).to(torch.bfloat16)
    got, want = call(d, [200, 64], device), reference(d, [200, 64])
    check(got, want, torch.bfloat16)
    for rows in (slice(64, 128), slice(200, 264)):  # each chunk against its own norm
        check([x[rows] for x in got[:3]], [x[rows] for x in want[:3]], torch.bfloat16, str(rows))


@pytest.mark.parametrize("decay", [0.0, -0.05])
@pytest.mark.parametrize("d_k,d_v", [(128, 64), (32, 64)])
def test_tokens_that_agree_in_bf16(device, d_k, d_v, decay):
    """Queries, keys, values and output gradients all along one direction: a
    chunk's sums over its tokens and channels have every term of one sign."""
    d = inputs(torch.bfloat16, [200, 64], 2, d_k, d_v, seed=8, state=False)
    for name, x in (("q", 1.9), ("v", 1.0), ("do", 1.9)):
        d[name] = (d[name].double() * 0.01 + x).to(torch.bfloat16)
    d["k"].fill_(d_k ** -0.5)
    d["beta"].fill_(0.02)
    d["g"].fill_(decay)
    check(call(d, [200, 64], device), reference(d, [200, 64]), torch.bfloat16)


@pytest.mark.parametrize("what", ["long keys", "beta above 1", "alpha above 1"])
def test_bf16_outside_the_domain(device, what):
    """One head of two leaves the fp16 path's domain and is computed in fp32;
    the other head's bits do not change.  A key scaled as here, beta |k|^2
    up to 4, lets the recurrence grow by up to 3 a token along it."""
    d = inputs(torch.bfloat16, [100, 60], 2, 64, 64, seed=11, gate="alpha")
    before = call(d, [100, 60], device)
    if what == "long keys":
        d["k"][:, 0] *= 2
    elif what == "beta above 1":
        d["beta"][30, 0] = 1.5
    else:
        d["alpha"][130, 0] = 1.25
    got, want = call(d, [100, 60], device), reference(d, [100, 60])
    check(got, want, torch.bfloat16)
    for x, y in zip(got[:5], before[:5]):
        assert torch.equal(x[:, 1], y[:, 1])
    assert torch.equal(got[5][:, 1], before[5][:, 1])


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
def test_not_finite(device, dtype):
    """A NaN or an infinity stays in its own sequence and head."""
    lengths = [70, 80, 66]
    d = inputs(dtype, lengths, 2, 64, 64, seed=12)
    want = call(d, lengths, device)
    for name, bad in (("q", math.nan), ("k", math.inf), ("v", math.nan), ("do", -math.inf), ("beta", math.nan)):
        e = {x: t.clone() for x, t in d.items()}
        if name == "beta":
            e[name][100, 1] = bad
        else:
            e[name][100, 1, 3] = bad
        got = call(e, lengths, device)
        for x, y in zip(got[:5], want[:5]):
            assert torch.equal(x[:, 0], y[:, 0]) and torch.equal(x[:70], y[:70]) and torch.equal(x[150:], y[150:])
        assert not bool(torch.isfinite(torch.cat([x[70:150, 1].reshape(-1).float() for x in got[:5]])).all()), name


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
def test_a_sequence_is_the_same_alone_and_in_a_pack(device, dtype):
    lengths = [65, 0, 200, 1, 127]
    d = inputs(dtype, lengths, 3, 64, 128, seed=13)
    got = call(d, lengths, device)
    at = 0
    for n, length in enumerate(lengths):
        one = {x: (t[n:n + 1] if "state" in x else t[at:at + length]) for x, t in d.items()}
        alone = call(one, [length], device, dense=length > 0)
        for name, x, y in zip(NAMES, got, alone):
            assert torch.equal(x[n:n + 1] if name == "dstate" else x[at:at + length], y), (n, name)
        at += length


def test_rows_outside_the_sequences_stay(device):
    """Offsets that leave rows before, between nothing, and behind: their gradients' memory is not written."""
    H, dk, dv = 2, 64, 64
    d = inputs(torch.bfloat16, [200], H, dk, dv, seed=14, state=False)
    a = {x: t.to(device) for x, t in d.items()}
    cu = torch.tensor([7, 90, 90, 163], dtype=torch.int32, device=device)
    args = dict(cu_seqlens=cu, **a)
    marked = rhizome_amd.train._empty
    rhizome_amd.train._empty = lambda like, shape, dtype=None: marked(like, shape, dtype).fill_(77)
    try:
        out = rhizome_amd.prefill_backward(**args)
    finally:
        rhizome_amd.train._empty = marked
    part = {x: t[7:163] for x, t in d.items()}
    want = call(part, [83, 0, 73], device)
    for x, y in zip(out[:5], want[:5]):
        x = x.cpu()
        assert torch.equal(x[7:163], y) and bool((x[:7] == 77).all()) and bool((x[163:] == 77).all())


@pytest.mark.parametrize("offsets", [[0, 150, 40, 200], [-5, 500, 100, 100]])
def test_bad_offsets_stay_inside(device, offsets):
    """Decreasing and out-of-range offsets are cut to the pack: some results, and no access outside."""
    d = inputs(torch.bfloat16, [200], 2, 64, 64, seed=15, state=False)
    a = {x: t.to(device) for x, t in d.items()}
    rhizome_amd.prefill_backward(**a, cu_seqlens=torch.tensor(offsets, dtype=torch.int32, device=device),
                                 output_dinitial_state=True)
    torch.cuda.synchronize()


def test_empty_batch_passes_the_state_gradient_on(device):
    d = inputs(torch.float32, [0, 0], 2, 32, 48, seed=16)
    got = call(d, [0, 0], device)
    assert torch.equal(got[5], d["dfinal_state"])


def test_unaligned_tensors(device):
    """Tensors that start 2 or 4 bytes into an allocation take element-wise accesses."""
    for dtype in DTYPES:
        d = inputs(dtype, [90], 2, 64, 64, seed=17)
        want = call(d, [90], device)
        a = {}
        for x, t in d.items():
            room = torch.empty(t.numel() + 1, dtype=t.dtype, device=device)
            room[1:] = t.reshape(-1).to(device)
            a[x] = room[1:].view(t.shape)
        cu = torch.tensor([0, 90], dtype=torch.int32, device=device)
        out = rhizome_amd.prefill_backward(**a, cu_seqlens=cu, output_dinitial_state=True)
        for x, y in zip(out, want):
            assert torch.equal(x.cpu(), y)


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
def test_differences(device, dtype):
    """The gradient along a direction against central differences of the forward prefill's loss in
    64 bits.  The step of 1e-4 leaves (1e-4)^2 of third derivatives and 1e-16 / 1e-4 of rounding."""
    lengths = [96]
    d = inputs(dtype, lengths, 2, 32, 32, seed=18)
    got = call(d, lengths, device)
    gen = torch.Generator().manual_seed(19)
    names = ("q", "k", "v", "g", "beta", "initial_state")

    def loss(x):
        S, total = x["initial_state"][0], 0.0
        for t in range(96):
            a, b, kt = x["g"][t].exp(), x["beta"][t], x["k"][t]
            u = b[:, None] * (x["v"][t] - a[:, None] * (S @ kt[..., None])[..., 0])
            S = a[:, None, None] * S + u[..., None] * kt[:, None, :]
            total = total + float(((S @ x["q"][t][..., None])[..., 0] * x["do"][t]).sum())
        return total + float((S * x["dfinal_state"][0]).sum())

    base = {x: t.double() for x, t in d.items()}
    for i, name in enumerate(names):
        way = torch.randn(base[name].shape, generator=gen, dtype=torch.float64)
        h = 1e-4
        ahead, behind = ({**base, name: base[name] + s * h * way} for s in (1, -1))
        slope = (loss(ahead) - loss(behind)) / (2 * h)
        mine = float((got[i].double() * way).sum())
        room = float(got[i].double().norm() * way.norm()) / math.sqrt(way.numel())
        assert abs(mine - slope) <= 6 * (TOL[dtype] + 1e-6) * room + 1e-6 * abs(slope), name


def test_twice_the_same_bits(device):
    for dtype in DTYPES:
        d = inputs(dtype, [300, 41], 4, 128, 128, seed=20)
        a, b = call(d, [300, 41], device), call(d, [300, 41], device)
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_other_streams_and_two_calls_at_once(device):
    d1, d2 = (inputs(torch.bfloat16, [700], 4, 128, 128, seed=s) for s in (21, 22))
    want = [call(d, [700], device, dense=True) for d in (d1, d2)]
    a = [{x: (t if "state" in x else t[None]).to(device) for x, t in d.items()} for d in (d1, d2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    out = [rhizome_amd.prefill_backward(**x, output_dinitial_state=True, stream=s) for x, s in zip(a, streams)]
    junk = [torch.full((1 << 20,), 3.0, device=device) for _ in range(8)]  # would reuse a workspace let go too early
    torch.cuda.synchronize()
    assert len(junk) == 8
    for o, w in zip(out, want):
        assert all(torch.equal(x.cpu().reshape(y.shape), y) for x, y in zip(o, w))


@pytest.mark.parametrize("packed", [False, True])
def test_captured_and_replayed(device, packed):
    d = inputs(torch.bfloat16, [90, 90], 2, 64, 64, seed=23)
    e = inputs(torch.bfloat16, [90, 90], 2, 64, 64, seed=24)
    a = {x: (t if "state" in x or packed else t.reshape(2, 90, *t.shape[1:])).to(device) for x, t in d.items()}
    if packed:
        a["cu_seqlens"] = torch.tensor([0, 90, 180], dtype=torch.int32, device=device)
    rhizome_amd.prefill_backward(**a, output_dinitial_state=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rhizome_amd.prefill_backward(**a, output_dinitial_state=True)
    for turn in (d, e, d):
        for x, t in turn.items():
            a[x].copy_(t.reshape(a[x].shape))
        graph.replay()
        torch.cuda.synchronize()
        want = call(turn, [90, 90], device, dense=not packed)  # eager work between the replays
        assert all(torch.equal(x.cpu().reshape(y.shape), y) for x, y in zip(out, want))


def test_refusals_of_the_front_end(device):
    d = {x: t.to(device)[None] if "state" not in x else t.to(device)
         for x, t in inputs(torch.bfloat16, [16], 2, 32, 32).items()}
    for over in (dict(do=d["do"][:, :8]), dict(do=d["do"].float()), dict(beta=None), dict(do=None),
                 dict(dfinal_state=d["dfinal_state"][:, :1]), dict(alpha=d["g"]), dict(q=d["q"].half()),
                 dict(v=d["v"].transpose(1, 2))):
        with pytest.raises(ValueError):
            rhizome_amd.prefill_backward(**{**d, **over})
    with pytest.raises(rhizome_amd.gdr.GdrError):
        rhizome_amd.prefill_backward(**d, workspace=torch.empty(256, dtype=torch.uint8, device=device))
