"""The latent attention's operators as a program calls them: on other streams,
two at once, in graphs, and over numbers of heads that share out unevenly."""
import pytest
import torch

import rhizome_amd
from attn_cases import DTYPES, make, normal, starts

pytestmark = pytest.mark.gpu
both = pytest.mark.parametrize("dtype", DTYPES.values(), ids=DTYPES.keys())


def values(shape, device, dtype=torch.bfloat16, seed=0):
    return normal(shape, torch.Generator().manual_seed(seed), dtype).to(device)


def paged(lens, H, d_c, d_r, page, device, dtype=torch.bfloat16, seed=0):
    gen = torch.Generator().manual_seed(seed)
    width = max(-(-n // page) for n in lens) + 1
    table = torch.randperm(len(lens) * width, generator=gen).to(torch.int32).view(len(lens), width)
    cache = normal((len(lens) * width, page, d_c + d_r), gen, dtype)
    q = normal((len(lens), 1, H, d_c + d_r), gen, dtype)
    return tuple(t.to(device) for t in (q, cache, table, torch.tensor(lens, dtype=torch.int32)))


def cases(device):
    """name: the call on a stream, its first result."""
    x, pos = values((1 << 14, 8, 128), device), torch.arange(1 << 14, dtype=torch.int32, device=device)
    freq = rhizome_amd.rope_frequencies(128, device=device)[0]
    q, cache, table, n = paged([4000] * 64, 64, 512, 64, 64, device)
    pq, kv, do = (values((1, 4096, 16, d), device, seed=s) for s, d in enumerate((128, 256, 128)))
    pk, pv = kv[..., :128], kv[..., 128:]
    o, lse = rhizome_amd.latent_prefill(pq, pk, pv)
    return {
        "rope": lambda s: rhizome_amd.rope(x, pos, freq, stream=s),
        "latent_decode": lambda s: rhizome_amd.latent_decode(q, cache, table, n, d_c=512, scale=0.04, stream=s)[0],
        "latent_prefill": lambda s: rhizome_amd.latent_prefill(pq, pk, pv, stream=s)[0],
        "latent_prefill_backward": lambda s: rhizome_amd.latent_prefill_backward(pq, pk, pv, None, o, lse, do, stream=s)[0],
    }


NAMES = ["rope", "latent_decode", "latent_prefill", "latent_prefill_backward"]


@pytest.mark.parametrize("name", NAMES)
def test_memory_that_the_current_stream_still_reads(device, name):
    """A tensor let go on the current stream while a copy of it waits there is not
    taken up for the outputs of a call on another stream."""
    run, side = cases(device)[name], torch.cuda.Stream()
    want = run(None)
    run(side)
    torch.cuda.synchronize()
    old = torch.full(want.shape, 7.0, dtype=want.dtype, device=device)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda._sleep(20_000_000)  # ends by itself: some 10 to 200 ms
    copy = torch.empty_like(old).copy_(old)
    del old
    got = run(side)
    torch.cuda.synchronize()
    assert bool((copy == 7.0).all())
    assert torch.equal(got, want)


@pytest.mark.parametrize("name", NAMES)
def test_two_at_once(device, name):
    """The same call on two streams, each with a workspace of its own."""
    run, streams = cases(device)[name], [torch.cuda.Stream() for _ in range(2)]
    want = run(None)
    torch.cuda.synchronize()
    got = [run(s) for _ in range(3) for s in streams]
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in got)


def test_append_on_another_stream(device):
    q, cache, table, n = paged([100, 33], 1, 128, 16, 8, device)
    new, side = values((2, 5, 144), device), torch.cuda.Stream()
    want = rhizome_amd.latent_append(new[..., :128], new[..., 128:], cache.clone(), table, n)
    torch.cuda.synchronize()
    got = rhizome_amd.latent_append(new[..., :128], new[..., 128:], cache, table, n, stream=side)
    torch.cuda.synchronize()
    assert torch.equal(got, want)


@both
def test_decoding_steps_in_a_graph(device, dtype):
    """rope in place, append and decode, captured once; every replay is one more
    token for each sequence, as it is for the eager calls on a cache of their own."""
    B, H, d_c, d_r, page = 3, 16, 256, 32, 16
    lens = [15, 300, 62]
    _, cache, table, n = paged([x + 8 for x in lens], H, d_c, d_r, page, device, dtype)
    n.copy_(torch.tensor(lens, dtype=torch.int32))
    freq, mag = rhizome_amd.rope_frequencies(d_r, device=device)
    norm = torch.rand(d_c, generator=torch.Generator().manual_seed(1)).to(device) + 0.5

    def step(q, c, r, cache, n):
        rhizome_amd.rope(q, n - 1, freq, offset=d_c, out=q)  # of a head's channels the last d_r
        rhizome_amd.latent_append(c, r, cache, table, n, frequencies=freq, norm_scale=norm)
        return rhizome_amd.latent_decode(q[:, None], cache, table, n, d_c=d_c, scale=0.06)

    q, c, r = values((B, H, d_c + d_r), device, dtype), values((B, 1, d_c), device, dtype), values((B, 1, d_r), device, dtype)
    eager_cache, eager_n = cache.clone(), n.clone()
    step(q.clone(), c, r, cache.clone(), n)  # loads what a first call loads
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        n.add_(1)
        o, lse = step(q, c, r, cache, n)
    assert torch.equal(n, eager_n)
    for i in range(4):
        for s, t in enumerate((q, c, r)):
            t.copy_(values(t.shape, device, dtype, seed=10 * i + s))
        new_q = q.clone()
        graph.replay()
        torch.cuda.synchronize()
        got = o.clone(), lse.clone(), q.clone()
        eager_n.add_(1)
        want = step(new_q, c, r, eager_cache, eager_n)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, (*want, new_q))), f"replay {i}"
        assert torch.equal(cache, eager_cache) and torch.equal(n, eager_n), f"replay {i}"


def test_two_graphs_with_one_workspace(device):
    """Replayed one after the other, in either order."""
    sets = [paged(lens, 16, 256, 64, 16, device, seed=i) for i, lens in enumerate(([700, 20], [3, 1500]))]
    ws = torch.empty(1 << 24, dtype=torch.uint8, device=device)
    run = lambda s: rhizome_amd.latent_decode(*s, d_c=256, scale=0.06, workspace=ws)
    want = [tuple(t.clone() for t in run(s)) for s in sets]
    graphs, got = [], []
    for s in sets:
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            got.append(run(s))
    for order in ((0, 1), (1, 0), (0, 0, 1)):
        for t in (t for pair in got for t in pair):
            t.fill_(7.0)
        ws.fill_(255)
        for k in order:
            graphs[k].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w)), order


@both
@pytest.mark.parametrize("B,H", [(1, 1), (1, 7), (2, 4), (3, 3), (1, 31), (4, 8), (3, 11), (1, 40), (5, 13)])
def test_every_head_of_every_sequence(device, dtype, B, H):
    """A head alone, in the same strides, comes out as among the others, whatever
    their number leaves over of eight XCDs and of four heads a group."""
    n, d, dr = 150, 64, 32
    q, kv, r, do = (t.view(B, n, *t.shape[1:]).to(device) for t in make([n] * B, [n] * B, H, d, dr, d, dtype, seed=H))
    k, v = kv[..., :d], kv[..., d:]
    o, lse = rhizome_amd.latent_prefill(q, k, v, r)
    dq, dk, dv, dkr = rhizome_amd.latent_prefill_backward(q, k, v, r, o, lse, do)
    for h in range(H):
        one = [t[:, :, h:h + 1] for t in (q, k, v)]
        oh, lh = rhizome_amd.latent_prefill(*one, r)
        assert torch.equal(oh, o[:, :, h:h + 1]) and torch.equal(lh, lse[:, :, h:h + 1]), h
        got = rhizome_amd.latent_prefill_backward(*one, r, oh, lh, do[:, :, h:h + 1].contiguous())
        for a, b in zip(got, (dq, dk, dv)):
            assert torch.equal(a, b[:, :, h:h + 1]), h
    cu = starts([n] * B).to(device)
    flat = [t.flatten(0, 1) for t in (q, k, v, r)]
    op, lp = rhizome_amd.latent_prefill(*flat, cu_seqlens=cu)
    assert torch.equal(op.view_as(o), o) and torch.equal(lp.view_as(lse), lse)
    got = rhizome_amd.latent_prefill_backward(*flat, op, lp, do.flatten(0, 1), cu_seqlens=cu)
    for a, b in zip(got, (dq, dk, dv, dkr)):
        assert torch.equal(a.view_as(b), b)


def test_tensors_elsewhere(device):
    x, pos = values((4, 2, 8), device), torch.arange(4, dtype=torch.int32, device=device)
    freq = rhizome_amd.rope_frequencies(8, device=device)[0]
    for args in ((x.cpu(), pos, freq), (x, pos.cpu(), freq), (x, pos, freq.cpu())):
        with pytest.raises(ValueError, match="on the GPU"):
            rhizome_amd.rope(*args)
    args = paged([10], 2, 16, 8, 4, device)
    for i in range(4):
        with pytest.raises(ValueError, match="on the GPU"):
            rhizome_amd.latent_decode(*(t.cpu() if k == i else t for k, t in enumerate(args)), d_c=16, scale=1.0)
    q = values((1, 4, 2, 8), device)
    o, lse = rhizome_amd.latent_prefill(q, q, q)
    for i in range(3):
        with pytest.raises(ValueError, match="on the GPU"):
            rhizome_amd.latent_prefill(*(q.cpu() if k == i else q for k in range(3)))
    for i in range(3):
        with pytest.raises(ValueError, match="on the GPU"):
            rhizome_amd.latent_prefill_backward(q, q, q, None, *(t.cpu() if k == i else t for k, t in enumerate((o, lse, q))))


@both
def test_tokens_beyond_32_bits(device, dtype):
    """The last tokens of tensors of more than 2^32 bytes, of a pack whose other tokens are in no sequence."""
    n, H, d_n, d_r, d_v = 140, 64, 128, 64, 128
    total = (5 << 30) // (H * (d_n + d_r) * (2 if dtype == torch.bfloat16 else 4))
    q, kv, r, do = (t.to(device) for t in make([n], [n], H, d_n, d_r, d_v, dtype, seed=19))

    def far(t):
        out = torch.empty(total, *t.shape[1:], dtype=t.dtype, device=device)
        out[-n:] = t
        return out

    long = [far(t) for t in (q, kv, r, do)]
    pos = torch.arange(total, dtype=torch.int32, device=device)
    freq = rhizome_amd.rope_frequencies(d_r, device=device)[0]
    rhizome_amd.rope(long[0], pos, freq, offset=d_n, out=long[0])
    rhizome_amd.rope(q, pos[-n:], freq, offset=d_n, out=q)
    assert torch.equal(long[0][-n:], q)
    cu = torch.tensor([total - n, total], dtype=torch.int32, device=device)
    run = lambda q, kv, r, do, cu: [t[-n:].clone() for t in _both_passes(q, kv, r, do, cu, d_n)]
    got = run(*long, cu)
    want = run(q, kv, r, do, torch.tensor([0, n], dtype=torch.int32, device=device))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def _both_passes(q, kv, r, do, cu, d_n):
    k, v = kv[..., :d_n], kv[..., d_n:]
    o, lse = rhizome_amd.latent_prefill(q, k, v, r, cu_seqlens=cu)
    return o, lse, *rhizome_amd.latent_prefill_backward(q, k, v, r, o, lse, do, cu_seqlens=cu)
