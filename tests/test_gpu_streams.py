"""Calls on a stream other than the current one: what the front end allocates
for them is free on that stream, not only on the current one."""
import pytest
import torch

import rhizome_amd

pytestmark = pytest.mark.gpu
ROWS, DIM = 1 << 14, 1024


def values(shape, device, dtype=torch.float32, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float32).to(device, dtype)


def delta(device):
    q, k, v, do = (values((1, 1 << 14, 8, 128), device, torch.bfloat16, s) for s in range(4))
    g, beta = -torch.rand((2, 1, 1 << 14, 8), generator=torch.Generator().manual_seed(5)).to(device)
    return dict(q=q, k=torch.nn.functional.normalize(k, dim=-1), v=v, g=g.contiguous(), beta=-beta), do


# name: the call on a stream, and the elements of its output that the test is about
def cases(device):
    x, w = values((ROWS, DIM), device), values((DIM,), device, seed=1)
    d, do = delta(device)
    return {
        "layernorm": lambda s: rhizome_amd.layernorm(x, w, stream=s),
        "layernorm_backward": lambda s: rhizome_amd.layernorm_backward(x, x, w, stream=s)[0],
        "rmsnorm_heads_backward": lambda s: rhizome_amd.rmsnorm_heads_backward(x, x, w, stream=s)[0],
        "rmsnorm_heads": lambda s: rhizome_amd.rmsnorm_heads(x, w, stream=s),
        "prefill": lambda s: rhizome_amd.prefill(**d, stream=s)[0],
        "prefill_backward": lambda s: rhizome_amd.prefill_backward(**d, do=do, stream=s)[0],
    }


@pytest.mark.parametrize("name", ["layernorm", "layernorm_backward", "rmsnorm_heads_backward", "rmsnorm_heads", "prefill",
                                  "prefill_backward"])
def test_memory_that_the_current_stream_still_reads(device, name):
    """A tensor let go on the current stream while a copy of it waits there: its
    memory is the only free block of an output's size, and is not taken up."""
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


@pytest.mark.parametrize("name", ["layernorm", "prefill", "prefill_backward"])
def test_results_and_workspaces_let_go(device, name):
    """Results dropped while the current stream still reads them, and a
    workspace while the call still runs: later allocations leave both alone."""
    run, side = cases(device)[name], torch.cuda.Stream()
    want = run(None)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    got = run(side)
    junk = [torch.full((1 << 22,), 3.0, device=device) for _ in range(32)]  # on the current stream
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda._sleep(20_000_000)
    copy = got.clone()
    del got
    again = [run(side) for _ in range(3)]
    torch.cuda.synchronize()
    assert len(junk) == 32 and torch.equal(copy, want) and all(torch.equal(x, want) for x in again)
