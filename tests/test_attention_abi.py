"""The latent attention's entry points (rhizome_attention.h) without a GPU:
exports, the rotary table, workspace sizes, and every validation error before
any HIP call."""
import ctypes
import math
import os
import subprocess
from ctypes import byref, c_double, c_float, c_size_t

import pytest
import torch
from hypothesis import given, settings, strategies as st

import rhizome_amd
from rhizome_amd import _abi
from rhizome_amd.attention import _token_stride

A = 1 << 40  # fake device addresses, 2^32 apart; never dereferenced
STEP = 1 << 32
INVALID, UNSUPPORTED, WORKSPACE = _abi.ERR_INVALID_ARG, _abi.ERR_UNSUPPORTED, _abi.ERR_WORKSPACE


def _fill(struct, values, pointers, over):
    a = struct()
    for i, name in enumerate(pointers):
        setattr(a, name, A + i * STEP)
    for name, v in {**values, **over}.items():
        setattr(a, name, v)
    return a


def refused(call, a, status, msg):
    assert getattr(_abi.lib(), call)(byref(a), None) == status, _abi.last_error()
    assert msg in _abi.last_error()
    assert getattr(_abi.lib(), call)(None, None) == INVALID


def _size(a, query):
    n = c_size_t(0)
    status = getattr(_abi.lib(), query)(byref(a), byref(n))
    return status, n.value


def test_exports_every_declared_function():
    declared = _abi.declared_functions(_abi.ATTENTION_HEADER)
    assert len(declared) == 8 and "rhz_latent_decode" in declared
    out = subprocess.run(["nm", "-D", "--defined-only", _abi.LIB_PATH], capture_output=True, text=True, check=True)
    exported = {line.split()[-1] for line in out.stdout.splitlines() if line.strip()}
    assert not [f for f in declared if f not in exported]


def test_structs_match_the_header(tmp_path):
    """Sizes and the offset of every field, as a C compiler lays them out."""
    structs = {"rhz_rope_frequency_args": _abi.RopeFrequencyArgs, "rhz_rope_args": _abi.RopeArgs,
               "rhz_latent_append_args": _abi.LatentAppendArgs, "rhz_latent_decode_args": _abi.LatentDecodeArgs,
               "rhz_latent_prefill_args": _abi.LatentPrefillArgs,
               "rhz_latent_prefill_backward_args": _abi.LatentPrefillBackwardArgs}
    lines = ["#include <stddef.h>", "#include <stdio.h>", '#include "rhizome_attention.h"', "int main(void) {"]
    want = []
    for name, struct in structs.items():
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        want.append(ctypes.sizeof(struct))
        for field, _ in struct._fields_:
            lines.append(f'printf("%zu\\n", offsetof({name}, {field}));')
            want.append(getattr(struct, field).offset)
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-I", os.path.dirname(_abi.ATTENTION_HEADER), str(src), "-o", str(tmp_path / "layout")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True)
    assert [int(x) for x in out.stdout.split()] == want


def test_frequencies():
    plain, one = rhizome_amd.rope_frequencies(64, theta=500.0, device="cpu")
    i = torch.arange(32, dtype=torch.float64)
    assert one == 1.0 and torch.allclose(plain, 500.0 ** (-i / 32) / (2 * math.pi), rtol=1e-14, atol=0)
    linear, one = rhizome_amd.rope_frequencies(64, theta=500.0, scaling="linear", factor=8.0, device="cpu")
    assert one == 1.0 and torch.equal(linear, plain / 8.0)
    parts, mag = rhizome_amd.rope_frequencies(64, scaling="by_parts", factor=40.0, trained_length=4096, device="cpu")
    f, _ = rhizome_amd.rope_frequencies(64, device="cpu")
    turns = 4096 * f
    assert abs(mag - (0.1 * math.log(40.0) + 1.0)) < 1e-6
    assert torch.equal(parts[turns > 32], f[turns > 32]) and torch.allclose(parts[turns < 1], f[turns < 1] / 40, rtol=1e-14, atol=0)
    between = (turns > 1) & (turns < 32)
    assert between.any() and bool(((parts < f) & (parts > f / 40))[between].all())


@pytest.mark.parametrize("dim", [-2 ** 32 + 1024, 2 ** 32 + 64, 2 ** 31, -2 ** 31 - 2, 2 ** 31 - 2, 1026, -2, 0, 3])
def test_frequencies_of_a_dimension_out_of_range(dim):
    """Refused, and not taken modulo 2^32: the library would write a table wider than the one it is given."""
    with pytest.raises((ValueError, _abi.GdrError), match="dim|2\\^31"):
        rhizome_amd.rope_frequencies(dim, device="cpu")


FREQ = dict(dim=64, scaling=_abi.ROPE_BY_PARTS, theta=1e4, factor=4.0, trained_length=4096.0, fast=32.0, slow=1.0)


@pytest.mark.parametrize("over,status,msg", [
    (dict(dim=0), INVALID, "dim"), (dict(dim=3), INVALID, "dim"), (dict(dim=-2), INVALID, "dim"),
    (dict(dim=1026), UNSUPPORTED, "dim"), (dict(scaling=3), INVALID, "scaling"), (dict(scaling=-1), INVALID, "scaling"),
    (dict(theta=1.0), INVALID, "theta"), (dict(theta=math.nan), INVALID, "theta"), (dict(theta=math.inf), INVALID, "theta"),
    (dict(factor=0.5), INVALID, "factor"), (dict(factor=math.nan), INVALID, "factor"),
    (dict(trained_length=0.0), INVALID, "trained_length"), (dict(slow=-1.0), INVALID, "slow"),
    (dict(fast=1.0), INVALID, "fast"), (dict(fast=math.inf), INVALID, "fast"), (dict(slow=math.nan), INVALID, "slow"),
])
def test_frequency_validation(over, status, msg):
    a = _fill(_abi.RopeFrequencyArgs, FREQ, (), over)
    turns, mag = (c_double * 1024)(), c_float()
    assert _abi.lib().rhz_rope_frequencies(byref(a), turns, byref(mag)) == status
    assert msg in _abi.last_error()
    good = _fill(_abi.RopeFrequencyArgs, FREQ, (), {})
    assert _abi.lib().rhz_rope_frequencies(byref(good), None, byref(mag)) == INVALID
    assert _abi.lib().rhz_rope_frequencies(byref(good), turns, None) == INVALID
    assert _abi.lib().rhz_rope_frequencies(None, turns, byref(mag)) == INVALID


ROPE = dict(tokens=100, heads=4, dim=96, offset=64, rot=32, dtype=_abi.BF16, magnitude=1.0, x_token_stride=384,
            x_head_stride=96, y_token_stride=384, y_head_stride=96)
ROPE_PTRS = ("x", "positions", "turns", "y")


@pytest.mark.parametrize("over,status,msg", [
    (dict(tokens=-1), INVALID, "tokens"), (dict(heads=0), INVALID, "heads"), (dict(rot=0), INVALID, "rot"),
    (dict(rot=31), INVALID, "rot"), (dict(rot=1026, dim=2000), UNSUPPORTED, "rot"), (dict(offset=-1), INVALID, "channels"),
    (dict(offset=65), INVALID, "channels"), (dict(offset=2 ** 31 - 1), INVALID, "channels"), (dict(dim=0), INVALID, "channels"),
    (dict(dtype=_abi.F64), INVALID, "dtype"), (dict(interleaved=2), INVALID, "interleaved"), (dict(inverse=-1), INVALID, "inverse"),
    (dict(magnitude=math.inf), INVALID, "magnitude"), (dict(x_head_stride=-96), INVALID, "strides"),
    (dict(heads=1 << 20), UNSUPPORTED, "heads * dim"), (dict(y_head_stride=95), INVALID, "overlap"),
    (dict(y_token_stride=383), INVALID, "overlap"), (dict(y_token_stride=0), INVALID, "overlap"),
    (dict(x_token_stride=1 << 62), INVALID, "strides are too large"), (dict(x=A + 1), INVALID, "x is not aligned"),
    (dict(turns=A + 2 * STEP + 4), INVALID, "turns is not aligned"), (dict(y=A + 64), INVALID, "y overlaps x"),
    (dict(y=A + STEP), INVALID, "y overlaps positions"), (dict(y=A, y_token_stride=400), INVALID, "same strides"),
] + [({p: None}, INVALID, f"{p} is NULL") for p in ROPE_PTRS])
def test_rope_validation(over, status, msg):
    refused("rhz_rope", _fill(_abi.RopeArgs, ROPE, ROPE_PTRS, over), status, msg)


APPEND = dict(batch=3, seq_len=2, d_c=512, d_r=64, page_size=16, num_pages=100, max_pages=10, dtype=_abi.BF16, magnitude=1.0,
              eps=1e-6, latent_stride=576, k_rope_stride=576)
APPEND_PTRS = ("latent", "k_rope", "lengths", "page_table", "cache")


@pytest.mark.parametrize("over,status,msg", [
    (dict(batch=0), INVALID, "batch"), (dict(seq_len=-1), INVALID, "seq_len"), (dict(d_c=0), INVALID, "d_c"),
    (dict(d_r=-1), INVALID, "d_r"), (dict(d_c=4097), UNSUPPORTED, "4096"), (dict(d_r=1026), UNSUPPORTED, "1024"),
    (dict(page_size=0), INVALID, "page_size"), (dict(num_pages=0), INVALID, "num_pages"), (dict(max_pages=0), INVALID, "max_pages"),
    (dict(page_size=1 << 20, num_pages=1 << 20), INVALID, "2^31"), (dict(dtype=2), INVALID, "dtype"),
    (dict(interleaved=2), INVALID, "interleaved"), (dict(magnitude=math.nan), INVALID, "magnitude"),
    (dict(eps=-1.0), INVALID, "eps"), (dict(d_r=63, turns=A + 20 * STEP), INVALID, "even"),
    (dict(batch=1 << 16, seq_len=1 << 16), INVALID, "2^31"), (dict(latent_stride=-1), INVALID, "strides"),
    (dict(latent_stride=1 << 62), INVALID, "strides"), (dict(latent=A + 1), INVALID, "latent is not aligned"),
    (dict(turns=A + 20 * STEP + 4), INVALID, "turns is not aligned"), (dict(cache=A), INVALID, "overlaps latent"),
    (dict(norm_scale=A + 4 * STEP + 64), INVALID, "overlaps norm_scale"),
] + [({p: None}, INVALID, f"{p} is NULL") for p in APPEND_PTRS])
def test_append_validation(over, status, msg):
    refused("rhz_latent_append", _fill(_abi.LatentAppendArgs, APPEND, APPEND_PTRS, over), status, msg)


DECODE = dict(batch=4, steps=2, heads=16, d_c=512, d_r=64, page_size=64, num_pages=1000, max_pages=100, dtype=_abi.BF16,
              scale=0.1)
DECODE_PTRS = ("q", "cache", "page_table", "lengths", "o")


@pytest.mark.parametrize("over,status,msg", [
    (dict(batch=0), INVALID, "batch"), (dict(steps=0), INVALID, "steps"), (dict(heads=0), INVALID, "heads"),
    (dict(steps=65), UNSUPPORTED, "steps"), (dict(heads=1025), UNSUPPORTED, "heads"), (dict(d_c=513), UNSUPPORTED, "d_c"),
    (dict(d_r=65), UNSUPPORTED, "d_r"), (dict(d_c=0), INVALID, "d_c"), (dict(d_r=-1), INVALID, "d_r"),
    (dict(page_size=-1), INVALID, "page_size"), (dict(num_pages=1 << 30), INVALID, "2^31"), (dict(dtype=3), INVALID, "dtype"),
    (dict(scale=0.0), INVALID, "scale"), (dict(scale=-1.0), INVALID, "scale"), (dict(scale=math.nan), INVALID, "scale"),
    (dict(scale=math.inf), INVALID, "scale"), (dict(batch=1 << 22, steps=64, heads=1024), INVALID, "2^31"),
    (dict(cache=A + STEP + 1), INVALID, "cache is not aligned"), (dict(o=A), INVALID, "o overlaps q"),
    (dict(lse=A + 3 * STEP), INVALID, "overlaps"), (dict(), WORKSPACE, "workspace is NULL"),
    (dict(workspace=A + 30 * STEP, workspace_bytes=64), WORKSPACE, "needed"),
    (dict(workspace=A + 30 * STEP + 128, workspace_bytes=1 << 31), WORKSPACE, "256-byte"),
    (dict(workspace=A + STEP, workspace_bytes=1 << 31), INVALID, "overlaps"),
] + [({p: None}, INVALID, f"{p} is NULL") for p in DECODE_PTRS])
def test_decode_validation(over, status, msg):
    refused("rhz_latent_decode", _fill(_abi.LatentDecodeArgs, DECODE, DECODE_PTRS, over), status, msg)


def test_decode_with_more_rows_than_a_grid_can_join():
    """Refused before the first of its two kernels: 65537 sequences of 128 heads, 512 channels and up to two splits."""
    far = {name: A + (i << 37) for i, name in enumerate((*DECODE_PTRS, "workspace"))}
    a = _fill(_abi.LatentDecodeArgs, DECODE, (), dict(batch=65537, steps=1, heads=128, page_size=256, max_pages=1,
                                                      workspace_bytes=1 << 36, **far))
    assert _abi.lib().rhz_latent_decode(byref(a), None) == _abi.ERR_HIP and "invalid configuration" in _abi.last_error()


def test_decode_workspace_size():
    query = "rhz_latent_decode_workspace_size"
    make = lambda **over: _fill(_abi.LatentDecodeArgs, DECODE, DECODE_PTRS, over)
    rows = 4 * 2 * 16
    status, n = _size(make(), query)
    # a part for every split: an fp32 row of o, a maximum and a sum
    assert status == _abi.OK and n % (rows * 514 * 4) == 0 and 2 <= n // (rows * 514 * 4) <= 128
    assert _size(make(max_pages=1 << 24, page_size=1 << 7, num_pages=100), query)[1] >= n  # a table of 2^31 rows
    assert _size(make(max_pages=1), query) == (_abi.OK, 0)  # one split
    assert _abi.lib().rhz_latent_decode_workspace_size(byref(make()), None) == INVALID
    assert _size(make(heads=0), query)[0] == INVALID


PREFILL = dict(batch=2, seq_len=100, seq_len_k=100, heads=4, d_n=128, d_r=64, d_v=128, dtype=_abi.BF16, causal=1, scale=0.1,
               q_token_stride=768, q_head_stride=192, k_token_stride=1024, k_head_stride=256, v_token_stride=1024,
               v_head_stride=256, k_rope_stride=64)
PREFILL_PTRS = ("q", "k", "v", "k_rope", "o", "lse")
PREFILL_REFUSALS = [
    (dict(batch=0), INVALID, "batch"), (dict(seq_len=-1), INVALID, "seq_len"), (dict(seq_len_k=-1), INVALID, "seq_len"),
    (dict(heads=0), INVALID, "heads"), (dict(d_n=0), INVALID, "d_n"), (dict(d_r=-1), INVALID, "d_r"), (dict(d_v=0), INVALID, "d_v"),
    (dict(d_n=129), UNSUPPORTED, "192"), (dict(d_r=65), UNSUPPORTED, "192"), (dict(d_v=129), UNSUPPORTED, "128"),
    (dict(d_n=2 ** 31 - 1, d_r=2 ** 31 - 1), UNSUPPORTED, "192"), (dict(dtype=2), INVALID, "dtype"),
    (dict(causal=2), INVALID, "causal"), (dict(scale=0.0), INVALID, "scale"), (dict(scale=math.inf), INVALID, "scale"),
    (dict(cu_seqlens_k=A + 20 * STEP), INVALID, "cu_seqlens_k without"),
    (dict(cu_seqlens=A + 20 * STEP, seq_len_k=99), INVALID, "differ"), (dict(batch=1 << 20, seq_len=1 << 20), INVALID, "2^31"),
    (dict(q_head_stride=-1), INVALID, "strides"), (dict(k_token_stride=(1 << 22) + 1), UNSUPPORTED, "apart"),
    (dict(v_head_stride=1 << 62), INVALID, "too large"), (dict(heads=1 << 16), UNSUPPORTED, "apart"),
    (dict(q=A + 1), INVALID, "q is not aligned"), (dict(o=A + 128), INVALID, "o overlaps q"),
    (dict(lse=A + STEP), INVALID, "lse overlaps k"),
]


@pytest.mark.parametrize("over,status,msg", PREFILL_REFUSALS + [({p: None}, INVALID, f"{p} is NULL") for p in PREFILL_PTRS])
def test_prefill_validation(over, status, msg):
    refused("rhz_latent_prefill", _fill(_abi.LatentPrefillArgs, PREFILL, PREFILL_PTRS, over), status, msg)


GRAD_PTRS = ("grad_o", "grad_q", "grad_k", "grad_v", "grad_k_rope")


def _backward(over, forward=None):
    a = _abi.LatentPrefillBackwardArgs()
    a.forward = _fill(_abi.LatentPrefillArgs, PREFILL, PREFILL_PTRS, forward or {})
    for i, name in enumerate(GRAD_PTRS):
        setattr(a, name, A + (30 + i) * STEP)
    for name, v in over.items():
        setattr(a, name, v)
    return a


@pytest.mark.parametrize("over,status,msg", PREFILL_REFUSALS[:-2] + [({p: None}, INVALID, f"{p} is NULL") for p in PREFILL_PTRS])
def test_backward_validates_the_forward_call(over, status, msg):
    refused("rhz_latent_prefill_backward", _backward({}, over), status, msg)


@pytest.mark.parametrize("over,status,msg", [
    (dict(grad_q=A), INVALID, "grad_q overlaps q"), (dict(grad_k=A + 5 * STEP), INVALID, "overlaps lse"),
    (dict(grad_v=A + 33 * STEP + 64, grad_k=A + 33 * STEP), INVALID, "overlaps"),
    (dict(grad_o=A + 30 * STEP + 1), INVALID, "grad_o is not aligned"), (dict(), WORKSPACE, "workspace is NULL"),
    (dict(workspace=A + 50 * STEP, workspace_bytes=64), WORKSPACE, "needed"),
    (dict(workspace=A + 50 * STEP + 16, workspace_bytes=1 << 30), WORKSPACE, "256-byte"),
    (dict(workspace=A, workspace_bytes=1 << 30), INVALID, "overlaps"),
] + [({p: None}, INVALID, f"{p} is NULL") for p in GRAD_PTRS])
def test_backward_validation(over, status, msg):
    refused("rhz_latent_prefill_backward", _backward(over), status, msg)


def test_backward_workspace_size():
    query = "rhz_latent_prefill_backward_workspace_size"
    status, n = _size(_backward({}), query)
    rows = 200 * 4
    assert status == _abi.OK and rows * (2 + 64) * 4 <= n <= rows * (2 + 64) * 4 + 3 * 256
    assert _size(_backward({}, dict(d_r=0)), query)[1] <= rows * 2 * 4 + 3 * 256
    assert _size(_backward({}, dict(batch=1, seq_len=1 << 22, seq_len_k=1 << 22, heads=64)), query)[1] > 1 << 36
    assert _size(_backward({}, dict(heads=0)), query)[0] == INVALID
    assert _abi.lib().rhz_latent_prefill_backward_workspace_size(byref(_backward({})), None) == INVALID


def test_calls_of_nothing():
    none = lambda ptrs: {p: None for p in ptrs}
    lib = _abi.lib()
    assert lib.rhz_rope(byref(_fill(_abi.RopeArgs, ROPE, (), dict(tokens=0))), None) == _abi.OK
    assert lib.rhz_latent_append(byref(_fill(_abi.LatentAppendArgs, APPEND, (), dict(seq_len=0))), None) == _abi.OK
    assert lib.rhz_latent_prefill(byref(_fill(_abi.LatentPrefillArgs, PREFILL, (), dict(seq_len=0))), None) == _abi.OK
    empty = _backward(none(GRAD_PTRS), dict(none(PREFILL_PTRS), seq_len=0, seq_len_k=0))
    assert lib.rhz_latent_prefill_backward(byref(empty), None) == _abi.OK


INT = st.sampled_from([-2 ** 31, -1, 0, 1, 2, 7, 64, 192, 1 << 16, 1 << 22, 2 ** 31 - 1])
LONG = st.sampled_from([-1, 0, 1, 192, 1 << 22, 1 << 40, 2 ** 63 - 1])


@settings(max_examples=300, deadline=None)
@given(st.data())
def test_any_sizes_end_in_a_status(data):
    """Sizes of any kind, with every pointer missing: refused (or nothing to do), never a crash."""
    ints = lambda struct, names: {n: data.draw(LONG if n.endswith("stride") else INT) for n in names}
    for call, struct, values in (("rhz_rope", _abi.RopeArgs, ROPE), ("rhz_latent_append", _abi.LatentAppendArgs, APPEND),
                                 ("rhz_latent_decode", _abi.LatentDecodeArgs, DECODE),
                                 ("rhz_latent_prefill", _abi.LatentPrefillArgs, PREFILL)):
        names = [n for n, v in values.items() if isinstance(v, int)]
        over = ints(struct, data.draw(st.lists(st.sampled_from(names), max_size=4, unique=True)))
        a = _fill(struct, values, (), over)
        assert getattr(_abi.lib(), call)(byref(a), None) in (_abi.OK, INVALID, UNSUPPORTED, WORKSPACE)
        if call == "rhz_latent_decode":
            _size(a, "rhz_latent_decode_workspace_size")
        if call == "rhz_latent_prefill":
            b = _abi.LatentPrefillBackwardArgs()
            b.forward = a
            assert _abi.lib().rhz_latent_prefill_backward(byref(b), None) in (_abi.OK, INVALID, UNSUPPORTED, WORKSPACE)
            _size(b, "rhz_latent_prefill_backward_workspace_size")


@pytest.mark.parametrize("call,message", [
    (lambda t, i: rhizome_amd.rope(t(2, 3, 8, 4, 2), i(2, 3, 8), t(2).double()), "x must be"),
    (lambda t, i: rhizome_amd.rope(t(3, 4, 8).half(), i(3), t(2).double()), "x must be"),
    (lambda t, i: rhizome_amd.rope(t(3, 4, 8), i(4), t(2).double()), "positions"),
    (lambda t, i: rhizome_amd.rope(t(3, 4, 8), i(3).long(), t(2).double()), "positions"),
    (lambda t, i: rhizome_amd.rope(t(3, 4, 8), i(3), t(2)), "frequencies"),
    (lambda t, i: rhizome_amd.rope(t(3, 4, 8), i(3), t(2).double(), out=t(3, 4, 6)), "out"),
    (lambda t, i: rhizome_amd.rope(t(3, 8, 4).transpose(1, 2), i(3), t(2).double()), "dense"),
    (lambda t, i: rhizome_amd.rope(t(2, 4, 3, 8).transpose(1, 2), i(2, 3), t(2).double()), "evenly spaced"),
    (lambda t, i: rhizome_amd.latent_append(t(2, 1, 8), t(2, 1, 4), t(5, 4, 11), i(2, 3), i(2)), "cache"),
    (lambda t, i: rhizome_amd.latent_append(t(2, 8), t(2, 4), t(5, 4, 12), i(2, 3), i(2)), "latent"),
    (lambda t, i: rhizome_amd.latent_append(t(2, 1, 8), t(2, 2, 4), t(5, 4, 12), i(2, 3), i(2)), "k_rope"),
    (lambda t, i: rhizome_amd.latent_append(t(3, 1, 8), t(3, 1, 4), t(5, 4, 12), i(2, 3), i(2)), "sequences"),
    (lambda t, i: rhizome_amd.latent_append(t(2, 1, 8), t(2, 1, 4), t(5, 4, 12), i(2, 3), i(3)), "lengths"),
    (lambda t, i: rhizome_amd.latent_append(t(2, 1, 8), t(2, 1, 4), t(5, 4, 12), i(2, 3).long(), i(2)), "page_table"),
    (lambda t, i: rhizome_amd.latent_append(t(2, 1, 8), t(2, 1, 4), t(5, 4, 12), i(2, 3), i(2), frequencies=t(3).double()),
     "frequencies"),
    (lambda t, i: rhizome_amd.latent_append(t(2, 1, 8), t(2, 1, 4), t(5, 4, 12), i(2, 3), i(2), norm_scale=t(9)), "norm_scale"),
    (lambda t, i: rhizome_amd.latent_append(t(7, 8), t(7, 4), t(5, 4, 12), i(2, 3), i(2), cu_seqlens=i(2)), "cu_seqlens"),
    (lambda t, i: rhizome_amd.latent_decode(t(2, 1, 4, 12), t(5, 4, 13), i(2, 3), i(2), d_c=8, scale=1.0), "cache"),
    (lambda t, i: rhizome_amd.latent_decode(t(3, 1, 4, 12), t(5, 4, 12), i(2, 3), i(2), d_c=8, scale=1.0), "sequences"),
    (lambda t, i: rhizome_amd.latent_decode(t(2, 1, 4, 12), t(5, 4, 12), i(2, 3), i(2), d_c=13, scale=1.0), "d_c"),
    (lambda t, i: rhizome_amd.latent_decode(t(2, 1, 4, 12), t(5, 4, 12), i(2, 3), i(2), d_c=8, scale=1.0, out=t(2, 1, 4, 12)), "out"),
    (lambda t, i: rhizome_amd.latent_decode(t(2, 4, 12), t(5, 4, 12), i(2, 3), i(2), d_c=8, scale=1.0), "q must be"),
    (lambda t, i: rhizome_amd.latent_prefill(t(2, 5, 4, 8), t(2, 5, 4, 6), t(2, 5, 4, 8)), "k_rope"),
    (lambda t, i: rhizome_amd.latent_prefill(t(2, 5, 4, 8), t(2, 5, 4, 6), t(2, 5, 4, 8), t(2, 5, 3)), "k_rope"),
    (lambda t, i: rhizome_amd.latent_prefill(t(2, 5, 4, 8), t(2, 5, 3, 8), t(2, 5, 3, 8)), "do not match"),
    (lambda t, i: rhizome_amd.latent_prefill(t(2, 5, 4, 8), t(2, 5, 4, 9), t(2, 5, 4, 8)), "do not match"),
    (lambda t, i: rhizome_amd.latent_prefill(t(2, 5, 4, 8), t(3, 5, 4, 8), t(3, 5, 4, 8)), "batch"),
    (lambda t, i: rhizome_amd.latent_prefill(t(9, 4, 8), t(9, 4, 8), t(9, 4, 8)), "cu_seqlens"),
    (lambda t, i: rhizome_amd.latent_prefill(t(9, 4, 8), t(9, 4, 8), t(9, 4, 8), cu_seqlens=i(3).long()), "cu_seqlens"),
    (lambda t, i: rhizome_amd.latent_prefill(t(9, 4, 8), t(9, 4, 8), t(9, 4, 8), cu_seqlens=i(3), cu_seqlens_k=i(4)), "cu_seqlens_k"),
    (lambda t, i: rhizome_amd.latent_prefill(t(2, 5, 4, 8), t(2, 5, 4, 8), t(2, 5, 4, 8), cu_seqlens_k=i(3)), "cu_seqlens_k"),
    (lambda t, i: rhizome_amd.latent_prefill(t(2, 5, 4, 8), t(2, 5, 4, 8), t(2, 5, 4, 8).double()), "one dtype"),
    (lambda t, i: rhizome_amd.latent_prefill(t(2, 5, 4, 8), t(2, 5, 4, 8), t(2, 5, 4, 8), out=t(2, 5, 4, 9)), "out"),
    (lambda t, i: rhizome_amd.latent_prefill_backward(t(2, 5, 4, 8), t(2, 5, 4, 8), t(2, 5, 4, 8), None, t(2, 5, 4, 8),
                                                      t(2, 5, 4), t(2, 5, 4, 7)), "do must be"),
    (lambda t, i: rhizome_amd.latent_prefill_backward(t(2, 5, 4, 8), t(2, 5, 4, 8), t(2, 5, 4, 8), None, t(2, 5, 4, 8),
                                                      t(2, 5, 3), t(2, 5, 4, 8)), "lse must be"),
])
def test_python_refusals(call, message):
    t = lambda *shape: torch.zeros(shape)
    i = lambda *shape: torch.zeros(shape, dtype=torch.int32)
    with pytest.raises((ValueError, RuntimeError), match=message):
        call(t, i)


def test_rust_bindings_agree():
    """The Rust declarations written out for maintainers have the header's constants, fields and parameters."""
    import re

    import test_integration_bindings as T

    to_rust = lambda t: T.c_to_rust(t).replace("double", "f64")
    text = T.strip_c_comments(open(_abi.ATTENTION_HEADER).read())
    text = re.sub(r"int64_t (\w+), (\w+);", r"int64_t \1; int64_t \2;", text)
    doc = open(os.path.join(_abi.ROOT, "INTEGRATION.md")).read()
    start = doc.index("```rust", doc.index("### src/sys_attention.rs"))
    rust = doc[start:doc.index("```", start + 7)]
    structs, found = {}, {}
    for name, body in re.findall(r"typedef struct (\w+) \{(.*?)\} \1;", text, flags=re.S):
        decls = [re.fullmatch(r"(.+?)\s*(\w+)", " ".join(d.split())) for d in body.split(";") if d.strip()]
        structs[name] = [(m.group(2), to_rust(m.group(1))) for m in decls]
    for name, body in re.findall(r"#\[repr\(C\)\]\s*pub struct (\w+) \{(.*?)\}", rust, flags=re.S):
        found[name] = [re.fullmatch(r"pub (\w+): (.+)", " ".join(f.split())).groups() for f in body.split(",") if f.strip()]
    assert found == structs and len(structs) == 6
    consts = dict(re.findall(r"(RHZ_ROPE_\w+)\s*=\s*(\d+)", text))
    assert dict(re.findall(r"pub const (RHZ_\w+): i32 = (\d+);", rust)) == consts and len(consts) == 3
    declared = re.findall(r"rhz_status\s+(rhz_\w+)\(([^)]*)\);", text)
    assert len(declared) == 8
    for name, params in declared:
        m = re.search(r"pub fn %s\(([^)]*)\)\s*->\s*i32;" % name, rust)
        assert m, name
        want = [to_rust(re.fullmatch(r"(.+?)\s*(\w+)", " ".join(x.split())).group(1)) for x in params.split(",")]
        assert [" ".join(x.split()).split(": ")[1] for x in m.group(1).split(",")] == want, name


def test_packed_arguments_are_the_structures():
    """What the front end lays out is what filling in the Structure gives."""
    for name in ("Rope", "LatentAppend", "LatentDecode", "LatentPrefill", "LatentPrefillBackward"):
        struct = getattr(_abi, name + "Args")
        flat = []
        for field, t in struct._fields_:
            flat += [(field, f, u) for f, u in t._fields_] if hasattr(t, "_fields_") else [(None, field, t)]
        a, values = struct(), []
        for i, (outer, field, t) in enumerate(flat):
            v = 0.5 * i if t is c_float else 3 * i + 1
            setattr(getattr(a, outer) if outer else a, field, v)
            values.append(v)
        pack = getattr(_abi, "pack_" + {"Rope": "rope", "LatentAppend": "latent_append", "LatentDecode": "latent_decode",
                                        "LatentPrefill": "latent_prefill",
                                        "LatentPrefillBackward": "latent_prefill_backward"}[name])
        got, want = pack(*values), bytes(a)
        assert len(got) == len(want)
        for outer, field, t in flat:  # padding may differ
            at = getattr(struct, outer).offset + getattr(dict(struct._fields_)[outer], field).offset if outer else \
                getattr(struct, field).offset
            assert got[at:at + ctypes.sizeof(t)] == want[at:at + ctypes.sizeof(t)], (name, field)


def test_token_strides():
    """The distance of a token from the next one, which a single token does not have, whatever its view says."""
    far = torch.empty(0).as_strided  # nothing is read
    stride = lambda shape, strides, batch, n: _token_stride("x", far(shape, strides), batch, n)
    big = 1 << 30
    for shape, strides, batch, n in (((1, 2, 0), (big, 8, 1), None, 1), ((1, 1, 2, 0), (big, big, 8, 1), 1, 1),
                                     ((1, 1, 2, 0), (big, 16, 8, 1), 1, 1), ((0, 2, 0), (big, 8, 1), None, 0),
                                     ((3, 0, 2, 0), (big, 16, 8, 1), 3, 0)):
        assert stride(shape, strides, batch, n) == 0
    assert stride((5, 2, 0), (40, 8, 1), None, 5) == 40
    assert stride((3, 5, 2, 0), (200, 40, 8, 1), 3, 5) == 40
    assert stride((1, 5, 2, 0), (big, 40, 8, 1), 1, 5) == 40
    assert stride((3, 1, 2, 0), (200, 40, 8, 1), 3, 1) == 200
    with pytest.raises(ValueError, match="evenly"):
        stride((3, 5, 2, 0), (300, 40, 8, 1), 3, 5)
    with pytest.raises(ValueError, match="dense"):
        _token_stride("x", torch.empty(5, 2, 8)[..., ::2], None, 5)
