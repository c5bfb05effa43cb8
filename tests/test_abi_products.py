"""Sizes whose products leave 64 bits are refused by every entry point, whatever
is left of the product: checked on the CPU, before anything reaches the GPU."""
from ctypes import byref

import pytest

from rhizome_amd import _abi

A, STEP = 1 << 32, 1 << 40  # made-up device addresses, far apart
TOP = 2**31 - 1


def _gpu_visible() -> bool:
    import torch

    return torch.cuda.device_count() > 0


@pytest.mark.skipif(_gpu_visible(), reason="made-up device addresses: CPU only")
@pytest.mark.parametrize("name,struct,sizes,says", [
    # (2^31 - 1)^2 * 256 = 256 - 2^40 modulo 2^64
    ("rhz_gdr_prepare", _abi.PrepareArgs, dict(tokens=TOP, heads=TOP, d_k=256, q_scale=1.0), "tokens * heads * d_k"),
    ("rhz_causal_conv1d", _abi.Conv1dArgs, dict(batch=TOP, seq_len=TOP, channels=4), "tokens * channels"),
    ("rhz_gdr_multistep", _abi.MultistepArgs, dict(batch=TOP, steps=4, heads=TOP, d_k=64, d_v=64),
     "batch * steps * heads"),
    ("rhz_gdr_conv_prepare", _abi.ConvPrepareArgs,
     dict(batch=TOP, seq_len=TOP, heads=TOP, d_k=64, d_v=64, q_scale=1.0), "tokens * channels"),
    ("rhz_gdr_prefill", _abi.PrefillArgs, dict(batch=TOP, seq_len=TOP, heads=4, d_k=64, d_v=64, chunk=64),
     "tokens * heads"),
    ("rhz_gdr_prefill_backward", _abi.PrefillBackwardArgs, dict(batch=TOP, seq_len=TOP, heads=4, d_k=64, d_v=64),
     "tokens * heads"),
    ("rhz_gdr_conv_prepare_backward", _abi.ConvPrepareBackwardArgs,
     dict(batch=TOP, seq_len=TOP, heads=TOP, d_k=64, d_v=64, q_scale=1.0), "tokens * channels"),
])
def test_products_beyond_64_bits(name, struct, sizes, says):
    a, at = struct(), A
    for field, kind in struct._fields_:
        if field in sizes:
            setattr(a, field, sizes[field])
        elif kind.__name__ == "c_void_p" and field not in ("cu_seqlens", "stream"):
            setattr(a, field, at)
            at += STEP
    a.dtype = _abi.F32
    status = getattr(_abi.lib(), name)(byref(a), None)
    message = _abi.last_error()
    assert status == _abi.ERR_INVALID_ARG and says in message, (status, message)
