"""The training entry points (rhizome_train.h) without a GPU: exports,
workspace sizes, and every validation error before any HIP call."""
import os
import re
import subprocess
from ctypes import byref, c_size_t

import pytest
from hypothesis import given, settings, strategies as st

from rhizome_amd import _abi

A = 1 << 40  # fake device addresses, 2^32 apart; never dereferenced
STEP = 1 << 32


def _gpu_visible() -> bool:
    try:
        import torch

        return torch.cuda.device_count() > 0
    except Exception:
        return False


def _fill(struct, values, pointers, over):
    a = struct()
    for i, name in enumerate(pointers):
        setattr(a, name, A + i * STEP)
    for name, v in {**values, **over}.items():
        setattr(a, name, v)
    return a


BACKWARD = dict(batch=4, seq_len=4096, heads=16, d_k=128, d_v=128, dtype=_abi.BF16, gate_kind=_abi.GATE_LOG_ALPHA)
BACKWARD_PTRS = ("q", "k", "v", "gate", "beta", "grad_o", "grad_q", "grad_k", "grad_v", "grad_gate", "grad_beta")


def _backward(**over):
    return _fill(_abi.PrefillBackwardArgs, BACKWARD, BACKWARD_PTRS, over)


def _size(a, query):
    n = c_size_t(0)
    status = getattr(_abi.lib(), query)(byref(a), byref(n))
    return status, n.value


def test_exports_every_declared_function():
    declared = _abi.declared_functions(_abi.TRAIN_HEADER)
    assert "rhz_gdr_prefill_backward" in declared
    out = subprocess.run(["nm", "-D", "--defined-only", _abi.LIB_PATH], capture_output=True, text=True, check=True)
    exported = {line.split()[-1] for line in out.stdout.splitlines() if line.strip()}
    assert not [f for f in declared if f not in exported]


def test_backward_workspace_size():
    query = "rhz_gdr_prefill_backward_workspace_size"
    status, full = _size(_backward(), query)
    # the states on either side of every (chunk, head): 64 KiB at d = 128 in bf16
    assert status == _abi.OK and full >= 4 * 64 * 16 * 64 * 1024
    assert _size(_backward(seq_len=0), query)[1] < full
    status, packed = _size(_backward(cu_seqlens=A, seq_len=4 * 4096), query)
    assert status == _abi.OK and packed > full  # a partial chunk for every sequence
    # sizes beyond 32 bits
    assert _size(_backward(batch=1, seq_len=1 << 20, heads=64), query)[1] > 1 << 36
    assert _abi.lib().rhz_gdr_prefill_backward_workspace_size(byref(_backward()), None) == _abi.ERR_INVALID_ARG


@pytest.mark.parametrize("over,status,msg", [
    (dict(batch=0), _abi.ERR_INVALID_ARG, "batch"),
    (dict(seq_len=-1), _abi.ERR_INVALID_ARG, "seq_len"),
    (dict(heads=0), _abi.ERR_INVALID_ARG, "heads"),
    (dict(d_k=0), _abi.ERR_INVALID_ARG, "d_k"),
    (dict(d_v=0), _abi.ERR_INVALID_ARG, "d_v"),
    (dict(d_k=129), _abi.ERR_UNSUPPORTED, "d_k"),
    (dict(d_v=1025), _abi.ERR_UNSUPPORTED, "d_v"),
    (dict(dtype=_abi.F64), _abi.ERR_INVALID_ARG, "dtype"),
    (dict(gate_kind=2), _abi.ERR_INVALID_ARG, "gate_kind"),
    (dict(batch=70000, seq_len=70000), _abi.ERR_INVALID_ARG, "2^31"),
    (dict(q=A + 1), _abi.ERR_INVALID_ARG, "q is not aligned"),
    (dict(beta=A + 4 * STEP + 2), _abi.ERR_INVALID_ARG, "beta is not aligned"),
    (dict(grad_q=A), _abi.ERR_INVALID_ARG, "grad_q overlaps q"),
    (dict(grad_k=A + 8 * STEP - 64), _abi.ERR_INVALID_ARG, "overlaps"),
    (dict(grad_final_state=A, grad_initial_state=A + 40 * STEP), _abi.ERR_WORKSPACE, "workspace is NULL"),
    (dict(grad_final_state=A + 40 * STEP, grad_initial_state=A + 40 * STEP), _abi.ERR_INVALID_ARG, "overlaps"),
    (dict(workspace=A + 50 * STEP, workspace_bytes=1024), _abi.ERR_WORKSPACE, "needed"),
    (dict(workspace=A + 50 * STEP + 128, workspace_bytes=1 << 31), _abi.ERR_WORKSPACE, "256-byte"),
    (dict(workspace=A, workspace_bytes=1 << 31), _abi.ERR_INVALID_ARG, "overlaps"),
] + [({p: None}, _abi.ERR_INVALID_ARG, f"{p} is NULL") for p in BACKWARD_PTRS])
def test_backward_validation(over, status, msg):
    assert _abi.lib().rhz_gdr_prefill_backward(byref(_backward(**over)), None) == status, _abi.last_error()
    assert msg in _abi.last_error()


def test_backward_of_nothing():
    a = _backward(seq_len=0, **{p: None for p in BACKWARD_PTRS})
    assert _abi.lib().rhz_gdr_prefill_backward(byref(a), None) == _abi.OK
    assert _abi.lib().rhz_gdr_prefill_backward(None, None) == _abi.ERR_INVALID_ARG


CONV = dict(batch=2, seq_len=100, heads=4, d_k=64, d_v=64, dtype=_abi.BF16, q_scale=8.0)
CONV_PTRS = ("x", "weight", "beta_logit", "alpha_logit", "a_log", "grad_q", "grad_k", "grad_v", "grad_beta", "grad_g",
             "grad_x", "grad_weight", "grad_beta_logit", "grad_alpha_logit", "grad_a_log")


@pytest.mark.parametrize("over,status,msg", [
    (dict(batch=0), _abi.ERR_INVALID_ARG, "batch"),
    (dict(seq_len=-1), _abi.ERR_INVALID_ARG, "seq_len"),
    (dict(heads=0), _abi.ERR_INVALID_ARG, "heads"),
    (dict(d_k=0), _abi.ERR_INVALID_ARG, "d_k"),
    (dict(d_k=24), _abi.ERR_UNSUPPORTED, "power of two"),
    (dict(d_v=12), _abi.ERR_UNSUPPORTED, "multiples of 8"),
    (dict(d_k=1024), _abi.ERR_UNSUPPORTED, "exceed"),
    (dict(dtype=_abi.F64), _abi.ERR_INVALID_ARG, "dtype"),
    (dict(q_scale=float("nan")), _abi.ERR_INVALID_ARG, "q_scale"),
    (dict(seq_len=1 << 24), _abi.ERR_INVALID_ARG, "2^31"),
    (dict(x=A + 8), _abi.ERR_INVALID_ARG, "x is not aligned"),
    (dict(grad_v=A + 7 * STEP + 8), _abi.ERR_INVALID_ARG, "grad_v is not aligned"),
    (dict(grad_x=A + 5 * STEP), _abi.ERR_INVALID_ARG, "overlaps"),
    (dict(grad_weight=A + STEP), _abi.ERR_INVALID_ARG, "overlaps"),
    (dict(), _abi.ERR_WORKSPACE, "workspace is NULL"),
    (dict(workspace=A + 50 * STEP, workspace_bytes=64), _abi.ERR_WORKSPACE, "needed"),
    (dict(workspace=A + 50 * STEP + 16, workspace_bytes=1 << 30), _abi.ERR_WORKSPACE, "256-byte"),
] + [({p: None}, _abi.ERR_INVALID_ARG, f"{p} is NULL") for p in CONV_PTRS])
def test_conv_prepare_backward_validation(over, status, msg):
    a = _fill(_abi.ConvPrepareBackwardArgs, CONV, CONV_PTRS, over)
    assert _abi.lib().rhz_gdr_conv_prepare_backward(byref(a), None) == status, _abi.last_error()
    assert msg in _abi.last_error()
    assert _abi.lib().rhz_gdr_conv_prepare_backward(None, None) == _abi.ERR_INVALID_ARG


NORM = dict(rows=100, dim=128, dtype=_abi.BF16, eps=1e-5)
NORM_PTRS = ("grad_y", "x", "weight", "grad_x", "grad_weight")


@pytest.mark.parametrize("over,status,msg", [
    (dict(rows=-1), _abi.ERR_INVALID_ARG, "rows"),
    (dict(dim=0), _abi.ERR_INVALID_ARG, "dim"),
    (dict(dim=8193), _abi.ERR_UNSUPPORTED, "dim"),
    (dict(dtype=2), _abi.ERR_INVALID_ARG, "dtype"),
    (dict(eps=-1.0), _abi.ERR_INVALID_ARG, "eps"),
    (dict(eps=float("nan")), _abi.ERR_INVALID_ARG, "eps"),
    (dict(rows=1 << 25), _abi.ERR_INVALID_ARG, "2^31"),
    (dict(x=A + STEP + 1), _abi.ERR_INVALID_ARG, "x is not aligned"),
    (dict(grad_x=A), _abi.ERR_INVALID_ARG, "overlaps"),
    (dict(), _abi.ERR_WORKSPACE, "workspace is NULL"),
    (dict(workspace=A + 50 * STEP, workspace_bytes=64), _abi.ERR_WORKSPACE, "needed"),
] + [({p: None}, _abi.ERR_INVALID_ARG, f"{p} is NULL") for p in NORM_PTRS])
def test_norm_backward_validation(over, status, msg):
    a = _fill(_abi.NormBackwardArgs, NORM, NORM_PTRS, over)
    for run in (_abi.lib().rhz_layernorm_backward, _abi.lib().rhz_rmsnorm_heads_backward):
        assert run(byref(a), None) == status, _abi.last_error()
        assert msg in _abi.last_error()


def test_layernorm_validation():
    run = _abi.lib().rhz_layernorm
    for over, status in ((dict(rows=-1), _abi.ERR_INVALID_ARG), (dict(dim=9000), _abi.ERR_UNSUPPORTED),
                         (dict(x=None), _abi.ERR_INVALID_ARG), (dict(y=A + 1), _abi.ERR_INVALID_ARG),
                         (dict(weight=None), _abi.ERR_INVALID_ARG), (dict(bias=A + 2), _abi.ERR_INVALID_ARG),
                         (dict(rows=0, x=None, y=None, weight=None), _abi.OK)):
        assert run(byref(_fill(_abi.LayernormArgs, NORM, ("x", "weight", "y"), over)), None) == status
    a = _fill(_abi.NormBackwardArgs, NORM, NORM_PTRS + ("grad_bias",), {})
    assert _abi.lib().rhz_rmsnorm_heads_backward(byref(a), None) == _abi.ERR_INVALID_ARG
    assert "no bias" in _abi.last_error()


@pytest.mark.parametrize("name,struct,values,pointers", [
    ("rhz_gdr_conv_prepare_backward", _abi.ConvPrepareBackwardArgs, CONV, CONV_PTRS),
    ("rhz_norm_backward", _abi.NormBackwardArgs, NORM, NORM_PTRS)])
def test_other_workspace_sizes(name, struct, values, pointers):
    query = name + "_workspace_size"
    status, n = _size(_fill(struct, values, pointers, {}), query)
    assert status == _abi.OK and n > 0
    empty = {"seq_len": 0} if "seq_len" in values else {"rows": 0}
    assert _size(_fill(struct, values, pointers, empty), query) == (_abi.OK, 0)
    assert getattr(_abi.lib(), query)(byref(_fill(struct, values, pointers, {})), None) == _abi.ERR_INVALID_ARG


VALIDATION = {_abi.ERR_INVALID_ARG, _abi.ERR_UNSUPPORTED, _abi.ERR_WORKSPACE}
ints = st.one_of(st.integers(-3, 300), st.sampled_from([0, 1, 64, 128, 1024, 4096, 65536]),
                 st.integers(-2**31, 2**31 - 1))
ptrs = st.sampled_from([None, A, A + 1, A + 2, A + 4, A + 8, A + 16, A + STEP])


@pytest.mark.skipif(_gpu_visible(), reason="fake device addresses: CPU-only property tests")
@settings(max_examples=300, deadline=None)
@given(st.data())
def test_backward_never_reaches_a_launch(data):
    """Whatever the fields hold, a call without grad_beta ends in an error, or in nothing to do."""
    a = _abi.PrefillBackwardArgs()
    for f in ("batch", "seq_len", "heads", "d_k", "d_v"):
        setattr(a, f, data.draw(ints, label=f))
    for f in ("dtype", "gate_kind"):
        setattr(a, f, data.draw(st.integers(-2, 4), label=f))
    for f in BACKWARD_PTRS + ("cu_seqlens", "initial_state", "grad_final_state", "workspace"):
        setattr(a, f, data.draw(ptrs, label=f))
    a.workspace_bytes = data.draw(st.sampled_from([0, 1, 1 << 20, 1 << 50]))
    a.grad_beta = None
    status = _abi.lib().rhz_gdr_prefill_backward(byref(a), None)
    if status == _abi.OK:
        assert a.seq_len == 0
    else:
        assert status in VALIDATION and _abi.last_error()


# ---- the Rust bindings written out for maintainers agree with this header too

def _rust_block():
    doc = open(os.path.join(_abi.ROOT, "INTEGRATION.md")).read()
    i = doc.index("### src/sys_train.rs")
    start = doc.index("```rust", i) + len("```rust")
    return re.sub(r"//[^\n]*", "", doc[start:doc.index("```", start)])


def test_rust_bindings_agree():
    import test_integration_bindings as T

    text = T.strip_c_comments(open(_abi.TRAIN_HEADER).read())
    rust = _rust_block()
    structs = {}
    for name, body in re.findall(r"typedef struct (\w+) \{(.*?)\} \1;", text, flags=re.S):
        decls = [" ".join(d.split()) for d in body.split(";")]
        structs[name] = [re.fullmatch(r"(.+?)\s*(\w+)", d) for d in decls if d]
        structs[name] = [(m.group(2), T.c_to_rust(m.group(1))) for m in structs[name]]
    found = {}
    for name, body in re.findall(r"#\[repr\(C\)\]\s*pub struct (\w+) \{(.*?)\}", rust, flags=re.S):
        fields = [" ".join(f.split()) for f in body.split(",")]
        found[name] = [re.fullmatch(r"pub (\w+): (.+)", f).groups() for f in fields if f]
    assert found == structs and structs
    for name, params in re.findall(r"rhz_status\s+(rhz_\w+)\(([^)]*)\);", text):
        m = re.search(r"pub fn %s\(([^)]*)\)\s*->\s*i32;" % name, rust)
        assert m, name
        want = [T.c_to_rust(re.fullmatch(r"(.+?)\s*(\w+)", " ".join(x.split())).group(1)) for x in params.split(",")]
        assert [re.fullmatch(r"\s*\w+: (.+?)\s*", x).group(1) for x in params_of(m.group(1))] == want, name


def params_of(text):
    return [" ".join(x.split()) for x in text.split(",") if x.strip()]


@pytest.mark.parametrize("over,msg", [
    (dict(y=A + 4), "x"), (dict(x=A + 7 * STEP - 4, y=A + 7 * STEP), "x"), (dict(weight=A + 64, y=A), "weight"),
    (dict(bias=A + 2 * STEP + 4), "bias"), (dict(x=A, y=A, weight=A), "weight")])
def test_layernorm_overlaps(over, msg):
    """y may be x itself, but not lie across it, a weight or a bias."""
    a = _fill(_abi.LayernormArgs, NORM, ("x", "weight", "y"), over)
    if "weight" in over and "x" not in over:
        a.x = A + 5 * STEP
    assert _abi.lib().rhz_layernorm(byref(a), None) == _abi.ERR_INVALID_ARG
    assert "y overlaps " + msg in _abi.last_error()


def test_a_stream_of_another_device_is_refused():
    """Before anything is allocated or launched there."""
    import types

    import torch

    import rhizome_amd

    x, w = torch.empty((4, 8), device="meta"), torch.empty(8, device="meta")
    other = types.SimpleNamespace(device=torch.device("cuda", 1), cuda_stream=0)
    for run in (rhizome_amd.layernorm, rhizome_amd.rmsnorm_heads):
        with pytest.raises(ValueError, match="stream's device"):
            run(x, w, stream=other)
