"""Torch-tensor front end of the training operators (include/rhizome_train.h):
the backward passes of the Local block's mixer and layer norm.

As in gdr.py, PyTorch is used only for device memory and streams: every
function checks shapes, fills the C argument struct with raw device pointers
and calls the library on the current HIP stream.  The functions take the
forward call's inputs again and the gradients of its outputs, and return the
gradients of its inputs; none keeps anything between calls.
"""
from __future__ import annotations

from ctypes import byref, c_size_t

import torch

from . import _abi
from .gdr import _DTYPES, _check_prefill_shapes, _empty, _gate, _ptr, _stream


def _same_device(*tensors):
    """Every tensor on the current device, whose stream the launch goes to."""
    here = torch.cuda.current_device()
    for t in tensors:
        if t is not None and t.is_cuda and t.device.index != here:
            raise ValueError(f"all tensors must be on the current device, cuda:{here}")


def _used_on(stream, *tensors):
    """Tensors that this module allocated, kept from reuse until a stream
    other than the current one is done with them."""
    if stream is not None:
        for t in tensors:
            if t is not None:
                t.record_stream(stream)


def _workspace(like, args, query, workspace):
    """Fill in args' workspace: the caller's, or a new one of the size that `query` gives; returns it."""
    if workspace is None:
        need = c_size_t(0)
        _abi.check(query(byref(args), byref(need)))
        if need.value:
            workspace = _empty(like, (need.value,), torch.uint8)
    if workspace is not None:
        args.workspace, args.workspace_bytes = _ptr(workspace), workspace.numel() * workspace.element_size()
    return workspace


def prefill_backward(q, k, v, g=None, beta=None, do=None, *, alpha=None, dfinal_state=None, cu_seqlens=None,
                     initial_state=None, output_dinitial_state=False, workspace=None, stream=None):
    """Backward pass of :func:`prefill` (rhz_gdr_prefill_backward).

    The forward call's inputs again, ``do`` the gradient of o and
    ``dfinal_state`` that of the final state (None: zeros).  Returns (dq, dk,
    dv, dgate, dbeta, dinitial_state or None): dgate is the gradient of g or of
    alpha, whichever was passed; all but the fp32 dinitial_state have q's dtype.
    Two calls that may run at the same time must not share a workspace.
    """
    gate, gate_kind = _gate(g, alpha)
    if beta is None or do is None:
        raise ValueError("beta and do are needed")
    n = _check_prefill_shapes(q, k, v, gate, beta, cu_seqlens, initial_state)
    if do.shape != v.shape or do.dtype != q.dtype:
        raise ValueError("do must have v's shape and q's dtype")
    H, d_k, d_v = q.shape[-2], q.shape[-1], v.shape[-1]
    want = (n, H, d_v, d_k)
    if dfinal_state is not None and (tuple(dfinal_state.shape) != want or dfinal_state.dtype != torch.float32):
        raise ValueError(f"dfinal_state must be fp32 {want}")
    _same_device(q, k, v, gate, beta, do, dfinal_state, cu_seqlens, initial_state, workspace)
    a = _abi.PrefillBackwardArgs()
    a.batch, a.seq_len = (q.shape[0], q.shape[1]) if cu_seqlens is None else (n, q.shape[0])
    a.heads, a.d_k, a.d_v, a.dtype, a.gate_kind = H, d_k, d_v, _DTYPES[q.dtype], gate_kind
    a.q, a.k, a.v, a.gate, a.beta, a.grad_o = _ptr(q), _ptr(k), _ptr(v), _ptr(gate), _ptr(beta), _ptr(do)
    a.cu_seqlens, a.initial_state, a.grad_final_state = _ptr(cu_seqlens), _ptr(initial_state), _ptr(dfinal_state)
    dq, dk, dv = _empty(q, q.shape), _empty(q, q.shape), _empty(q, v.shape)
    dgate, dbeta = _empty(q, gate.shape), _empty(q, gate.shape)
    dinit = _empty(q, want, torch.float32) if output_dinitial_state else None
    a.grad_q, a.grad_k, a.grad_v = _ptr(dq), _ptr(dk), _ptr(dv)
    a.grad_gate, a.grad_beta, a.grad_initial_state = _ptr(dgate), _ptr(dbeta), _ptr(dinit)
    workspace = _workspace(q, a, _abi.lib().rhz_gdr_prefill_backward_workspace_size, workspace)
    _abi.check(_abi.lib().rhz_gdr_prefill_backward(byref(a), _stream(stream)))
    _used_on(stream, dq, dk, dv, dgate, dbeta, dinit, workspace)
    return dq, dk, dv, dgate, dbeta, dinit
