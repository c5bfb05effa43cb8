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
from .gdr import _DTYPES, _check_prefill_shapes, _count, _empty, _gate, _on_stream, _ptr, _stream


def _same_device(*tensors):
    """Every tensor on the current device, whose stream the launch goes to."""
    here = torch.cuda.current_device()
    for t in tensors:
        if t is not None and t.is_cuda and t.device.index != here:
            raise ValueError(f"all tensors must be on the current device, cuda:{here}")


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
    if stream is not None:
        return _on_stream(prefill_backward, locals())
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
    a.batch, a.seq_len = (q.shape[0], q.shape[1]) if cu_seqlens is None else (n, _count(q.shape[0]))
    a.heads, a.d_k, a.d_v, a.dtype, a.gate_kind = H, d_k, d_v, _DTYPES[q.dtype], gate_kind
    a.q, a.k, a.v, a.gate, a.beta, a.grad_o = _ptr(q), _ptr(k), _ptr(v), _ptr(gate), _ptr(beta), _ptr(do)
    a.cu_seqlens, a.initial_state, a.grad_final_state = _ptr(cu_seqlens), _ptr(initial_state), _ptr(dfinal_state)
    dq, dk, dv = _empty(q, q.shape), _empty(q, q.shape), _empty(q, v.shape)
    dgate, dbeta = _empty(q, gate.shape), _empty(q, gate.shape)
    dinit = _empty(q, want, torch.float32) if output_dinitial_state else None
    a.grad_q, a.grad_k, a.grad_v = _ptr(dq), _ptr(dk), _ptr(dv)
    a.grad_gate, a.grad_beta, a.grad_initial_state = _ptr(dgate), _ptr(dbeta), _ptr(dinit)
    workspace = _workspace(q, a, _abi.lib().rhz_gdr_prefill_backward_workspace_size, workspace)
    _abi.check(_abi.lib().rhz_gdr_prefill_backward(byref(a), _stream()))
    return dq, dk, dv, dgate, dbeta, dinit


def conv_prepare_backward(x, weight, bias, beta_logit, alpha_logit, a_log, dq, dk, dv, dbeta, dg, *, heads, d_k, d_v,
                          q_scale=None, cu_seqlens=None, initial_state=None, dfinal_state=None, workspace=None,
                          stream=None):
    """Backward pass of :func:`conv_prepare` (rhz_gdr_conv_prepare_backward).

    The forward call's inputs again and the gradients of its outputs: dq, dk,
    dv, dbeta and dg of x's dtype, ``dfinal_state`` [N, C, 3] fp32 that of the
    final conv state (None: zeros).  Returns (dx, dweight, dbias or None,
    dbeta_logit, dalpha_logit, da_log, dinitial_state or None): dbias where
    there is a bias, dinitial_state where there is an initial state; all but dx
    are fp32.
    """
    if stream is not None:
        return _on_stream(conv_prepare_backward, locals())
    C = heads * (2 * d_k + d_v)
    lead = x.shape[:-1]
    if x.shape[-1] != C or x.dim() != (3 if cu_seqlens is None else 2) or x.dtype not in _DTYPES:
        raise ValueError(f"x must be fp32 or bf16 [B, T, {C}] (dense) or [tokens, {C}] (packed)")
    batch, seq_len = (x.shape[0], x.shape[1]) if cu_seqlens is None else (cu_seqlens.numel() - 1, _count(x.shape[0]))
    if cu_seqlens is not None and cu_seqlens.dtype != torch.int32:
        raise ValueError("cu_seqlens must be int32")
    f32 = torch.float32
    for name, t, shape, dtype in (
            ("weight", weight, (C, 4), f32), ("bias", bias, (C,), f32), ("beta_logit", beta_logit, (*lead, heads), f32),
            ("alpha_logit", alpha_logit, (*lead, heads), f32), ("a_log", a_log, (heads,), f32),
            ("dq", dq, (*lead, heads, d_k), x.dtype), ("dk", dk, (*lead, heads, d_k), x.dtype),
            ("dv", dv, (*lead, heads, d_v), x.dtype), ("dbeta", dbeta, (*lead, heads), x.dtype),
            ("dg", dg, (*lead, heads), x.dtype), ("initial_state", initial_state, (batch, C, 3), f32),
            ("dfinal_state", dfinal_state, (batch, C, 3), f32)):
        if t is None and name in ("bias", "initial_state", "dfinal_state"):
            continue
        if tuple(t.shape) != tuple(shape) or t.dtype != dtype:
            raise ValueError(f"{name} must be {dtype} {tuple(shape)}")
    _same_device(x, weight, bias, beta_logit, alpha_logit, a_log, dq, dk, dv, dbeta, dg, cu_seqlens, initial_state,
                 dfinal_state, workspace)
    a = _abi.ConvPrepareBackwardArgs()
    a.batch, a.seq_len, a.heads, a.d_k, a.d_v, a.dtype = batch, seq_len, heads, d_k, d_v, _DTYPES[x.dtype]
    a.q_scale = float(d_k) ** 0.5 if q_scale is None else float(q_scale)
    a.x, a.weight, a.bias, a.cu_seqlens = _ptr(x), _ptr(weight), _ptr(bias), _ptr(cu_seqlens)
    a.initial_state, a.grad_final_state = _ptr(initial_state), _ptr(dfinal_state)
    a.beta_logit, a.alpha_logit, a.a_log = _ptr(beta_logit), _ptr(alpha_logit), _ptr(a_log)
    a.grad_q, a.grad_k, a.grad_v, a.grad_beta, a.grad_g = _ptr(dq), _ptr(dk), _ptr(dv), _ptr(dbeta), _ptr(dg)
    dx, dw = _empty(x, x.shape), _empty(weight, weight.shape)
    db = _empty(weight, (C,)) if bias is not None else None
    dbl, dal, da = _empty(beta_logit, beta_logit.shape), _empty(beta_logit, beta_logit.shape), _empty(a_log, a_log.shape)
    dinit = _empty(weight, (batch, C, 3)) if initial_state is not None else None
    a.grad_x, a.grad_weight, a.grad_bias, a.grad_initial_state = _ptr(dx), _ptr(dw), _ptr(db), _ptr(dinit)
    a.grad_beta_logit, a.grad_alpha_logit, a.grad_a_log = _ptr(dbl), _ptr(dal), _ptr(da)
    workspace = _workspace(x, a, _abi.lib().rhz_gdr_conv_prepare_backward_workspace_size, workspace)
    _abi.check(_abi.lib().rhz_gdr_conv_prepare_backward(byref(a), _stream()))
    return dx, dw, db, dbl, dal, da, dinit


def _check_norm(x, weight, *like_x):
    dim = x.shape[-1]
    if x.dtype not in _DTYPES:
        raise ValueError("x must be fp32 or bf16")
    if tuple(weight.shape) != (dim,) or weight.dtype != torch.float32:
        raise ValueError(f"the weight must be fp32 ({dim},)")
    for t in like_x:
        if t.shape != x.shape or t.dtype != x.dtype:
            raise ValueError("tensors of rows must share x's shape and dtype")
    return dim


def layernorm(x, weight, bias=None, eps: float = 1e-5, *, out=None, stream=None):
    """Layer norm over the last dimension: (x - mean) / sqrt(variance + eps) * weight + bias."""
    if stream is not None:
        return _on_stream(layernorm, locals())
    y = out if out is not None else _empty(x, x.shape)
    dim = _check_norm(x, weight, y)
    if bias is not None and (tuple(bias.shape) != (dim,) or bias.dtype != torch.float32):
        raise ValueError(f"bias must be fp32 ({dim},)")
    _same_device(x, weight, bias, y)
    a = _abi.LayernormArgs()
    a.rows, a.dim, a.dtype, a.eps = _count(x.numel() // max(dim, 1)), dim, _DTYPES[x.dtype], eps
    a.x, a.weight, a.bias, a.y = _ptr(x), _ptr(weight), _ptr(bias), _ptr(y)
    _abi.check(_abi.lib().rhz_layernorm(byref(a), _stream()))
    return y


def _norm_backward(run, dy, x, weight, eps, bias, workspace):
    dim = _check_norm(x, weight, dy)
    _same_device(dy, x, weight, workspace)
    a = _abi.NormBackwardArgs()
    a.rows, a.dim, a.dtype, a.eps = _count(x.numel() // max(dim, 1)), dim, _DTYPES[x.dtype], eps
    dx, dw = _empty(x, x.shape), _empty(weight, weight.shape)
    db = _empty(weight, weight.shape) if bias else None
    a.grad_y, a.x, a.weight = _ptr(dy), _ptr(x), _ptr(weight)
    a.grad_x, a.grad_weight, a.grad_bias = _ptr(dx), _ptr(dw), _ptr(db)
    workspace = _workspace(x, a, _abi.lib().rhz_norm_backward_workspace_size, workspace)
    _abi.check(run(byref(a), _stream()))
    return dx, dw, db


def layernorm_backward(dy, x, weight, eps: float = 1e-5, *, workspace=None, stream=None):
    """Backward pass of :func:`layernorm` from the gradient dy of its output
    and its x.  Returns (dx, dweight, dbias), the last two summed over the
    rows in fp32."""
    if stream is not None:
        return _on_stream(layernorm_backward, locals())
    return _norm_backward(_abi.lib().rhz_layernorm_backward, dy, x, weight, eps, True, workspace)


def rmsnorm_heads_backward(dy, x, scale, eps: float = 1e-6, *, workspace=None, stream=None):
    """Backward pass of :func:`rmsnorm_heads` from the gradient dy of its
    output and its x.  Returns (dx, dscale), dscale summed over the rows in
    fp32."""
    if stream is not None:
        return _on_stream(rmsnorm_heads_backward, locals())
    return _norm_backward(_abi.lib().rhz_rmsnorm_heads_backward, dy, x, scale, eps, False, workspace)[:2]
