"""Torch-tensor front end of the Global block's latent attention
(include/rhizome_attention.h): rotary positions, the paged cache of latents,
and the prefill over expanded keys and values with its backward pass.

As in gdr.py, PyTorch is used only for device memory and streams: every
function checks shapes, fills the C argument struct with raw device pointers
and calls the library on the current HIP stream.  A tensor of heads may be a
view with strides of its own -- the halves of one projection's output, a slice
of a head's channels -- as long as its last dimension is dense and the tokens
of a batch are evenly spaced.

A decoding step of the block, with the projections around it:

    rope(q_rope, positions, freq, out=q_rope)          # in place
    latent_append(c, k_rope, cache, page_table, lengths, frequencies=freq, norm_scale=w)
    o = latent_decode(q, cache, page_table, lengths, d_c=d_c, scale=scale)[0]
"""
from __future__ import annotations

from ctypes import byref, c_double, c_float

import torch

from . import _abi
from .gdr import _DTYPES, _count, _empty, _on_stream
from .train import _workspace

_SCALINGS = {"none": _abi.ROPE_PLAIN, "linear": _abi.ROPE_LINEAR, "by_parts": _abi.ROPE_BY_PARTS}


# A decoding step's calls are bounded by the host: the device is asked for once
# a call, and the argument structs are filled in by position, which is what
# most of a call's time went to (rope of one position of 8 sequences: 8.0 us).
def _here() -> int:
    return torch.cuda.current_device()


def _stream(here: int) -> int | None:
    return torch._C._cuda_getCurrentRawStream(here) or None


def _view(t: torch.Tensor | None, here: int) -> int | None:
    """The address of a tensor whose strides have been read, on the current device."""
    if t is None:
        return None
    if t.get_device() != here:
        if not t.is_cuda:
            raise ValueError("all tensors must be on the GPU")
        raise ValueError(f"all tensors must be on the current device, cuda:{here}")
    return t.data_ptr() or None


def _dense(t: torch.Tensor | None, here: int) -> int | None:
    """The same of a tensor that has to be contiguous."""
    if t is not None and not t.is_contiguous():
        raise ValueError("all tensors but those of heads must be contiguous")
    return _view(t, here)


def _strides(name, t, heads=True):
    """Strides in elements from token to token, and from head to head."""
    shape, st = t.shape, t.stride()
    if st[-1] != 1 and shape[-1] > 1:
        raise ValueError(f"{name}'s last dimension must be dense")
    at = -3 if heads else -2  # the tokens' dimension
    token = st[at]
    if len(shape) + at == 1:  # a batch before it
        batch, n = shape[0], shape[at]
        if n == 1:
            token = st[0] if batch > 1 else 0
        elif batch > 1 and st[0] != token * n and n > 0:
            raise ValueError(f"{name}'s tokens must be evenly spaced over the batch")
    return token, st[-2] if heads and shape[-2] > 1 else 0


def _check_positions(name, t, shape):
    if t.dtype != torch.int32 or t.shape != shape:
        raise ValueError(f"{name} must be int32 {tuple(shape)}")


def _check_frequencies(frequencies):
    if frequencies.dtype != torch.float64 or frequencies.dim() != 1:
        raise ValueError("frequencies must be fp64 [pairs], as rope_frequencies gives them")


def rope_frequencies(dim: int, *, theta: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                     trained_length: float = 4096.0, fast: float = 32.0, slow: float = 1.0, device="cuda"):
    """The table of a rotary embedding of ``dim`` channels (rhz_rope_frequencies):
    (turns per position of every pair, fp64 [dim / 2] on the device; the rotated
    values' magnitude).

    scaling "linear" divides every frequency by ``factor``; "by_parts" keeps
    those of pairs that turn more than ``fast`` times over ``trained_length``,
    divides those below ``slow`` turns and mixes between, with a magnitude of
    0.1 ln(factor) + 1.
    """
    if scaling not in _SCALINGS:
        raise ValueError(f"scaling must be one of {sorted(_SCALINGS)}")
    a = _abi.RopeFrequencyArgs(dim, _SCALINGS[scaling], theta, factor, trained_length, fast, slow)
    turns, magnitude = (c_double * max(dim // 2, 1))(), c_float(0.0)
    _abi.check(_abi.lib().rhz_rope_frequencies(byref(a), turns, byref(magnitude)))
    return torch.tensor(list(turns), dtype=torch.float64, device=device), magnitude.value


def rope(x, positions, frequencies, *, offset: int = 0, interleaved: bool = False, magnitude: float = 1.0,
         inverse: bool = False, out=None, stream=None):
    """Rotary positions (rhz_rope): of every head's channels the 2 n from
    ``offset`` on, n the number of ``frequencies``, are turned by their
    position's angles; the others are copied.

    x [tokens, H, d] or [B, T, H, d], positions int32 of its leading
    dimensions.  Pairs are (i, i + n), or neighbours when ``interleaved``.
    ``out`` may be x itself.  ``inverse`` turns back and is the backward pass:
    dx = rope(dy, ..., inverse=True).
    """
    if stream is not None:
        return _on_stream(rope, locals())
    if x.dim() not in (3, 4) or x.dtype not in _DTYPES:
        raise ValueError("x must be fp32 or bf16 [tokens, H, d] or [B, T, H, d]")
    _check_positions("positions", positions, x.shape[:-2])
    _check_frequencies(frequencies)
    y = out if out is not None else _empty(x, x.shape)
    if y.shape != x.shape or y.dtype != x.dtype:
        raise ValueError("out must have x's shape and dtype")
    xt, xh = _strides("x", x)
    yt, yh = (xt, xh) if y is x else _strides("out", y)
    here = _here()
    a = _abi.RopeArgs(_count(positions.numel()), x.shape[-2], x.shape[-1], offset, 2 * frequencies.numel(), _DTYPES[x.dtype],
                      interleaved, inverse, magnitude, xt, xh, yt, yh, _view(x, here), _dense(positions, here),
                      _dense(frequencies, here), _view(y, here))
    _abi.check(_abi.lib().rhz_rope(byref(a), _stream(here)))
    return y


def _check_paged(cache, page_table, lengths, D):
    if cache.dim() != 3 or cache.dtype not in _DTYPES or cache.shape[-1] != D:
        raise ValueError(f"cache must be fp32 or bf16 [pages, page_size, {D}]")
    if page_table.dim() != 2:
        raise ValueError("page_table must be int32 [sequences, pages]")
    _check_positions("page_table", page_table, page_table.shape)
    _check_positions("lengths", lengths, page_table.shape[:1])
    return page_table.shape[0]


def latent_append(latent, k_rope, cache, page_table, lengths, *, cu_seqlens=None, frequencies=None,
                  interleaved: bool = False, magnitude: float = 1.0, norm_scale=None, eps: float = 1e-6, stream=None):
    """Write new tokens into the paged cache of latents (rhz_latent_append); returns the cache.

    latent [B, n, d_c] (dense: n new tokens of every sequence) or [tokens, d_c]
    with ``cu_seqlens``; k_rope likewise with d_r, or None; cache [pages,
    page_size, d_c + d_r]; page_table int32 [B, max_pages]; lengths int32 [B],
    the new tokens included.  The latent is RMS-normalised where ``norm_scale``
    [d_c] is given, the rotary key turned where ``frequencies`` are.
    """
    if stream is not None:
        return _on_stream(latent_append, locals())
    dense = cu_seqlens is None
    if latent.dim() != (3 if dense else 2) or latent.dtype != cache.dtype:
        raise ValueError(f"latent must be {'[B, n, d_c]' if dense else '[tokens, d_c]'} of the cache's dtype")
    if k_rope is not None and (k_rope.shape[:-1] != latent.shape[:-1] or k_rope.dtype != cache.dtype):
        raise ValueError("k_rope must have latent's tokens and dtype")
    d_c, d_r = latent.shape[-1], k_rope.shape[-1] if k_rope is not None else 0
    batch = _check_paged(cache, page_table, lengths, d_c + d_r)
    if dense and latent.shape[0] != batch:
        raise ValueError(f"latent has {latent.shape[0]} sequences, the page table {batch}")
    if not dense:
        _check_positions("cu_seqlens", cu_seqlens, (batch + 1,))
    if frequencies is not None:
        _check_frequencies(frequencies)
        if 2 * frequencies.numel() != d_r:
            raise ValueError(f"{frequencies.numel()} frequencies for a rotary key of {d_r}")
    if norm_scale is not None and (norm_scale.shape != (d_c,) or norm_scale.dtype != torch.float32):
        raise ValueError(f"norm_scale must be fp32 ({d_c},)")
    latent_stride = _strides("latent", latent, heads=False)[0]
    k_rope_stride = _strides("k_rope", k_rope, heads=False)[0] if d_r else 0
    here = _here()
    a = _abi.LatentAppendArgs(
        batch, _count(latent.shape[-2]), d_c, d_r, cache.shape[1], cache.shape[0], page_table.shape[1], _DTYPES[cache.dtype],
        interleaved, magnitude, eps, latent_stride, k_rope_stride, _view(latent, here), _view(k_rope, here),
        _dense(cu_seqlens, here), _dense(lengths, here), _dense(page_table, here), _dense(frequencies, here),
        _dense(norm_scale, here), _dense(cache, here))
    _abi.check(_abi.lib().rhz_latent_append(byref(a), _stream(here)))
    return cache


def latent_decode(q, cache, page_table, lengths, *, d_c: int, scale: float, out=None, workspace=None, stream=None):
    """Attention of the last positions of every sequence over its cached
    latents, absorbed (rhz_latent_decode).

    q [B, n, H, d_c + d_r], the queries of the last n positions in the latents'
    space; cache, page_table and lengths as for :func:`latent_append`, which has
    written them.  Returns (o [B, n, H, d_c], lse fp32 [B, n, H]).  Two calls
    that may run at the same time must not share a workspace.
    """
    if stream is not None:
        return _on_stream(latent_decode, locals())
    if q.dim() != 4 or q.dtype != cache.dtype:
        raise ValueError("q must be [B, n, H, d_c + d_r] of the cache's dtype")
    batch = _check_paged(cache, page_table, lengths, q.shape[-1])
    if q.shape[0] != batch or not 0 < d_c <= q.shape[-1]:
        raise ValueError(f"q is of {q.shape[0]} sequences and {q.shape[-1]} channels, the page table of {batch}, d_c is {d_c}")
    want = (*q.shape[:-1], d_c)
    o = out if out is not None else _empty(q, want)
    if o.shape != want or o.dtype != q.dtype:
        raise ValueError(f"out must be {q.dtype} {want}")
    here = _here()
    lse = _empty(q, want[:-1], torch.float32)
    a = _abi.LatentDecodeArgs(
        batch, want[1], want[2], d_c, q.shape[-1] - d_c, cache.shape[1], cache.shape[0], page_table.shape[1], _DTYPES[q.dtype],
        scale, _dense(q, here), _dense(cache, here), _dense(page_table, here), _dense(lengths, here), _dense(o, here),
        _dense(lse, here))
    workspace = _workspace(q, a, _abi.lib().rhz_latent_decode_workspace_size, workspace)
    _view(workspace, here)
    _abi.check(_abi.lib().rhz_latent_decode(byref(a), _stream(here)))
    return o, lse


def _prefill_args(q, k, v, k_rope, scale, causal, cu_seqlens, cu_seqlens_k) -> _abi.LatentPrefillArgs:
    """Check the shapes and fill in sizes and strides; _prefill_pointers does the rest."""
    nd = 4 if cu_seqlens is None else 3
    if q.dim() != nd or k.dim() != nd or v.dim() != nd:
        raise ValueError("q, k and v must be [B, T, H, d], or [tokens, H, d] with cu_seqlens")
    if q.dtype not in _DTYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("q, k, v must share one dtype, fp32 or bf16")
    H, d_n, d_v = q.shape[-2], k.shape[-1], v.shape[-1]
    d_r = q.shape[-1] - d_n
    if v.shape[:-1] != k.shape[:-1] or k.shape[-2] != H or d_r < 0:
        raise ValueError(f"q/k/v shapes {tuple(q.shape)} {tuple(k.shape)} {tuple(v.shape)} do not match")
    if (k_rope is None) != (d_r == 0):
        raise ValueError(f"q has {d_r} channels more than k: k_rope must have them, or be None for none")
    if k_rope is not None and (k_rope.shape != (*k.shape[:-2], d_r) or k_rope.dtype != q.dtype):
        raise ValueError(f"k_rope must be {q.dtype} {(*k.shape[:-2], d_r)}")
    if cu_seqlens is None:
        if cu_seqlens_k is not None:
            raise ValueError("cu_seqlens_k without cu_seqlens")
        if k.shape[0] != q.shape[0]:
            raise ValueError("q and k must have the same batch")
        batch, seq_len, seq_len_k = q.shape[0], q.shape[1], k.shape[1]
    else:
        _check_positions("cu_seqlens", cu_seqlens, cu_seqlens.shape)
        if cu_seqlens_k is not None:
            _check_positions("cu_seqlens_k", cu_seqlens_k, cu_seqlens.shape)
        batch, seq_len, seq_len_k = cu_seqlens.numel() - 1, _count(q.shape[0]), _count(k.shape[0])
    return _abi.LatentPrefillArgs(
        batch, seq_len, seq_len_k, H, d_n, d_r, d_v, _DTYPES[q.dtype], causal, q.shape[-1] ** -0.5 if scale is None else scale,
        *_strides("q", q), *_strides("k", k), *_strides("v", v), _strides("k_rope", k_rope, heads=False)[0] if d_r else 0)


def _prefill_pointers(a, here, q, k, v, k_rope, cu_seqlens, cu_seqlens_k, o, lse):
    a.q, a.k, a.v, a.k_rope = _view(q, here), _view(k, here), _view(v, here), _view(k_rope, here)
    a.cu_seqlens, a.cu_seqlens_k = _dense(cu_seqlens, here), _dense(cu_seqlens_k, here)
    a.o, a.lse = _dense(o, here), _dense(lse, here)


def latent_prefill(q, k, v, k_rope=None, *, scale=None, causal: bool = True, cu_seqlens=None, cu_seqlens_k=None,
                   out=None, stream=None):
    """Latent attention over expanded keys and values (rhz_latent_prefill).

    q [B, T, H, d_n + d_r], k [B, S, H, d_n], v [B, S, H, d_v], k_rope [B, S,
    d_r] for all heads (None: d_r = 0), or [tokens, ...] with ``cu_seqlens`` and,
    where the keys are others, ``cu_seqlens_k``.  Causal: the last query of a
    sequence sees all of its keys.  scale defaults to (d_n + d_r) ** -0.5.
    Returns (o [B, T, H, d_v], lse fp32 [B, T, H]), which the backward pass takes.
    """
    if stream is not None:
        return _on_stream(latent_prefill, locals())
    a = _prefill_args(q, k, v, k_rope, scale, causal, cu_seqlens, cu_seqlens_k)
    want = (*q.shape[:-1], v.shape[-1])
    o = out if out is not None else _empty(q, want)
    if o.shape != want or o.dtype != q.dtype:
        raise ValueError(f"out must be {q.dtype} {want}")
    lse = _empty(q, want[:-1], torch.float32)
    here = _here()
    _prefill_pointers(a, here, q, k, v, k_rope, cu_seqlens, cu_seqlens_k, o, lse)
    _abi.check(_abi.lib().rhz_latent_prefill(byref(a), _stream(here)))
    return o, lse


def latent_prefill_backward(q, k, v, k_rope, o, lse, do, *, dlse=None, scale=None, causal: bool = True, cu_seqlens=None,
                            cu_seqlens_k=None, workspace=None, stream=None):
    """Backward pass of :func:`latent_prefill` (rhz_latent_prefill_backward).

    The forward call's inputs again, its o and lse, ``do`` the gradient of o and
    ``dlse`` that of lse (None: zeros).  Returns (dq, dk, dv, dk_rope or None),
    contiguous and of q's dtype, dk_rope summed over the heads.  Two calls that
    may run at the same time must not share a workspace.
    """
    if stream is not None:
        return _on_stream(latent_prefill_backward, locals())
    a = _abi.LatentPrefillBackwardArgs()
    a.forward = _prefill_args(q, k, v, k_rope, scale, causal, cu_seqlens, cu_seqlens_k)
    want = (*q.shape[:-1], v.shape[-1])
    for name, t in (("o", o), ("do", do)):
        if t.shape != want or t.dtype != q.dtype:
            raise ValueError(f"{name} must be {q.dtype} {want}")
    for name, t in (("lse", lse), ("dlse", dlse)):
        if t is not None and (t.shape != q.shape[:-1] or t.dtype != torch.float32):
            raise ValueError(f"{name} must be fp32 {tuple(q.shape[:-1])}")
    here = _here()
    _prefill_pointers(a.forward, here, q, k, v, k_rope, cu_seqlens, cu_seqlens_k, o, lse)
    dq, dk, dv = _empty(q, q.shape), _empty(k, k.shape), _empty(v, v.shape)
    dr = _empty(k_rope, k_rope.shape) if k_rope is not None else None
    a.grad_o, a.grad_lse = _dense(do, here), _dense(dlse, here)
    a.grad_q, a.grad_k, a.grad_v, a.grad_k_rope = _view(dq, here), _view(dk, here), _view(dv, here), _view(dr, here)
    workspace = _workspace(q, a, _abi.lib().rhz_latent_prefill_backward_workspace_size, workspace)
    _view(workspace, here)
    _abi.check(_abi.lib().rhz_latent_prefill_backward(byref(a), _stream(here)))
    return dq, dk, dv, dr
