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

from ctypes import byref, c_double, c_float, c_size_t

import torch

from . import _abi
from .gdr import _DTYPES, _count, _empty, _on_stream

_SCALINGS = {"none": _abi.ROPE_PLAIN, "linear": _abi.ROPE_LINEAR, "by_parts": _abi.ROPE_BY_PARTS}


# A decoding step's calls are bounded by the host: the device is asked for once
# a call, shapes are taken apart once, and the arguments are laid out in one go
# (_abi.pack_*): a rope of 8 tokens takes 6.8 us a call instead of 8.6.
def _here() -> int:
    return torch.cuda.current_device()


def _stream(here: int) -> int | None:
    return torch._C._cuda_getCurrentRawStream(here) or None


def _view(t: torch.Tensor | None, here: int) -> int:
    """The address of a tensor whose strides have been read, on the current device; 0 for None."""
    if t is None:
        return 0
    if t.get_device() != here:
        if not t.is_cuda:
            raise ValueError("all tensors must be on the GPU")
        raise ValueError(f"all tensors must be on the current device, cuda:{here}")
    return t.data_ptr()


def _dense(t: torch.Tensor | None, here: int) -> int:
    """The same of a tensor that has to be contiguous."""
    if t is not None and not t.is_contiguous():
        raise ValueError("all tensors but those of heads must be contiguous")
    return _view(t, here)


def _token_stride(name, t, batch, n):
    """In elements, of a tensor of n tokens of every sequence of a batch, whose
    last dimension has to be dense; batch None: of tokens alone.  A single token
    has no distance to a next one."""
    st = t.stride()
    if st[-1] != 1 and t.shape[-1] > 1:
        raise ValueError(f"{name}'s last dimension must be dense")
    if (n if batch is None else batch * n) <= 1:
        return 0
    if batch is None or n == 1:
        return st[0]
    if batch > 1 and st[0] != st[1] * n:
        raise ValueError(f"{name}'s tokens must be evenly spaced over the batch")
    return st[1]


def _workspace(size, a, like, workspace, here):
    """Address and bytes of the caller's workspace, or of a new one of the size
    that `size` gives for the arguments; and the new one, to be kept until the call."""
    if workspace is None:
        need = c_size_t()
        _abi.check(size(a, byref(need)))
        if not need.value:
            return 0, 0, None
        workspace = like.new_empty((need.value,), dtype=torch.uint8)
    return _dense(workspace, here), workspace.numel() * workspace.element_size(), workspace


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
    _count(abs(dim))  # the struct's field would take it modulo 2^32, the table's size not
    a = _abi.RopeFrequencyArgs(dim, _SCALINGS[scaling], theta, factor, trained_length, fast, slow)
    turns, magnitude = (c_double * 512)(), c_float(0.0)  # of the widest that is supported
    _abi.check(_abi.lib().rhz_rope_frequencies(byref(a), turns, byref(magnitude)))
    return torch.tensor(turns[:dim // 2], dtype=torch.float64, device=device), magnitude.value


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
    dtype, shape = _DTYPES.get(x.dtype), x.shape
    if dtype is None or len(shape) not in (3, 4):
        raise ValueError("x must be fp32 or bf16 [tokens, H, d] or [B, T, H, d]")
    batch, n = (shape[0], shape[1]) if len(shape) == 4 else (None, shape[0])
    H, d = shape[-2], shape[-1]
    _check_positions("positions", positions, (n,) if batch is None else (batch, n))
    _check_frequencies(frequencies)
    y = out if out is not None else _empty(x, shape)
    if y is not x and (y.shape != shape or y.dtype != x.dtype):
        raise ValueError("out must have x's shape and dtype")
    xt, xh = _token_stride("x", x, batch, n), x.stride(-2) if H > 1 else 0
    yt, yh = (xt, xh) if y is x else (_token_stride("out", y, batch, n), y.stride(-2) if H > 1 else 0)
    here = _here()
    a = _abi.pack_rope(_count(n if batch is None else batch * n), H, d, offset, 2 * frequencies.numel(), dtype, interleaved,
                       inverse, magnitude, xt, xh, yt, yh, _view(x, here), _dense(positions, here), _dense(frequencies, here),
                       _view(y, here))
    _abi.check(_abi.lib().rhz_rope(a, _stream(here)))
    return y


def _check_paged(cache, page_table, lengths, D):
    """Sequences, and what the argument structs have of the cache: page_size, num_pages, max_pages, dtype."""
    dtype, at, table = _DTYPES.get(cache.dtype), cache.shape, page_table.shape
    if len(at) != 3 or dtype is None or at[2] != D:
        raise ValueError(f"cache must be fp32 or bf16 [pages, page_size, {D}]")
    if len(table) != 2 or page_table.dtype != torch.int32:
        raise ValueError("page_table must be int32 [sequences, pages]")
    batch, width = table
    if lengths.dtype != torch.int32 or lengths.dim() != 1 or lengths.numel() != batch:
        raise ValueError(f"lengths must be int32 ({batch},)")
    return batch, (at[1], at[0], width, dtype)


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
    shape, dense = latent.shape, cu_seqlens is None
    if len(shape) != (3 if dense else 2) or latent.dtype != cache.dtype:
        raise ValueError(f"latent must be {'[B, n, d_c]' if dense else '[tokens, d_c]'} of the cache's dtype")
    n, d_c = shape[-2], shape[-1]
    d_r = k_rope.shape[-1] if k_rope is not None else 0
    if k_rope is not None and (k_rope.shape != ((shape[0], n, d_r) if dense else (n, d_r)) or k_rope.dtype != cache.dtype):
        raise ValueError("k_rope must have latent's tokens and dtype")
    batch, paged = _check_paged(cache, page_table, lengths, d_c + d_r)
    if dense and shape[0] != batch:
        raise ValueError(f"latent has {shape[0]} sequences, the page table {batch}")
    if not dense:
        _check_positions("cu_seqlens", cu_seqlens, (batch + 1,))
    if frequencies is not None:
        _check_frequencies(frequencies)
        if 2 * frequencies.numel() != d_r:
            raise ValueError(f"{frequencies.numel()} frequencies for a rotary key of {d_r}")
    if norm_scale is not None and (norm_scale.shape != (d_c,) or norm_scale.dtype != torch.float32):
        raise ValueError(f"norm_scale must be fp32 ({d_c},)")
    rows = batch if dense else None
    latent_stride, k_rope_stride = _token_stride("latent", latent, rows, n), _token_stride("k_rope", k_rope, rows, n) if d_r else 0
    here = _here()
    a = _abi.pack_latent_append(
        batch, _count(n), d_c, d_r, *paged, interleaved, magnitude, eps, latent_stride, k_rope_stride, _view(latent, here),
        _view(k_rope, here), _dense(cu_seqlens, here), _dense(lengths, here), _dense(page_table, here),
        _dense(frequencies, here), _dense(norm_scale, here), _dense(cache, here))
    _abi.check(_abi.lib().rhz_latent_append(a, _stream(here)))
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
    shape = q.shape
    if len(shape) != 4 or q.dtype != cache.dtype:
        raise ValueError("q must be [B, n, H, d_c + d_r] of the cache's dtype")
    rows, steps, H, D = shape
    batch, paged = _check_paged(cache, page_table, lengths, D)
    if rows != batch or not 0 < d_c <= D:
        raise ValueError(f"q is of {rows} sequences and {D} channels, the page table of {batch}, d_c is {d_c}")
    want = (batch, steps, H, d_c)
    o = out if out is not None else q.new_empty(want)
    if o.shape != want or o.dtype != q.dtype:
        raise ValueError(f"out must be {q.dtype} {want}")
    here, L = _here(), _abi.lib()
    lse = q.new_empty((batch, steps, H), dtype=torch.float32)
    args = (batch, steps, H, d_c, D - d_c, *paged, scale, _dense(q, here), _dense(cache, here), _dense(page_table, here),
            _dense(lengths, here), _dense(o, here), _view(lse, here))
    at, size, workspace = _workspace(L.rhz_latent_decode_workspace_size, _abi.pack_latent_decode(*args, 0, 0), q, workspace, here)
    _abi.check(L.rhz_latent_decode(_abi.pack_latent_decode(*args, at, size), _stream(here)))
    return o, lse


def _prefill_args(q, k, v, k_rope, scale, causal, cu_seqlens, cu_seqlens_k):
    """Check the shapes; (the argument struct's sizes and strides, the shapes of the queries' rows and of their outputs)."""
    qs, ks, vs, nd = q.shape, k.shape, v.shape, 4 if cu_seqlens is None else 3
    if len(qs) != nd or len(ks) != nd or len(vs) != nd:
        raise ValueError("q, k and v must be [B, T, H, d], or [tokens, H, d] with cu_seqlens")
    dtype = _DTYPES.get(q.dtype)
    if dtype is None or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("q, k, v must share one dtype, fp32 or bf16")
    if cu_seqlens is None:
        if cu_seqlens_k is not None:
            raise ValueError("cu_seqlens_k without cu_seqlens")
        (batch, n_q, H, d_q), (batch_k, n_k, H_k, d_n), d_v = qs, ks, vs[3]
        if batch_k != batch:
            raise ValueError("q and k must have the same batch")
        spread, rows = batch, (batch, n_q, H)
    else:
        (n_q, H, d_q), (n_k, H_k, d_n), d_v = qs, ks, vs[2]
        _check_positions("cu_seqlens", cu_seqlens, cu_seqlens.shape)
        if cu_seqlens_k is not None:
            _check_positions("cu_seqlens_k", cu_seqlens_k, cu_seqlens.shape)
        batch, spread, rows = cu_seqlens.numel() - 1, None, (n_q, H)
    d_r = d_q - d_n
    if vs[:-1] != ks[:-1] or H_k != H or d_r < 0:
        raise ValueError(f"q/k/v shapes {tuple(qs)} {tuple(ks)} {tuple(vs)} do not match")
    if (k_rope is None) != (d_r == 0):
        raise ValueError(f"q has {d_r} channels more than k: k_rope must have them, or be None for none")
    if k_rope is not None and (k_rope.shape != (*ks[:-2], d_r) or k_rope.dtype != q.dtype):
        raise ValueError(f"k_rope must be {q.dtype} {(*ks[:-2], d_r)}")
    one = H == 1  # whose distance to a next one is nothing's
    sizes = (batch, _count(n_q), _count(n_k), H, d_n, d_r, d_v, dtype, causal, (d_q or 1) ** -0.5 if scale is None else scale,
             _token_stride("q", q, spread, n_q), 0 if one else q.stride(-2),
             _token_stride("k", k, spread, n_k), 0 if one else k.stride(-2),
             _token_stride("v", v, spread, n_k), 0 if one else v.stride(-2),
             _token_stride("k_rope", k_rope, spread, n_k) if d_r else 0)
    return sizes, rows, (*rows, d_v)


def latent_prefill(q, k, v, k_rope=None, *, scale=None, causal: bool = True, cu_seqlens=None, cu_seqlens_k=None,
                   out=None, stream=None):
    """Latent attention over expanded keys and values (rhz_latent_prefill).

    q [B, T, H, d_n + d_r], k [B, S, H, d_n], v [B, S, H, d_v], k_rope [B, S,
    d_r] for all heads (None: d_r = 0), or [tokens, ...] with ``cu_seqlens`` and,
    where the keys are others, ``cu_seqlens_k``.  Causal: the last query of a
    sequence sees all of its keys.  scale defaults to (d_n + d_r) ** -0.5.
    Returns (o [B, T, H, d_v], lse fp32 [B, T, H]), which the backward pass takes.
    Rows of a pack outside every sequence are not written.
    """
    if stream is not None:
        return _on_stream(latent_prefill, locals())
    sizes, rows, want = _prefill_args(q, k, v, k_rope, scale, causal, cu_seqlens, cu_seqlens_k)
    o = out if out is not None else q.new_empty(want)
    if o.shape != want or o.dtype != q.dtype:
        raise ValueError(f"out must be {q.dtype} {want}")
    lse = q.new_empty(rows, dtype=torch.float32)
    here = _here()
    a = _abi.pack_latent_prefill(*sizes, _view(q, here), _view(k, here), _view(v, here), _view(k_rope, here),
                                 _dense(cu_seqlens, here), _dense(cu_seqlens_k, here), _dense(o, here), _view(lse, here))
    _abi.check(_abi.lib().rhz_latent_prefill(a, _stream(here)))
    return o, lse


def latent_prefill_backward(q, k, v, k_rope, o, lse, do, *, dlse=None, scale=None, causal: bool = True, cu_seqlens=None,
                            cu_seqlens_k=None, workspace=None, stream=None):
    """Backward pass of :func:`latent_prefill` (rhz_latent_prefill_backward).

    The forward call's inputs again, its o and lse, ``do`` the gradient of o and
    ``dlse`` that of lse (None: zeros).  Returns (dq, dk, dv, dk_rope or None),
    contiguous and of q's dtype, dk_rope summed over the heads.  Rows of a pack
    outside every sequence are not written.  Two calls that may run at the same
    time must not share a workspace.
    """
    if stream is not None:
        return _on_stream(latent_prefill_backward, locals())
    sizes, rows, want = _prefill_args(q, k, v, k_rope, scale, causal, cu_seqlens, cu_seqlens_k)
    for name, t in (("o", o), ("do", do)):
        if t.shape != want or t.dtype != q.dtype:
            raise ValueError(f"{name} must be {q.dtype} {want}")
    for name, t in (("lse", lse), ("dlse", dlse)):
        if t is not None and (t.shape != rows or t.dtype != torch.float32):
            raise ValueError(f"{name} must be fp32 {rows}")
    here, L = _here(), _abi.lib()
    dq, dk, dv = q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)
    dr = k_rope.new_empty(k_rope.shape) if k_rope is not None else None
    args = (*sizes, _view(q, here), _view(k, here), _view(v, here), _view(k_rope, here), _dense(cu_seqlens, here),
            _dense(cu_seqlens_k, here), _dense(o, here), _dense(lse, here), _dense(do, here), _dense(dlse, here),
            _view(dq, here), _view(dk, here), _view(dv, here), _view(dr, here))
    at, size, workspace = _workspace(L.rhz_latent_prefill_backward_workspace_size,
                                     _abi.pack_latent_prefill_backward(*args, 0, 0), q, workspace, here)
    _abi.check(L.rhz_latent_prefill_backward(_abi.pack_latent_prefill_backward(*args, at, size), _stream(here)))
    return dq, dk, dv, dr
