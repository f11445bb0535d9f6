"""Attention of whole prompts over themselves on the GPU: what runs before a prompt's keys and values are packed.

The reference computes it with ``reference_attn`` (omnistack_rs/attention/reference.py:72) over dense tensors and an additive
mask; here a prompt's bounds and the causal order are arguments, and prompts of different lengths share a call.
"""
from __future__ import annotations

import math
import struct
from typing import Optional

import torch

from .. import _lib
from .hadamard import HEAD_DIM
from .position import _place

_SCALE = 1.0 / math.sqrt(HEAD_DIM)
# ``omni_prompt_t`` of the C header, field by field
_PROMPT = struct.Struct("@7P9q3q4if")


def _tiles(x: torch.Tensor):
    """Rows a kernel can copy in boxes: tensor maps have no stride of 0, so rows shared by one are copied."""
    if not x.is_contiguous() and 0 in x.stride()[:3]:
        x = x.contiguous()
    return _place(x)


def prompt_attn(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, cu_seqlens: Optional[torch.Tensor] = None,
                seq_lens: Optional[torch.Tensor] = None, causal: bool = True, scale: Optional[float] = None) -> torch.Tensor:
    """``softmax(scale q k^T) v`` within every prompt; returns a new contiguous tensor of ``q``'s shape and dtype.

    ``q`` (B, n_heads, T, 128), ``k`` and ``v`` (B, n_kv_heads, T, 128), float32, bfloat16 or float16, any strides over users,
    heads and tokens; n_heads is a multiple of n_kv_heads.  Query t sees the keys up to t (``causal``) or all keys of its
    prompt.  ``scale`` defaults to 1/sqrt(128).

    Padded prompts: user b's prompt is its first ``seq_lens[b]`` rows (all T without ``seq_lens``).
    Packed prompts: B is 1 and ``cu_seqlens`` (n + 1,) gives the row at which each prompt begins, and the end of the last.
    Lengths held on the host are checked here; lengths on the device are taken as they are, cut to the T rows there are.
    Rows that belong to no prompt are zeros in the result, and what they hold in ``k`` and ``v`` reaches no other row, nor do
    the keys and values behind a query's own position (infinities and NaN included).

    Scores, softmax statistics and sums are float32.  For bfloat16 and float16 the tensor cores multiply the weights, rounded
    to that type, with the values; float32 stays float32 throughout.  A row that shares a tile with values that are
    infinite or NaN and that it must not see is formed again over its own keys, and may differ by the rounding of the weights."""
    q_shape, k_shape = q.shape, k.shape
    if len(q_shape) != 4 or len(k_shape) != 4 or v.dim() != 4:
        raise ValueError("q, k and v must be (B, n_heads, T, 128)")
    B, Hq, T, D = q_shape
    if D != HEAD_DIM:
        raise ValueError(f"attention requires last dim = {HEAD_DIM} (head_dim), got {D}")
    Hkv = k_shape[1]
    if k_shape[0] != B or k_shape[2] != T or k_shape[3] != HEAD_DIM or v.shape != k_shape:
        raise ValueError(f"k and v must be ({B}, n_kv_heads, {T}, {HEAD_DIM}) like q, got {tuple(k_shape)} and {tuple(v.shape)}")
    if Hkv == 0 or Hq % Hkv or Hq == 0:
        raise ValueError(f"n_heads={Hq} is not a multiple of n_kv_heads={Hkv}")
    dtype = q.dtype
    code = _lib.DTYPE_CODE.get(dtype)
    if code is None:
        raise TypeError(f"unsupported dtype {dtype}; use float32, bfloat16 or float16")
    if k.dtype is not dtype or v.dtype is not dtype:
        raise TypeError(f"q, k and v have different dtypes: {dtype}, {k.dtype} and {v.dtype}")
    packed = cu_seqlens is not None
    lengths = None
    if packed:
        if seq_lens is not None:
            raise ValueError("give cu_seqlens (packed prompts) or seq_lens (padded ones), not both")
        if B != 1:
            raise ValueError(f"packed prompts are the rows of one user (B = 1), got B = {B}")
        if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1:
            raise ValueError(f"cu_seqlens must have shape (n_prompts + 1,), got {tuple(cu_seqlens.shape)}")
        lengths, name = cu_seqlens, "cu_seqlens"
    elif seq_lens is not None:
        if seq_lens.shape != (B,):
            raise ValueError(f"seq_lens must have shape ({B},), got {tuple(seq_lens.shape)}")
        lengths, name = seq_lens, "seq_lens"
    if lengths is not None:
        if lengths.dtype is not torch.int32 and lengths.dtype is not torch.int64:
            raise TypeError(f"{name} must be int32 or int64, got {lengths.dtype}")
        if not lengths.is_cuda and lengths.numel():
            if int(lengths.min()) < 0 or int(lengths.max()) > T:
                raise ValueError(f"{name} must lie in [0, {T}]")
            if packed and bool((lengths[1:] < lengths[:-1]).any()):
                raise ValueError("cu_seqlens must ascend")
    dev = _lib.require_cuda(q, k, v)
    lib = _lib.load()
    n_seqs, cu_at, lens_at = B, 0, 0
    if lengths is not None:
        lengths = _lib.as_device(lengths, dev, torch.int32)
        if packed:
            n_seqs, cu_at = lengths.numel() - 1, lengths.data_ptr()
        else:
            lens_at = lengths.data_ptr()
    q, q_at, q0, q1, q2 = _tiles(q)
    k, k_at, k0, k1, k2 = _tiles(k)
    v, v_at, v0, v1, v2 = _tiles(v)
    out = torch.empty(B, Hq, T, HEAD_DIM, dtype=dtype, device=dev)
    call = _PROMPT.pack(q_at, k_at, v_at, out.data_ptr(), cu_at, lens_at, _lib.status_ptr(dev), q0, q1, q2, k0, k1, k2, v0, v1, v2,
                        n_seqs, B, T, code, Hq, Hkv, bool(causal), _SCALE if scale is None else scale)
    with _lib.on_device(dev):
        _lib.check(lib.omni_prompt_attn(call, _lib.stream_ptr(dev)))
    return out
