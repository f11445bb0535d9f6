"""Per-head norms of queries and keys with their position rotation, in one pass on the GPU.

No counterpart in the reference, whose queries and keys arrive rotated by their positions: this is the step in front of
:func:`omnistack_rs_b200.kernels.prompt_attention.prompt_attn` and of a cache's ``append``.
"""
from __future__ import annotations

import struct
from typing import Optional, Sequence, Tuple

import torch

from .. import _lib
from .hadamard import HEAD_DIM

MAX_AXES: int = 4


# ``omni_norm_rope_t`` of the C header, field by field (packed in one go: filling a ctypes structure costs several microseconds)
_NORM_ROPE = struct.Struct("@2P2P2PPP6q3q2q2i2i4i7if")


def _place(x: torch.Tensor):
    """(tensor, address, strides of users, heads and tokens) of rows a kernel can read: ``x`` itself when its 128-element rows are
    contiguous and start on 16-byte boundaries, else a contiguous copy.  Strides of extents of one do not count and are 0."""
    n0, n1, n2, _ = x.shape
    at = x.data_ptr()
    if not at & 15 and x.is_contiguous():
        return x, at, n1 * n2 * HEAD_DIM, n2 * HEAD_DIM, HEAD_DIM
    s0, s1, s2, s3 = x.stride()
    if n0 < 2:
        s0 = 0
    if n1 < 2:
        s1 = 0
    if n2 < 2:
        s2 = 0
    if s3 != 1 or at & 15 or (s0 | s1 | s2) & (3 if x.dtype is torch.float32 else 7):
        x = x.clone(memory_format=torch.contiguous_format)
        return x, x.data_ptr(), n1 * n2 * HEAD_DIM, n2 * HEAD_DIM, HEAD_DIM
    return x, at, s0, s1, s2


def _check_weight(w: Optional[torch.Tensor], name: str) -> None:
    if w is None:
        return
    if w.shape != (HEAD_DIM,):
        raise ValueError(f"{name} must have shape ({HEAD_DIM},) (head_dim), got {tuple(w.shape)}")
    if w.dtype not in _lib.DTYPE_CODE:
        raise TypeError(f"unsupported {name} dtype {w.dtype}; use float32, bfloat16 or float16")


def _weight(w: Optional[torch.Tensor], dev):
    """(tensor, address, dtype code) of a norm weight as the kernel reads it."""
    if w is None:
        return None, 0, 0
    if w.device != dev or not w.is_contiguous():
        w = w.to(dev).contiguous()
    if w.data_ptr() & 15:
        w = w.clone()
    return w, w.data_ptr(), _lib.DTYPE_CODE[w.dtype]


def qk_norm_rope(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, inv_freq: torch.Tensor, *,
                 q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, eps: Optional[float] = 1e-6,
                 axis_pairs: Optional[Sequence[int]] = None, interleaved: bool = False
                 ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Normalise every head's row by its root mean square (times a weight of 128) and rotate it by its position.

    ``q`` (B, n_heads, T, 128) and ``k`` (B, n_kv_heads, T, 128, or ``None``), float32, bfloat16 or float16, any strides over
    users, heads and tokens (views of a projection's output are read in place).  Returns new contiguous tensors of their
    shapes and dtype; everything inside is float32 and rounded once.

    ``positions``: integer tensor (B, T) or (T,); with ``axis_pairs = (n_0, n_1, ...)`` (at most four axes, e.g. time, height
    and width) it is (n_axes, B, T) or (n_axes, T), and the first n_0 pairs follow axis 0, the next n_1 axis 1, and so on.
    ``inv_freq``: float32 or float64 (P,), one frequency per pair, P <= 64; pair i turns by position * inv_freq[i], formed in
    float64.  The pairs are dims (i, i + P), or (2i, 2i + 1) with ``interleaved``; dims from 2P on are not rotated.
    ``eps=None`` leaves the norm (and the weights) out."""
    q_shape = q.shape
    if len(q_shape) != 4 or (k is not None and k.dim() != 4):
        raise ValueError("q and k must be (B, n_heads, T, 128)")
    B, Hq, T, D = q_shape
    if D != HEAD_DIM:
        raise ValueError(f"norm and rotation require last dim = {HEAD_DIM} (head_dim), got {D}")
    Hkv, k_at, k_strides, k_out, k_out_at = 0, 0, (0, 0, 0), None, 0
    if k is not None:
        k0, Hkv, k2, k3 = k.shape
    if k is not None and (k0 != B or k2 != T or k3 != HEAD_DIM):
        raise ValueError(f"k must be ({B}, n_kv_heads, {T}, {HEAD_DIM}) like q, got {tuple(k.shape)}")
    code = _lib.DTYPE_CODE.get(q.dtype)
    if code is None:
        raise TypeError(f"unsupported dtype {q.dtype}; use float32, bfloat16 or float16")
    if k is not None and k.dtype is not q.dtype:
        raise TypeError(f"q and k have different dtypes: {q.dtype} and {k.dtype}")
    if inv_freq.dim() != 1 or inv_freq.numel() > HEAD_DIM // 2:
        raise ValueError(f"inv_freq must have shape (P,) with P <= {HEAD_DIM // 2}, got {tuple(inv_freq.shape)}")
    P = inv_freq.numel()
    if inv_freq.dtype not in (torch.float32, torch.float64):
        raise TypeError(f"inv_freq must be float32 or float64, got {inv_freq.dtype}")
    if positions.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"positions must be int32 or int64, got {positions.dtype}")
    if axis_pairs is None:
        n_axes, ends, lead = 1, (P, 0, 0, 0), ()
    else:
        axis_pairs = tuple(int(n) for n in axis_pairs)
        n_axes, lead = len(axis_pairs), (len(axis_pairs),)
        ends = tuple(sum(axis_pairs[:i + 1]) for i in range(n_axes)) + (0,) * (MAX_AXES - n_axes)
        if not 1 <= len(axis_pairs) <= MAX_AXES or min(axis_pairs) < 0 or sum(axis_pairs) != P:
            raise ValueError(f"axis_pairs must be 1 to {MAX_AXES} pair counts that add up to {P} (the length of inv_freq), got {axis_pairs}")
    if positions.shape != lead + (B, T) and positions.shape != lead + (T,):
        raise ValueError(f"positions must have shape {lead + (B, T)} or {lead + (T,)}, got {tuple(positions.shape)}")
    if eps is None and (q_weight is not None or k_weight is not None):
        raise ValueError("eps=None leaves the norm out, so it takes no weights")
    _check_weight(q_weight, "q_weight")
    _check_weight(k_weight, "k_weight")
    dev = _lib.require_cuda(q, k)
    lib = _lib.load()
    q, q_at, *q_strides = _place(q)
    q_out = torch.empty(B, Hq, T, HEAD_DIM, dtype=q.dtype, device=dev)
    if k is not None:
        k, k_at, *k_strides = _place(k)
        k_out = torch.empty(B, Hkv, T, HEAD_DIM, dtype=q.dtype, device=dev)
        k_out_at = k_out.data_ptr()
    q_weight, qw_at, qw_code = _weight(q_weight, dev)
    k_weight, kw_at, kw_code = _weight(k_weight, dev)
    if positions.device != dev:
        positions = positions.to(dev)
    if inv_freq.device != dev or not inv_freq.is_contiguous():
        inv_freq = inv_freq.to(dev).contiguous()
    ps = positions.stride()
    call = _NORM_ROPE.pack(
        q_at, k_at, q_out.data_ptr(), k_out_at, qw_at, kw_at, positions.data_ptr(), inv_freq.data_ptr(), *q_strides, *k_strides,
        ps[0] if lead else 0, ps[-2] if positions.dim() == len(lead) + 2 else 0, ps[-1], B, T, Hq, Hkv, qw_code, kw_code, *ends,
        code, n_axes, P, positions.dtype is torch.int64, inv_freq.dtype is torch.float64, bool(interleaved),
        eps is not None, 0.0 if eps is None else eps)
    with _lib.on_device(dev):
        _lib.check(lib.omni_qk_norm_rope(call, _lib.stream_ptr(dev)))
    return q_out, k_out
