"""Per-head norms of queries and keys with their position rotation, in one pass on the GPU.

No counterpart in the reference, whose queries and keys arrive rotated by their positions: this is the step in front of
:func:`omnistack_rs_b200.kernels.prompt_attention.prompt_attn` and of a cache's ``append``.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Sequence, Tuple

import torch

from .. import _lib
from .hadamard import HEAD_DIM

MAX_AXES: int = 4


class _NormRope(C.Structure):
    """``omni_norm_rope_t`` of the C header."""
    _fields_ = [("x", C.c_void_p * 2), ("y", C.c_void_p * 2), ("weight", C.c_void_p * 2), ("positions", C.c_void_p),
                ("inv_freq", C.c_void_p), ("xs", (C.c_int64 * 3) * 2), ("ps", C.c_int64 * 3), ("B", C.c_int64), ("T", C.c_int64),
                ("heads", C.c_int32 * 2), ("weight_dtype", C.c_int32 * 2), ("axis_end", C.c_int32 * MAX_AXES),
                ("dtype", C.c_int32), ("n_axes", C.c_int32), ("n_pairs", C.c_int32), ("positions64", C.c_int32),
                ("inv_freq64", C.c_int32), ("interleaved", C.c_int32), ("normalize", C.c_int32), ("eps", C.c_float)]


def _rows(x: torch.Tensor) -> torch.Tensor:
    """``x`` itself when a kernel can read its 128-element rows in place (16-byte boundaries), else a contiguous copy."""
    unit = 4 if x.dtype is torch.float32 else 8
    s = x.stride()
    if s[-1] != 1 or any(n > 1 and (st % unit or st < 0) for st, n in zip(s[:-1], x.shape[:-1])) or x.data_ptr() % 16:
        return x.contiguous() if x.data_ptr() % 16 == 0 or not x.is_contiguous() else x.clone()
    return x


def _strides(x: torch.Tensor):
    """Strides of users, heads and tokens; those of extents of one do not count and are given as 0."""
    return [st if n > 1 else 0 for st, n in zip(x.stride()[:3], x.shape[:3])]


def _check_weight(w: Optional[torch.Tensor], name: str) -> None:
    if w is None:
        return
    if w.shape != (HEAD_DIM,):
        raise ValueError(f"{name} must have shape ({HEAD_DIM},) (head_dim), got {tuple(w.shape)}")
    if w.dtype not in _lib.DTYPE_CODE:
        raise TypeError(f"unsupported {name} dtype {w.dtype}; use float32, bfloat16 or float16")


def _weight(w: Optional[torch.Tensor], dev) -> Optional[torch.Tensor]:
    if w is None:
        return None
    w = w.detach()
    if not (w.device == dev and w.is_contiguous()):
        w = w.to(dev).contiguous()
    return w if w.data_ptr() % 16 == 0 else w.clone()


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
    if q.dim() != 4 or (k is not None and k.dim() != 4):
        raise ValueError("q and k must be (B, n_heads, T, 128)")
    B, Hq, T, D = q.shape
    if D != HEAD_DIM:
        raise ValueError(f"norm and rotation require last dim = {HEAD_DIM} (head_dim), got {D}")
    if k is not None and (k.shape[0] != B or k.shape[2] != T or k.shape[3] != HEAD_DIM):
        raise ValueError(f"k must be ({B}, n_kv_heads, {T}, {HEAD_DIM}) like q, got {tuple(k.shape)}")
    if q.dtype not in _lib.DTYPE_CODE:
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
        axis_pairs, lead = (P,), ()
    else:
        axis_pairs = tuple(int(n) for n in axis_pairs)
        lead = (len(axis_pairs),)
        if not 1 <= len(axis_pairs) <= MAX_AXES or min(axis_pairs) < 0 or sum(axis_pairs) != P:
            raise ValueError(f"axis_pairs must be 1 to {MAX_AXES} pair counts that add up to {P} (the length of inv_freq), got {axis_pairs}")
    if tuple(positions.shape) not in (lead + (B, T), lead + (T,)):
        raise ValueError(f"positions must have shape {lead + (B, T)} or {lead + (T,)}, got {tuple(positions.shape)}")
    if eps is None and (q_weight is not None or k_weight is not None):
        raise ValueError("eps=None leaves the norm out, so it takes no weights")
    _check_weight(q_weight, "q_weight")
    _check_weight(k_weight, "k_weight")
    dev = _lib.require_cuda(q, k)
    lib = _lib.load()
    q_rows = _rows(q)
    k_rows = None if k is None else _rows(k)
    qw, kw = _weight(q_weight, dev), _weight(k_weight, dev)
    positions = positions.to(dev)
    inv_freq = inv_freq.detach()
    if inv_freq.device != dev or not inv_freq.is_contiguous():
        inv_freq = inv_freq.to(dev).contiguous()
    q_out = torch.empty(B, Hq, T, HEAD_DIM, dtype=q.dtype, device=dev)
    k_out = None if k is None else torch.empty(B, k.shape[1], T, HEAD_DIM, dtype=q.dtype, device=dev)
    ps = positions.stride()
    a = _NormRope()
    a.x[:] = [q_rows.data_ptr(), _lib.ptr(k_rows)]
    a.y[:] = [q_out.data_ptr(), _lib.ptr(k_out)]
    a.weight[:] = [_lib.ptr(qw), _lib.ptr(kw)]
    a.positions, a.inv_freq = positions.data_ptr(), inv_freq.data_ptr()
    a.xs[0][:] = _strides(q_rows)
    if k_rows is not None:
        a.xs[1][:] = _strides(k_rows)
    a.ps[:] = [ps[0] if lead else 0, ps[-2] if positions.dim() == len(lead) + 2 else 0, ps[-1]]
    a.B, a.T = B, T
    a.heads[:] = [Hq, 0 if k is None else k.shape[1]]
    a.weight_dtype[:] = [0 if w is None else _lib.DTYPE_CODE[w.dtype] for w in (qw, kw)]
    end = 0
    for i, n in enumerate(axis_pairs):
        end += n
        a.axis_end[i] = end
    a.dtype, a.n_axes, a.n_pairs = _lib.DTYPE_CODE[q.dtype], len(axis_pairs), P
    a.positions64, a.inv_freq64 = int(positions.dtype is torch.int64), int(inv_freq.dtype is torch.float64)
    a.interleaved, a.normalize, a.eps = int(bool(interleaved)), int(eps is not None), 0.0 if eps is None else float(eps)
    with _lib.on_device(dev):
        _lib.check(lib.omni_qk_norm_rope(C.byref(a), _lib.stream_ptr(dev)))
    return q_out, k_out
