"""Eviction from the packed cache by accumulated attention weight, on the GPU.

No counterpart in the reference.  :func:`attn_weight_sums` measures how much every cached key is attended to,
:func:`evict_keys` keeps the heaviest and the latest keys of every head in a smaller cache;
``serving.QuantizedKVCache.observe`` and ``.evict`` do both on a resident cache.
"""
from __future__ import annotations

import math
import struct
from typing import NamedTuple, Optional

import torch

from .. import _lib
from .hadamard import HEAD_DIM
from .quantize import _NBYTES_NIBBLE, _NBYTES_QJL, _prep_codebooks, _user_args


# ``omni_weight_sums_t`` and ``omni_evict_t`` of the C header, field by field
_WEIGHT_SUMS = struct.Struct("@10P2qQ10if")
_EVICT = struct.Struct("@8P7P2P5q2i")


class EvictedCache(NamedTuple):
    """What :func:`evict_keys` returns: the kept positions, the new lengths, and the kept rows of every array."""
    index: torch.Tensor
    seq_lens: torch.Tensor
    sums: torch.Tensor
    k_nibbles: torch.Tensor
    k_qjl: torch.Tensor
    k_norms: torch.Tensor
    v_nibbles: torch.Tensor
    v_qjl: Optional[torch.Tensor]
    v_norms: Optional[torch.Tensor]


def _check_rows(x: torch.Tensor, name: str, shape, dtype) -> None:
    if x.shape != shape or x.dtype is not dtype:
        raise ValueError(f"{name} must be {tuple(shape)} {dtype}, got {tuple(x.shape)} {x.dtype}")


def _lens(seq_lens: Optional[torch.Tensor], B: int, S: int, dev) -> Optional[torch.Tensor]:
    if seq_lens is None:
        return None
    if seq_lens.shape != (B,):
        raise ValueError(f"seq_lens must have shape ({B},), got {tuple(seq_lens.shape)}")
    if seq_lens.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"seq_lens must be int32 or int64, got {seq_lens.dtype}")
    if seq_lens.device.type == "cpu" and B and (int(seq_lens.min()) < 0 or int(seq_lens.max()) > S):
        raise ValueError(f"seq_lens must lie in [0, {S}]")
    return _lib.as_device(seq_lens, dev, torch.int32)


def attn_weight_sums(q: torch.Tensor, k_nibbles: torch.Tensor, k_qjl: torch.Tensor, k_norms: torch.Tensor, codebooks: torch.Tensor,
                     user_id=0, scale: Optional[float] = None, with_qjl: bool = True, *, seq_lens: Optional[torch.Tensor] = None,
                     rotate_q: bool = False, causal: bool = True, into: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Softmax weight that every cached key receives from ``q`` (B, n_heads, T, 128), summed over the T tokens and the heads of
    the key's group: float32 (B, n_kv_heads, S).  Cache arguments, ``scale``, ``with_qjl``, ``user_id`` and ``rotate_q`` as in
    ``omni_attn``, whose weights these are.

    ``causal``: the T tokens are the last ones of the cache, so token t sees the keys up to ``len - T + t`` (the window of a
    prompt's last tokens; one token sees everything); ``False``: every token sees all keys below the length.  A token without
    keys adds nothing; a NaN query reaches the keys its token sees, and no others.  Without ``into`` the result is a new tensor, zeros at and behind the length; with it the weights are
    added to ``into`` in place (entries at and behind the length stay as they are) and ``into`` is returned.  ``q`` and the
    nibble rows start on 16-byte boundaries, sign bytes on 8 (``ValueError``); arrays that are not contiguous are copied."""
    if q.dim() != 4 or k_nibbles.dim() != 4:
        raise ValueError("q must be (B, n_heads, T, 128) and k_nibbles (B, n_kv_heads, S, 64)")
    B, Hq, T, D = q.shape
    if D != HEAD_DIM:
        raise ValueError(f"attention requires last dim = {HEAD_DIM} (head_dim), got {D}")
    n_users, Hkv, S, _ = k_nibbles.shape
    if n_users != B:
        raise ValueError(f"cache holds {n_users} users but q has batch {B}")
    if Hkv == 0 or Hq == 0 or Hq % Hkv:
        raise ValueError(f"n_heads={Hq} is not a multiple of n_kv_heads={Hkv}")
    if q.dtype not in _lib.DTYPE_CODE:
        raise TypeError(f"unsupported q dtype {q.dtype}")
    _check_rows(k_nibbles, "k_nibbles", (B, Hkv, S, _NBYTES_NIBBLE), torch.uint8)
    _check_rows(k_qjl, "k_qjl", (B, Hkv, S, _NBYTES_QJL), torch.uint8)
    _check_rows(k_norms, "k_norms", (B, Hkv, S), torch.float32)
    if into is not None:
        _check_rows(into, "into", (B, Hkv, S), torch.float32)
        if not into.is_contiguous():
            raise ValueError("into must be contiguous")
    dev = _lib.require_cuda(q, k_nibbles, k_qjl, k_norms, into)
    lib = _lib.ensure_init(dev)
    lens = _lens(seq_lens, B, S, dev)
    cb, per_head = _prep_codebooks(codebooks, Hkv, dev)
    ids, uid = _user_args(user_id, B, dev)
    q, k_nibbles, k_qjl, k_norms = q.contiguous(), k_nibbles.contiguous(), k_qjl.contiguous(), k_norms.contiguous()
    sums = torch.empty(B, Hkv, S, dtype=torch.float32, device=dev) if into is None else into
    nbytes = lib.omni_attn_weight_sums_workspace_bytes(B, Hq, Hkv, T, S)
    scratch = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    call = _WEIGHT_SUMS.pack(q.data_ptr(), k_nibbles.data_ptr(), k_qjl.data_ptr(), k_norms.data_ptr(), cb.data_ptr(),
                             0 if ids is None else ids.data_ptr(), 0 if lens is None else lens.data_ptr(), 0 if scratch is None else scratch.data_ptr(),
                             sums.data_ptr(), _lib.status_ptr(dev), B, S, nbytes, _lib.DTYPE_CODE[q.dtype], per_head, uid, Hq, Hkv, T,
                             bool(with_qjl), bool(rotate_q), bool(causal), into is not None, 1.0 / math.sqrt(HEAD_DIM) if scale is None else scale)
    with _lib.on_device(dev):
        _lib.check(lib.omni_attn_weight_sums(call, _lib.stream_ptr(dev)))
    return sums


def evict_keys(sums: torch.Tensor, k_nibbles: torch.Tensor, k_qjl: torch.Tensor, k_norms: torch.Tensor, v_nibbles: torch.Tensor,
               budget: int, *, recent: int = 0, seq_lens: Optional[torch.Tensor] = None, v_qjl: Optional[torch.Tensor] = None,
               v_norms: Optional[torch.Tensor] = None, v_paired: bool = False, capacity: Optional[int] = None) -> EvictedCache:
    """Keep at most ``budget`` keys of every (user, head): the ``recent`` last ones and, of the others, those with the largest
    ``sums`` (B, n_kv_heads, S); of equal sums the earlier key stays, and NaN counts as the largest.  Users with at most
    ``budget`` keys keep all of them.

    The kept rows leave in their order, bit for bit, in new arrays of ``capacity`` rows per head (``budget`` when ``None``),
    zeros behind the new length; the arrays given are not changed.  ``index`` (B, n_kv_heads, budget) int32 holds the old
    positions, -1 behind the new length, and ``seq_lens`` the new lengths, int32.  Alignment as in :func:`attn_weight_sums`.  ``v_paired``: V's nibble rows are in a
    resident cache's pair layout for the old lengths, and are again for the new ones."""
    if k_nibbles.dim() != 4:
        raise ValueError("k_nibbles must be (B, n_kv_heads, S, 64)")
    B, H, S, _ = k_nibbles.shape
    budget, recent = int(budget), int(recent)
    capacity = budget if capacity is None else int(capacity)
    if budget < 1 or not 0 <= recent <= budget or capacity < budget:
        raise ValueError(f"need 0 <= recent <= budget <= capacity and budget >= 1, got recent={recent}, budget={budget}, capacity={capacity}")
    if (v_qjl is None) != (v_norms is None):
        raise ValueError("v_qjl and v_norms must both be given or both be None")
    _check_rows(sums, "sums", (B, H, S), torch.float32)
    for name, x, shape, dtype in (("k_nibbles", k_nibbles, (B, H, S, _NBYTES_NIBBLE), torch.uint8), ("k_qjl", k_qjl, (B, H, S, _NBYTES_QJL), torch.uint8),
                                  ("k_norms", k_norms, (B, H, S), torch.float32), ("v_nibbles", v_nibbles, (B, H, S, _NBYTES_NIBBLE), torch.uint8),
                                  ("v_qjl", v_qjl, (B, H, S, _NBYTES_QJL), torch.uint8), ("v_norms", v_norms, (B, H, S), torch.float32)):
        if x is not None:
            _check_rows(x, name, shape, dtype)
    dev = _lib.require_cuda(sums, k_nibbles, k_qjl, k_norms, v_nibbles, v_qjl, v_norms)
    lib = _lib.load()
    lens = _lens(seq_lens, B, S, dev)
    src = [None if x is None else x if x.is_contiguous() else x.contiguous() for x in (sums, k_nibbles, k_qjl, k_norms, v_nibbles, v_qjl, v_norms)]
    out = [None if x is None else torch.empty(B, H, capacity, *x.shape[3:], dtype=x.dtype, device=dev) for x in src]
    index = torch.empty(B, H, budget, dtype=torch.int32, device=dev)
    new_lens = torch.empty(B, dtype=torch.int32, device=dev)
    at = [0 if x is None else x.data_ptr() for x in (src[0], lens, *src[1:], *out, index, new_lens)]
    with _lib.on_device(dev):
        _lib.check(lib.omni_evict_keys(_EVICT.pack(*at, B, S, budget, recent, capacity, H, bool(v_paired)), _lib.stream_ptr(dev)))
    return EvictedCache(index, new_lens, *out)
