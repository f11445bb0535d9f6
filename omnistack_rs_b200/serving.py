"""Per-user cache container, user sharding across GPUs, and the host-buffer decode step.

The reference has no cache object (its README lists a paged cache as planned) and no
multi-GPU code; its serving loop (scripts/run_criteo_benchmark.py:481-560) keeps the packed
tensors resident on one GPU and sends a fresh query per step.  This module provides the same
loop for one process per GPU: users are independent, so rank r of n simply owns a contiguous
block of users and no collective is needed on the data path.
"""
from __future__ import annotations

import ctypes as C
import math
import os
from typing import Optional, Tuple

import torch

from . import _lib
from .kernels.quantize import _NBYTES_NIBBLE, _NBYTES_QJL, _codec_rows, _prep_codebooks, _user_args, rotate_quantize_append
from .kernels.eviction import EvictedCache, attn_weight_sums, evict_keys
from .kernels.fused_attention import _qattn, _auto_splits, pair_v_rows
from .kernels.prompt_attention import prompt_attn

HEAD_DIM = 128


def shard_range(n_units: int, world_size: int, rank: int) -> Tuple[int, int]:
    """Contiguous block [begin, end) of ``n_units`` owned by ``rank``; the first
    ``n_units % world_size`` ranks get one extra unit."""
    if not 0 <= rank < world_size:
        raise ValueError(f"rank {rank} outside world of {world_size}")
    base, extra = divmod(n_units, world_size)
    begin = rank * base + min(rank, extra)
    return begin, begin + base + (1 if rank < extra else 0)


def gather_rows_to_rank0(local: torch.Tensor, n_units: int, group=None) -> Optional[torch.Tensor]:
    """Gather per-rank row blocks (sharded with :func:`shard_range`) to rank 0 in user order.
    Blocks are padded to a common height because ``gather`` needs equal shapes.  Returns the
    ``(n_units, ...)`` tensor on rank 0 and ``None`` elsewhere.  Verification only -- the
    data path itself has no collective."""
    import torch.distributed as dist
    world, rank = dist.get_world_size(group), dist.get_rank(group)
    spans = [shard_range(n_units, world, r) for r in range(world)]
    height = max(e - b for b, e in spans)
    padded = local.new_zeros((height,) + tuple(local.shape[1:]))
    padded[: local.shape[0]] = local
    bufs = [torch.empty_like(padded) for _ in range(world)] if rank == 0 else None
    dist.gather(padded, bufs, dst=0, group=group)
    if rank != 0:
        return None
    return torch.cat([buf[: e - b] for buf, (b, e) in zip(bufs, spans)])


class ShardLiveness:
    """Host-side liveness record of the ranks of a sharded serving job, kept in a key-value store
    (``torch.distributed.TCPStore`` or any object with ``set`` / ``get`` / ``check``).  The data path has no
    collective, so a rank that stops cannot hang its peers; this record is how they learn of it before they next
    depend on that rank (a verification gather, a barrier): every rank posts the number of the step it has
    finished, and a rank that leaves on purpose says so.  Nothing here touches a GPU."""

    def __init__(self, store, rank: int, world_size: int):
        self.store, self.rank, self.world = store, rank, world_size

    def beat(self, step: int) -> None:
        self.store.set(f"omni/beat/{self.rank}", str(int(step)))

    def leave(self) -> None:
        self.store.set(f"omni/left/{self.rank}", "1")

    def _step_of(self, r: int) -> int:
        key = f"omni/beat/{r}"
        return int(self.store.get(key)) if self.store.check([key]) else -1

    def missing(self, step: int, timeout_s: float = 2.0, poll_s: float = 0.02):
        """Ranks that have not finished ``step`` within ``timeout_s`` (or announced that they left)."""
        import time
        deadline = time.monotonic() + timeout_s
        waiting = [r for r in range(self.world) if r != self.rank]
        gone = []
        while waiting:
            for r in list(waiting):
                if self.store.check([f"omni/left/{r}"]):
                    waiting.remove(r); gone.append(r)
                elif self._step_of(r) >= step:
                    waiting.remove(r)
            if not waiting or time.monotonic() >= deadline:
                break
            time.sleep(poll_s)
        return sorted(gone + waiting)


def collect_rows_via_store(store, rank: int, world_size: int, local: torch.Tensor, n_units: int, missing=()):
    """Verification gather that survives absent ranks: every live rank posts its row block (sharded with
    :func:`shard_range`) to the store and rank 0 assembles them.  Returns, on rank 0,
    ``(rows, missing_spans)`` -- the ``(n_units, ...)`` tensor with the rows of absent ranks left at zero and
    the ``[begin, end)`` unit ranges nobody delivered -- and ``None`` elsewhere."""
    import io
    if rank != 0:
        buf = io.BytesIO()
        torch.save(local.cpu(), buf)
        store.set(f"omni/rows/{rank}", buf.getvalue())
        return None
    rows = local.new_zeros((n_units,) + tuple(local.shape[1:]), device="cpu")
    b0, e0 = shard_range(n_units, world_size, 0)
    rows[b0:e0] = local.cpu()
    missing_spans = []
    for r in range(1, world_size):
        b, e = shard_range(n_units, world_size, r)
        if r in missing:
            missing_spans.append((b, e))
            continue
        rows[b:e] = torch.load(io.BytesIO(store.get(f"omni/rows/{r}")))
    return rows, missing_spans


class QuantizedKVCache:
    """Preallocated packed K/V cache for ``n_users`` users on one device.

    K rows hold nibbles + sign bytes + norm (4.75 bits per element); V rows are stored the
    same way (the codec produces all three) although attention reads only V's nibbles.
    """

    def __init__(self, n_users: int, n_kv_heads: int, max_len: int, codebooks: torch.Tensor,
                 device, user_ids: Optional[torch.Tensor] = None, store_v_residual: bool = True,
                 pair_v: bool = False):
        self.device = torch.device(device)
        self.n_users, self.n_kv_heads, self.max_len = n_users, n_kv_heads, max_len
        self.codebooks = codebooks.to(device=self.device, dtype=torch.float32).contiguous()
        shape = (n_users, n_kv_heads, max_len)
        mk = lambda *s, dt=torch.uint8: torch.zeros(*s, dtype=dt, device=self.device)  # noqa: E731
        self.k_nib, self.k_qjl, self.k_norms = mk(*shape, _NBYTES_NIBBLE), mk(*shape, _NBYTES_QJL), mk(*shape, dt=torch.float32)
        self.v_nib = mk(*shape, _NBYTES_NIBBLE)
        if store_v_residual:
            self.v_qjl, self.v_norms = mk(*shape, _NBYTES_QJL), mk(*shape, dt=torch.float32)
        else:   # attention never reads V's sign bits or norms: they are neither stored nor computed
            self.v_qjl = self.v_norms = None
        # pair_v: V nibble rows are kept in the pair layout the tensor-core kernel reads fastest; every append
        # converts the groups of eight keys it completes (``v_nib`` is then not interchangeable with the reference's)
        self.pair_v = bool(pair_v)
        self.lens = torch.zeros(n_users, dtype=torch.int64, device=self.device)
        # the same lengths as the attention entry points take them (int32, same storage for the cache's lifetime, so
        # repeated ``attend`` calls reuse one prepared call)
        self.lens32 = torch.zeros(n_users, dtype=torch.int32, device=self.device)
        self.user_ids = (torch.arange(n_users, dtype=torch.int32, device=self.device) if user_ids is None
                         else user_ids.to(device=self.device, dtype=torch.int32).contiguous())
        self.weight_sums: Optional[torch.Tensor] = None     # accumulated attention weight per key (see observe)

    def bytes_per_key(self) -> int:
        return 2 * (_NBYTES_NIBBLE + _NBYTES_QJL + 4) if self.v_qjl is not None else 2 * _NBYTES_NIBBLE + _NBYTES_QJL + 4

    def append(self, k_new: torch.Tensor, v_new: torch.Tensor, rotate: bool = True) -> None:
        """Quantize-append ``(n_users, n_kv_heads, T_new, 128)`` keys and values for every
        user at its current length."""
        T = k_new.shape[2]
        if self._append_together(k_new, v_new, T, rotate):
            return
        if int(self.lens.max()) + T > self.max_len:
            raise ValueError("append would run past the cache capacity")
        self._forget_sums(T)
        rotate_quantize_append(k_new, self.k_nib, self.k_qjl, self.k_norms, self.lens, self.codebooks,
                               self.user_ids, rotate=rotate)
        rotate_quantize_append(v_new, self.v_nib, self.v_qjl, self.v_norms, self.lens, self.codebooks,
                               self.user_ids, rotate=rotate)
        if self.pair_v:
            pair_v_rows(self.v_nib, self.lens, self.lens + T)
        self.lens += T
        self.lens32.copy_(self.lens)

    def _append_together(self, k_new, v_new, T: int, rotate: bool) -> bool:
        """The whole append as one library call behind one check of the lengths (``omni_kv_append``: both codec passes in
        one launch, the pair layout and the new lengths after them), for keys and values of one shape and dtype and the
        cache's own tensors as the constructor made them.  False: nothing was done, the general path takes the call.
        (Separate calls wait for the device five times to check the lengths and launch six kernels: one token for 64
        users, appended and attended to, 233 us against 96 us.)"""
        n, H, S, _ = self.k_nib.shape
        dev = self.k_nib.device
        packed = [(self.k_nib, _NBYTES_NIBBLE), (self.k_qjl, _NBYTES_QJL), (self.v_nib, _NBYTES_NIBBLE), (self.v_qjl, _NBYTES_QJL)]
        norms = [self.k_norms, self.v_norms]
        if not (dev.type == "cuda" and T > 0 and n > 0 and k_new.shape == v_new.shape == (n, H, T, HEAD_DIM)
                and k_new.dtype == v_new.dtype and k_new.dtype in _lib.DTYPE_CODE and k_new.device == v_new.device == dev
                and S == self.max_len and self.k_qjl is not None and self.k_norms is not None
                and (self.v_qjl is None) == (self.v_norms is None)
                and all(t is None or (t.shape == (n, H, S, w) and t.dtype is torch.uint8) for t, w in packed)
                and all(t is None or (t.shape == (n, H, S) and t.dtype is torch.float32) for t in norms)
                and self.lens.shape == self.lens32.shape == (n,) and self.lens.dtype is torch.int64 and self.lens32.dtype is torch.int32
                and all(t is None or (t.device == dev and t.is_contiguous())
                        for t in [t for t, _ in packed] + norms + [self.lens, self.lens32])
                and not torch.cuda.is_current_stream_capturing()):
            return False
        lo, hi = _lib.index_range(self.lens)
        if hi + T > self.max_len or lo < 0:
            raise ValueError("append would run past the cache capacity")
        self._forget_sums(T)
        lib = _lib.ensure_init(dev)
        k_new, v_new = _codec_rows(k_new), _codec_rows(v_new)
        cb, per_head = _prep_codebooks(self.codebooks, H, dev)
        ids, uid = _user_args(self.user_ids, n, dev)
        strides = [(C.c_int64 * 3)(*t.stride()[:3]) for t in (k_new, v_new)]
        with _lib.on_device(dev):
            _lib.check(lib.omni_kv_append(
                _lib.ptr(k_new), _lib.ptr(v_new), _lib.DTYPE_CODE[k_new.dtype], int(bool(rotate)), _lib.ptr(cb), per_head,
                _lib.ptr(ids), uid, n, H, T, strides[0], strides[1],
                _lib.ptr(self.k_nib), _lib.ptr(self.k_qjl), _lib.ptr(self.k_norms), _lib.ptr(self.v_nib), _lib.ptr(self.v_qjl),
                _lib.ptr(self.v_norms), S, _lib.ptr(self.lens), _lib.ptr(self.lens32), int(self.pair_v), _lib.stream_ptr(dev)))
        return True

    def _forget_sums(self, T: int) -> None:
        """No weight has reached the T keys that every user is about to get, whatever stood in their rows before: ``lens`` may
        have been set back, for another continuation or another prompt."""
        sums = self.weight_sums
        if sums is None or T == 0:
            return
        if sums.shape != (self.n_users, self.n_kv_heads, self.max_len) or sums.dtype is not torch.float32 or not sums.is_contiguous():
            raise ValueError(f"weight_sums must be contiguous float32 {(self.n_users, self.n_kv_heads, self.max_len)}, got {tuple(sums.shape)} {sums.dtype}")
        dev = _lib.require_cuda(sums)
        lens = _lib.as_device(self.lens, dev, torch.int64)
        with _lib.on_device(dev):
            _lib.check(_lib.load().omni_clear_new_sums(_lib.ptr(sums), _lib.ptr(lens), *sums.shape, T, _lib.stream_ptr(dev)))

    def _capturing(self) -> bool:
        return self.device.type == "cuda" and torch.cuda.is_current_stream_capturing()

    def prefill(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, prompt_lens: Optional[torch.Tensor] = None, *,
                causal: bool = True, scale: Optional[float] = None, rotate: bool = True) -> torch.Tensor:
        """Take in every user's prompt: ``prompt_attn`` of ``q`` (n_users, n_heads, T, 128) over ``k`` and ``v`` (n_users,
        n_kv_heads, T, 128) in full precision, and the keys and values packed into the (empty) cache.  ``prompt_lens`` (n_users,):
        user b's prompt is its first ``prompt_lens[b]`` rows; the others are neither attended to nor kept (the longest prompt has to
        fit the cache, its padding need not).  Returns the attention's result, zeros in the rows behind a prompt."""
        T = longest = k.shape[2]
        lens = None
        if prompt_lens is not None:
            if prompt_lens.shape != (self.n_users,):
                raise ValueError(f"prompt_lens must have shape ({self.n_users},), got {tuple(prompt_lens.shape)}")
            lens = prompt_lens.to(device=self.device, dtype=torch.int64)
            lo, longest = _lib.index_range(lens) if self.n_users else (0, 0)
            if lo < 0 or longest > T:
                raise ValueError(f"prompt_lens must lie in [0, {T}]")
        if longest > self.max_len:
            raise ValueError("prefill would run past the cache capacity")
        if self.n_users and _lib.index_range(self.lens) != (0, 0):
            raise ValueError("prefill takes whole prompts: the cache already holds keys")
        out = prompt_attn(q, k, v, seq_lens=lens, causal=causal, scale=scale)
        self.append(k[:, :, :longest], v[:, :, :longest], rotate=rotate)           # rows behind the longest prompt are nobody's
        if lens is not None:
            if self.pair_v:                        # groups that are not complete below the prompt's length go back to single rows
                pair_v_rows(self.v_nib, lens, self.lens)
            self.lens.copy_(lens)
            self.lens32.copy_(lens)
        return out

    def observe(self, q: torch.Tensor, scale: Optional[float] = None, with_qjl: bool = True, rotate_q: bool = False,
                causal: bool = True) -> torch.Tensor:
        """Add the attention weight that every cached key receives from ``q`` (n_users, n_heads, T, 128), the queries of the last T
        tokens, to ``weight_sums`` (float32 (n_users, n_kv_heads, max_len), kept from the first call on; new keys begin with
        zero), which decides what :meth:`evict` keeps.  Arguments as in :meth:`attend`; returns ``weight_sums``.  A CUDA graph may
        hold every call but the first."""
        if self.weight_sums is None:
            if self._capturing():                  # the zeros would be part of the graph, and every replay would start from them
                raise RuntimeError("the first observe makes weight_sums: call it once before the capture")
            self.weight_sums = torch.zeros(self.n_users, self.n_kv_heads, self.max_len, dtype=torch.float32, device=self.device)
        return attn_weight_sums(q, self.k_nib, self.k_qjl, self.k_norms, self.codebooks, self.user_ids, scale, with_qjl,
                                seq_lens=self.lens32, rotate_q=rotate_q, causal=causal, into=self.weight_sums)

    def evict(self, budget: int, recent: int = 0, max_len: Optional[int] = None) -> torch.Tensor:
        """Keep at most ``budget`` keys per user and head: the ``recent`` last ones and the heaviest others by ``weight_sums``
        (without a call of :meth:`observe`, the first ones).  The kept rows move into new arrays of ``max_len`` rows (the cache's
        present capacity when ``None``; a smaller one gives memory back), their sums with them.  Returns the kept keys' old
        positions, int32 (n_users, n_kv_heads, budget), -1 behind a user's keys.  Calls captured on the old arrays
        (``GraphedAttention``, ``HostDecodeStep``) have to be made anew, and the call itself takes no part in a capture."""
        if self._capturing():                      # the new arrays would hold nothing until a replay, and every replay would move old rows
            raise RuntimeError("evict replaces the cache's arrays: it cannot be captured (evict_keys can)")
        capacity = self.max_len if max_len is None else int(max_len)
        sums = self.weight_sums
        if sums is None:
            sums = torch.zeros(self.n_users, self.n_kv_heads, self.max_len, dtype=torch.float32, device=self.device)
        kept: EvictedCache = evict_keys(sums, self.k_nib, self.k_qjl, self.k_norms, self.v_nib, budget, recent=recent, seq_lens=self.lens32,
                                        v_qjl=self.v_qjl, v_norms=self.v_norms, v_paired=self.pair_v, capacity=capacity)
        self.k_nib, self.k_qjl, self.k_norms, self.v_nib = kept.k_nibbles, kept.k_qjl, kept.k_norms, kept.v_nibbles
        self.v_qjl, self.v_norms, self.max_len = kept.v_qjl, kept.v_norms, capacity
        if self.weight_sums is not None:
            self.weight_sums = kept.sums
        self.lens32.copy_(kept.seq_lens)
        self.lens.copy_(kept.seq_lens)
        return kept.index

    def attend(self, q: torch.Tensor, scale: Optional[float] = None, with_qjl: bool = True,
               rotate_q: bool = False, unrotate_out: bool = False, n_splits: Optional[int] = None) -> torch.Tensor:
        """Decode attention of ``q`` (n_users, n_heads, T, 128) against each user's valid prefix."""
        if scale is None:
            scale = 1.0 / math.sqrt(HEAD_DIM)
        return _qattn(q, self.k_nib, self.k_qjl, self.k_norms, self.v_nib, self.codebooks, self.user_ids, scale,
                      with_qjl, seq_lens=self.lens32, rotate_q=rotate_q, unrotate_out=unrotate_out, n_splits=n_splits,
                      v_paired=self.pair_v)


class HostDecodeStep:
    """One serving step with HOST buffers (``omni_qattn_decode_host``): the query comes from host memory, the fused
    attention runs over the resident cache, the result lands in page-locked host memory.  With a page-locked query
    tensor the kernels read and write the host buffers themselves (``mode == "direct"``: the transfer overlaps the
    attention work, one launch); a pageable query tensor is staged through device buffers in user chunks whose
    copies and kernels overlap on two internal streams (``"staged"``; ``OMNI_HOST_STEP=staged`` forces it).  The
    cache tensors must be complete before the first call (the internal streams do not wait on the caller's
    stream)."""

    def __init__(self, k_nib, k_qjl, k_norms, v_nib, codebooks, n_heads: int, batch: int, q_dtype=torch.bfloat16,
                 user_id=0, seq_lens=None, cache_slots=None, scale: Optional[float] = None, with_qjl: bool = True,
                 T: int = 1, n_chunks: Optional[int] = None, n_splits: Optional[int] = None, v_paired: bool = False):
        self.dev = _lib.require_cuda(k_nib, k_qjl, k_norms, v_nib)
        self.lib = _lib.ensure_init(self.dev)
        self.k_nib, self.k_qjl, self.k_norms, self.v_nib = k_nib, k_qjl, k_norms, v_nib
        n_slots, self.Hkv, self.S, _ = k_nib.shape
        if cache_slots is None and n_slots != batch:
            raise ValueError(f"cache holds {n_slots} users but the step batch is {batch}")
        self.cb, self.per_head = _prep_codebooks(codebooks, self.Hkv, self.dev)
        self.B, self.Hq, self.T, self.q_dtype = batch, n_heads, T, q_dtype
        if isinstance(user_id, torch.Tensor):
            self.ids, self.uid = user_id.to(device=self.dev, dtype=torch.int32).contiguous(), 0
        else:
            self.ids, self.uid = None, int(user_id) % 1024
        self.lens = None if seq_lens is None else seq_lens.to(device=self.dev, dtype=torch.int32).contiguous()
        self.slots = None if cache_slots is None else cache_slots.to(device=self.dev, dtype=torch.int32).contiguous()
        self.scale = float(scale if scale is not None else 1.0 / math.sqrt(HEAD_DIM))
        if n_chunks is None:                       # chunks of at least ~2k users keep every SM busy
            n_chunks = max(1, min(8, batch // 2048))
        self.with_qjl, self.n_chunks, self.v_paired = int(bool(with_qjl)), int(n_chunks), int(bool(v_paired))
        per_chunk = -(-batch // self.n_chunks)
        self.n_splits = int(n_splits) if n_splits is not None else _auto_splits(per_chunk, n_heads, self.Hkv, T, self.S, seq_lens is not None)
        self.ws_bytes = 2 * self.lib.omni_qattn_workspace_bytes(per_chunk, n_heads, T, self.n_splits)
        self.ws = torch.empty(max(self.ws_bytes // 4, 1), dtype=torch.float32, device=self.dev)
        shape = (batch, n_heads, T, HEAD_DIM)
        self.q_stage = self.out_stage = None            # device staging: allocated when a step first needs it
        self.mode = None                                # "direct" / "staged": how the last step moved its data
        self.q_host = torch.empty(shape, dtype=q_dtype).pin_memory()
        self.out_host = torch.empty(shape, dtype=torch.float32).pin_memory()
        self.h2d_bytes = self.q_host.numel() * self.q_host.element_size()
        self.d2h_bytes = self.out_host.numel() * 4
        torch.cuda.synchronize(self.dev)

    def step(self, q_host: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Runs one step; returns the pinned host result tensor (overwritten by the next step)."""
        src = self.q_host if q_host is None else q_host
        if src.is_cuda or src.shape != self.q_host.shape or src.dtype != self.q_dtype or not src.is_contiguous():
            raise ValueError("q_host must be a contiguous CPU tensor of the step's shape and dtype")
        direct = src.is_pinned() and not os.environ.get("OMNI_HOST_STEP", "").startswith("s")
        self.mode = "direct" if direct else "staged"
        if not direct and self.q_stage is None:
            self.q_stage = torch.empty(self.q_host.shape, dtype=self.q_dtype, device=self.dev)
            self.out_stage = torch.empty(self.q_host.shape, dtype=torch.float32, device=self.dev)
        with torch.cuda.device(self.dev):
            _lib.check(self.lib.omni_qattn_decode_host(
                _lib.ptr(src), _lib.DTYPE_CODE[self.q_dtype], _lib.ptr(self.q_stage),
                _lib.ptr(self.k_nib), _lib.ptr(self.k_qjl), _lib.ptr(self.k_norms), _lib.ptr(self.v_nib),
                _lib.ptr(self.cb), self.per_head, _lib.ptr(self.ids), self.uid, _lib.ptr(self.lens), _lib.ptr(self.slots),
                self.B, self.Hq, self.Hkv, self.T, self.S, self.Hkv * self.S, self.S, self.scale, self.with_qjl,
                self.v_paired, _lib.ptr(self.out_stage), _lib.ptr(self.out_host), self.n_chunks,
                self.n_splits, _lib.ptr(self.ws), self.ws_bytes, _lib.ptr(_lib.status_word(self.dev))))
        return self.out_host


class GraphedAttention:
    """``omni_attn`` on fixed device buffers, captured once into a CUDA graph and replayed per query.

    Small decode calls (the reference benchmark's 64-user query is 20 us of device work behind about as much host
    work: Python, two or three kernel launches) are bound by the host when issued one by one; a replayed graph costs
    one launch.  The query (and, with adapters, the hidden state and adapter indices) lives in buffers owned by this
    object: write into ``q`` / ``x`` / ``lora_indices`` (or pass tensors to ``__call__``, which copies them in) and
    read the result from ``out``, which the next replay overwrites.  Everything else -- cache tensors, codebooks,
    per-user lengths, adapter stacks -- is captured by address, so in-place changes of their contents are seen and the
    tensors must stay alive (this object keeps references)."""

    def __init__(self, q_shape, q_dtype, k_nibbles, k_qjl, k_norms, v_nibbles, codebooks, user_id=0, *, hidden=None,
                 lora_a=None, lora_b=None, lora_alpha: float = 1.0, **attn_kwargs):
        from .kernels.fused_attention import omni_attn
        dev = _lib.require_cuda(k_nibbles, k_qjl, k_norms, v_nibbles)
        # a replay reads the addresses the capture saw: an argument the call would have to convert (other device,
        # dtype or layout) would be captured as a temporary copy, so every tensor must already be in its final form
        final = [("k_nibbles", k_nibbles, torch.uint8), ("k_qjl", k_qjl, torch.uint8), ("k_norms", k_norms, torch.float32),
                 ("v_nibbles", v_nibbles, torch.uint8), ("codebooks", codebooks, torch.float32),
                 ("lora_a", lora_a, torch.float32), ("lora_b", lora_b, torch.float32),
                 ("seq_lens", attn_kwargs.get("seq_lens"), torch.int32), ("cache_slots", attn_kwargs.get("cache_slots"), torch.int32),
                 ("user_id", user_id if isinstance(user_id, torch.Tensor) else None, torch.int32)]
        for name, t, dt in final:
            if t is not None and not (t.device == dev and t.dtype is dt and t.is_contiguous()):
                raise ValueError(f"GraphedAttention: {name} must be a contiguous {dt} tensor on {dev}")
        B, _, T, _ = q_shape
        self.q = torch.zeros(q_shape, dtype=q_dtype, device=dev)
        self.x = self.lora_indices = None
        lora = {}
        if lora_a is not None:
            self.x = torch.zeros(B, T, lora_a.shape[2] if hidden is None else hidden, dtype=torch.float32, device=dev)
            self.lora_indices = torch.full((B,), -1, dtype=torch.int32, device=dev)
            lora = dict(x=self.x, lora_a=lora_a, lora_b=lora_b, lora_indices=self.lora_indices, lora_alpha=lora_alpha)
        self._keep = (k_nibbles, k_qjl, k_norms, v_nibbles, codebooks, user_id, lora_a, lora_b, attn_kwargs)

        def call():
            return omni_attn(self.q, k_nibbles, k_qjl, k_norms, v_nibbles, codebooks, user_id=user_id, **lora, **attn_kwargs)

        side = torch.cuda.Stream(device=dev)
        side.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(side):
            for _ in range(2):                      # first-call set-up (kernel attributes, tensor maps, workspace) is not captured
                call()
        torch.cuda.current_stream(dev).wait_stream(side)
        torch.cuda.synchronize(dev)
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph):
            self.out = call()

    def __call__(self, q=None, x=None, lora_indices=None) -> torch.Tensor:
        if q is not None:
            self.q.copy_(q, non_blocking=True)
        if x is not None:
            self.x.copy_(x, non_blocking=True)
        if lora_indices is not None:
            self.lora_indices.copy_(lora_indices, non_blocking=True)
        self.graph.replay()
        return self.out
