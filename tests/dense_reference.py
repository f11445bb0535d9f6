"""Prompt attention and key weights from their definitions in 64 bits as dense products, for calls too large for per-row loops.
They run on the device of their inputs."""
from __future__ import annotations

import functools

import torch

import oracle as orc
from tests import operator_reference as ref


@functools.lru_cache(maxsize=None)
def _sign_rows(seed):
    return orc.rademacher_matrix(seed).double()


def prompt(q, k, v, spans, causal, scale):
    """spans: (b, first row, length) per prompt.  Returns the result and the error bound of every element (``ref.prompt_tolerance``
    with each prompt's own length); rows of no prompt have zeros in both."""
    G = q.shape[1] // k.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    for b, r0, n in spans:
        if n == 0:
            continue
        Q = q[b, :, r0:r0 + n].double()
        K, V = (x[b, :, r0:r0 + n].double().repeat_interleave(G, 0) for x in (k, v))
        shut = torch.full((n, n), float("-inf"), dtype=torch.float64, device=q.device).triu(1) if causal else 0.0
        w = torch.softmax(Q @ K.transpose(-1, -2) * scale + shut, dim=-1)
        reach = Q.abs() @ K.abs().transpose(-1, -2)
        reach = (reach.tril() if causal else reach).amax(-1) * abs(scale)
        got = w @ V
        out[b, :, r0:r0 + n] = got
        tol[b, :, r0:r0 + n] = ref.prompt_tolerance(q.dtype, w @ V.abs(), reach, got, n)
    return out, tol


def dequantized_keys(k_nib, k_qjl, k_norms, cb, ids, with_qjl):
    """(B, H, S, 128) fp64 keys; cb (H, 16) or (16,), ids: a list."""
    B, H, S, _ = k_nib.shape
    codes = torch.stack([k_nib & 15, k_nib >> 4], -1).reshape(B, H, S, 128).long()
    k = torch.stack([(cb if cb.dim() == 1 else cb[h]).double()[codes[:, h]] for h in range(H)], 1)
    if with_qjl:
        bits = (k_qjl[..., None] >> torch.arange(8, dtype=torch.uint8, device=k.device)) & 1
        sign = bits.reshape(B, H, S, 64).double() * 2 - 1
        rows = torch.stack([torch.stack([_sign_rows(orc.qjl_seed(int(i), h)) for h in range(H)]) for i in ids]).to(k.device)
        k += k_norms[..., None].double() * ref.QJL_COEF * (sign @ rows)
    return k


def weight_sums(q, keys, lens, scale, causal):
    """Returns the sums and, per (b, h), the largest scale * sum_d |q_d k_d| (see ``check_weights``)."""
    B, Hq, T, _ = q.shape
    H, S = keys.shape[1:3]
    G = Hq // H
    out = torch.zeros(B, H, S, dtype=torch.float64, device=q.device)
    reach = torch.zeros(B, H, dtype=torch.float64, device=q.device)
    step = torch.arange(S, device=q.device)
    for b, n in enumerate(lens):
        if n == 0:
            continue
        t0 = max(0, T - n) if causal else 0                              # the first token that has a key
        Q, K = q[b].double().view(H, G, T, 128)[:, :, t0:].reshape(H, -1, 128), keys[b, :, :n]
        s = (Q @ K.transpose(-1, -2) * scale).view(H, G, T - t0, n)
        last = n - T + torch.arange(t0, T, device=q.device) if causal else torch.full((T - t0,), n - 1, device=q.device)
        open_ = step[None, :n] <= last[:, None]
        out[b, :, :n] = torch.softmax(s.masked_fill(~open_, float("-inf")), dim=-1).sum((1, 2))
        size = (Q.abs() @ K.abs().transpose(-1, -2)).view(H, G, T - t0, n) * open_
        reach[b] = size.amax((1, 2, 3)) * abs(scale)
    return out, reach


def check_weights(got, q, keys, lens, causal, scale):
    """Scores: centroids and queries may be split in two 11-bit parts (2^-22 each), 192 products and two factors in fp32
    (200 * 2^-24): |ds| <= 52 * 2^-22 * reach; the exponential adds 2^-22 and the normaliser the same again.  Adding up S weights of
    one column and the columns in fp32: (S + columns) * 2^-24."""
    want, reach = weight_sums(q, keys, lens, scale, causal)
    S, cols = want.shape[2], q.shape[1] // want.shape[1] * q.shape[2]
    rel = 4 * (52 * 2.0 ** -22 * reach[..., None] + 2.0 ** -22) + (S + cols) * 2.0 ** -24
    err = (got.double() - want).abs()
    assert bool((err <= rel * want + 1e-30).all()), float((err / (rel * want + 1e-30)).max())
    for b, n in enumerate(lens):
        assert bool((got[b, :, n:] == 0).all())
