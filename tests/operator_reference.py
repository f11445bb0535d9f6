"""The prompt-side and eviction operators from their definitions, in 64 bits, for the GPU tests."""
from __future__ import annotations

import math

import torch

import oracle as orc

QJL_COEF = math.sqrt(2.0 / math.pi) / 128


def half_step(dtype) -> float:
    """Largest relative error of one rounding to ``dtype``."""
    return torch.finfo(dtype).eps / 2


def norm_rope(x, positions, inv_freq, weight, eps, axis_pairs, interleaved):
    """x (B, H, T, 128); positions (axes, B, T).  Returns the result and, per element, |y_u| + |y_v| of its pair."""
    y = x.double()
    if eps is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps)
        if weight is not None:
            y = y * weight.double()
    P = inv_freq.numel()
    axis = sum(([a] * n for a, n in enumerate(axis_pairs)), [])
    out, size = y.clone(), y.abs()
    for i in range(P):
        u, v = (2 * i, 2 * i + 1) if interleaved else (i, i + P)
        th = (positions[axis[i]].double() * inv_freq[i].double())[:, None]
        c, s = torch.cos(th), torch.sin(th)
        out[..., u] = y[..., u] * c - y[..., v] * s
        out[..., v] = y[..., v] * c + y[..., u] * s
        size[..., u] = size[..., v] = y[..., u].abs() + y[..., v].abs()
    return out, size


def prompt(q, k, v, spans, causal, scale):
    """spans: (b, first row, length) per prompt.  Returns the result, sum_j w_j |v_j| and, per row, the largest
    scale * sum_d |q_d k_d| (what errors of weights and scores are relative to)."""
    G = q.shape[1] // k.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64)
    mass = torch.zeros(q.shape, dtype=torch.float64)
    reach = torch.zeros(q.shape[:3], dtype=torch.float64)
    for b, r0, n in spans:
        for h in range(q.shape[1]):
            Q, K, V = (x.double()[r0:r0 + n] for x in (q[b, h], k[b, h // G], v[b, h // G]))
            for i in range(n):
                m = i + 1 if causal else n
                w = torch.softmax((K[:m] @ Q[i]) * scale, dim=0)
                out[b, h, r0 + i] = w @ V[:m]
                mass[b, h, r0 + i] = w @ V[:m].abs()
                reach[b, h, r0 + i] = (K[:m].abs() @ Q[i].abs()).max() * abs(scale)
    return out, mass, reach


def prompt_tolerance(dtype, mass, reach, out, n):
    """Error bound of one row of n keys.

    Scores: 128 products added in fp32 and the scaling, each step relative 2^-24, so |ds| <= 130 * 2^-24 * reach, and the
    exponential (2 ulp) adds 2^-22; a weight and the normaliser are both off by exp(ds) - 1 <= 2 ds.  Adding up n weights and n
    products in fp32: n * 2^-24 each.  16-bit types round every weight once more (half a step), and its sum is or is not of the
    rounded ones: at most two half steps.  The result is rounded once."""
    ds = 130 * 2.0 ** -24 * reach[..., None] + 2.0 ** -22
    rel = 4 * ds + 2 * n * 2.0 ** -24
    if dtype is not torch.float32:
        rel = rel + 2 * half_step(dtype)
    tiny = torch.finfo(dtype).smallest_normal
    return rel * mass + half_step(dtype) * (out.abs() + rel * mass) + tiny


def dequantized_keys(k_nib, k_qjl, k_norms, cb, user_ids, with_qjl):
    """(B, H, S, 128) fp64 keys from the packed rows."""
    B, H, S, _ = k_nib.shape
    codes = torch.stack([k_nib & 15, k_nib >> 4], -1).reshape(B, H, S, 128).long()
    k = torch.stack([(cb if cb.dim() == 1 else cb[h]).double()[codes[:, h]] for h in range(H)], 1)
    if with_qjl:
        bits = (k_qjl[..., None] >> torch.arange(8, dtype=torch.uint8)) & 1
        sign = bits.reshape(B, H, S, 64).double() * 2 - 1
        for b in range(B):
            for h in range(H):
                G = orc.rademacher_matrix(orc.qjl_seed(int(user_ids[b]), h)).double()
                k[b, h] += k_norms[b, h, :, None].double() * QJL_COEF * (sign[b, h] @ G)
    return k


def weight_sums(q, keys, lens, scale, causal):
    """Returns the sums and, per (b, h), a bound of their relative error (see the tests)."""
    B, Hq, T, _ = q.shape
    H, S = keys.shape[1:3]
    out = torch.zeros(B, H, S, dtype=torch.float64)
    reach = torch.zeros(B, H, dtype=torch.float64)
    for b in range(B):
        for hq in range(Hq):
            h = hq // (Hq // H)
            for t in range(T):
                n = int(lens[b])
                m = n - T + t + 1 if causal else n
                if m <= 0:
                    continue
                K = keys[b, h, :m]
                out[b, h, :m] += torch.softmax((K @ q[b, hq, t].double()) * scale, dim=0)
                reach[b, h] = max(reach[b, h], float((K.abs() @ q[b, hq, t].double().abs()).max()) * abs(scale))
    return out, reach


def pair_rows(v, lens):
    """The pair layout of V's nibble rows for whole groups of eight below the length (its own inverse)."""
    out = v.clone()
    for b in range(v.shape[0]):
        for g in range(int(lens[b]) // 8):
            for first in (0, 1, 4, 5):
                f, s = v[b, :, 8 * g + first], v[b, :, 8 * g + (first ^ 3)]
                out[b, :, 8 * g + first] = (f & 15) | ((s & 15) << 4)
                out[b, :, 8 * g + (first ^ 3)] = (f >> 4) | (s & 240)
    return out


def kept_positions(sums, n, budget, recent):
    """Positions that stay of one head's n keys, by plain sorting (NaN above everything, equal sums by position)."""
    if n <= budget:
        return list(range(n))
    rank = lambda i: (0.0, i) if math.isnan(sums[i]) else (1.0, -sums[i] if sums[i] else 0.0, i)  # noqa: E731
    head = sorted(range(n - recent), key=rank)[:budget - recent]
    return sorted(head) + list(range(n - recent, n))
