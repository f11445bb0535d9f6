"""``prompt_attn`` beside infinities and NaN: what belongs in a result stays in it, without a second pass over the keys, and what a row
must not see is kept out of it, over many tiles."""
import pytest
import torch

from tests import dense_reference as dense
from tests.helpers import device_us

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SCALE = 1.0 / 128 ** 0.5
NAN, INF = float("nan"), float("inf")


def inputs(B, Hq, Hkv, T, dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [(torch.randn(B, H, T, 128, generator=g, device=DEV) * s).to(dtype) for H, s in ((Hq, 1.5), (Hkv, 1.5), (Hkv, 1.0))]


def check(q, k, v, spans, causal=True, **lengths):
    """Rows and dims that a NaN of their own query, or a NaN or infinity of a visible key or value reaches are not finite; all others are
    what they are without any of these."""
    from omnistack_rs_b200.kernels.prompt_attention import prompt_attn
    got = prompt_attn(q, k, v, causal=causal, **lengths)
    want, tol = dense.prompt(*[torch.nan_to_num(x, nan=0.0, posinf=0.0, neginf=0.0) for x in (q, k, v)], spans, causal, SCALE)
    G = q.shape[1] // k.shape[1]
    touched = torch.zeros(q.shape, dtype=torch.bool, device=DEV)
    for b, r0, n in spans:
        if n == 0:
            continue
        bad = ~torch.isfinite(v[b, :, r0:r0 + n]) | ~torch.isfinite(k[b, :, r0:r0 + n]).all(-1, keepdim=True)
        bad = bad.int().cummax(1).values.bool() if causal else bad.any(1, keepdim=True).expand_as(bad)
        touched[b, :, r0:r0 + n] = bad.repeat_interleave(G, 0) | ~torch.isfinite(q[b, :, r0:r0 + n]).all(-1, keepdim=True)
    assert not bool(torch.isfinite(got[touched]).any())
    assert bool(((got.double() - want).abs() <= tol)[~touched].all())
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("Hq,Hkv", [(8, 2), (3, 1), (16, 1), (2, 2)])
def test_values_here_and_there(dtype, Hq, Hkv):
    """Early values that belong in most rows next to late ones that share a tile with rows in front of them, in other dims."""
    lens = [700, 0, 130, 1, 389]
    T = sum(lens)
    ends = torch.tensor([0] + lens).cumsum(0)
    spans = [(0, int(e) - n, n) for e, n in zip(ends[1:], lens)]
    q, k, v = inputs(1, Hq, Hkv, T, dtype, seed=1)
    v[0, 0, 3, 5], v[0, 0, 600, 7], v[0, -1, 699, 127], v[0, 0, 690, 64] = NAN, NAN, INF, -INF
    v[0, 0, 700, 0], v[0, 0, 829, 1] = INF, NAN
    v[0, -1, 831, 2:9], v[0, -1, 1100, 100] = NAN, INF
    for causal in (True, False):
        check(q, k, v, spans, causal, cu_seqlens=ends.to(device=DEV, dtype=torch.int32))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_everything_is_nan_or_infinite_from_some_token_on(dtype):
    T = 1100
    for start in (0, 1, 127, 500, 1099):
        for name, fill in (("v", NAN), ("v", INF), ("k", NAN), ("q", NAN)):
            q, k, v = inputs(1, 4, 2, T, dtype, seed=start)
            dict(q=q, k=k, v=v)[name][0, :, start:] = fill
            check(q, k, v, [(0, 0, T)])
    q, k, v = inputs(1, 4, 2, T, dtype, seed=7)                          # infinities of both signs cancel to NaN
    v[0, :, 40], v[0, :, 900] = INF, -INF
    out = check(q, k, v, [(0, 0, T)])
    assert bool(torch.isnan(out[0, :, 900:]).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_padding_of_a_batch(dtype):
    lens = [640, 0, 333, 128, 129, 1]
    q, k, v = inputs(6, 8, 2, 640, dtype, seed=2)
    for b, n in enumerate(lens):
        for x, fill in ((q, NAN), (k, INF), (v, NAN if b % 2 else INF)):
            x[b, :, n:] = fill
    for causal in (True, False):
        check(q, k, v, [(b, 0, n) for b, n in enumerate(lens)], causal, seq_lens=torch.tensor(lens, device=DEV))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_scores_of_minus_infinity(dtype):
    """Keys that every query scores minus infinity weigh nothing beside others, and rows that see no others are NaN."""
    from omnistack_rs_b200.kernels.prompt_attention import prompt_attn
    T, shut = 700, 300
    q, k, v = inputs(1, 4, 2, T, dtype, seed=3)
    q[..., 9] = q[..., 9].abs() + 0.1
    k[:, :, :shut, 9] = -INF
    out = prompt_attn(q, k, v)
    assert bool(torch.isnan(out[:, :, :shut]).all())
    Q, K, V = q.double(), torch.nan_to_num(k, neginf=0.0).double().repeat_interleave(2, 1), v.double().repeat_interleave(2, 1)
    s = Q @ K.transpose(-1, -2) * SCALE
    closed = torch.ones(T, T, device=DEV, dtype=torch.bool).triu(1)
    closed[:, :shut] = True
    w = torch.softmax(s.masked_fill(closed, -INF)[:, :, shut:], -1)
    want = w @ V
    from tests import operator_reference as ref
    reach = (Q.abs() @ K.abs().transpose(-1, -2)).amax(-1)[:, :, shut:] * SCALE
    tol = ref.prompt_tolerance(dtype, w @ V.abs(), reach, want, T)
    assert bool(((out[:, :, shut:].double() - want).abs() <= tol).all())


@pytest.mark.parametrize("where,at", [("v", 0), ("v", 2000), ("k", 0), ("q", 0), ("-k", 0)])
def test_nan_that_belongs_there_costs_no_second_pass(where, at):
    """A NaN in an early token is in nearly every row's result, and is no reason to form the rows again: key by key that took 330
    times as long as the call (21 ms).  (A NaN value is looked for among the row's values, a read of them.)"""
    from omnistack_rs_b200.kernels.prompt_attention import prompt_attn
    q, k, v = inputs(1, 8, 2, 4096, torch.bfloat16, seed=4)
    clean = device_us(lambda: prompt_attn(q, k, v), calls=3, replays=3)
    if where == "q":
        q[...] = NAN
    elif where == "-k":                                                  # the first block's scores are all minus infinity
        q[..., 0] = q[..., 0].abs() + 0.1
        k[:, :, :200, 0] = -INF
    else:
        dict(v=v, k=k)[where][:, :, at, 3] = NAN
    assert device_us(lambda: prompt_attn(q, k, v), calls=3, replays=3) < 8 * clean
