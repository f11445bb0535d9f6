"""``attn_weight_sums`` where a query is NaN, and where queries, centroids and norms are of sizes far apart."""
import pytest
import torch

from tests import dense_reference as dense

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SCALE = 1.0 / 128 ** 0.5


def packed(B, H, S, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    byte = lambda n: torch.randint(0, 256, (B, H, S, n), generator=g, device=DEV, dtype=torch.uint8)  # noqa: E731
    return byte(64), byte(8), torch.rand(B, H, S, generator=g, device=DEV) + 0.5, torch.sort(torch.randn(H, 16, generator=g, device=DEV), dim=1).values


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("G,T", [(2, 3), (1, 8), (2, 7), (4, 32), (1, 150)])
def test_a_nan_query_reaches_the_keys_it_sees(dtype, G, T):
    from omnistack_rs_b200.kernels.eviction import attn_weight_sums
    B, H, S = 3, 2, 400
    rows, lens, at = packed(B, H, S, T), [400, 130, T + 1], T // 2
    q = torch.randn(B, H * G, T, 128, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).to(dtype)
    q[1, 0, at, 5] = float("nan")                                         # one head of a group, one token
    q[2, :, at] = float("inf")
    seq = torch.tensor(lens, device=DEV)
    got = attn_weight_sums(q, *rows, seq_lens=seq)
    clean = torch.nan_to_num(q, nan=0.0, posinf=0.0)
    keys = dense.dequantized_keys(*rows, [0] * B, True)
    want, reach = dense.weight_sums(clean, keys, lens, SCALE, True)
    touched = torch.zeros(got.shape, dtype=torch.bool, device=DEV)
    touched[1, 0, :lens[1] - T + at + 1] = True
    touched[2, :, :lens[2] - T + at + 1] = True
    assert bool(torch.isnan(got[touched]).all()) and bool(touched.any()) and not bool(touched[1, 0, :lens[1]].all())
    rel = 4 * (52 * 2.0 ** -22 * reach[..., None] + 2.0 ** -22) + (S + G * T) * 2.0 ** -24       # as dense.check_weights
    assert bool(((got.double() - want).abs() <= rel * want + 1e-30)[~touched].all())
    into = torch.ones(got.shape, device=DEV)
    attn_weight_sums(q, *rows, seq_lens=seq, into=into)
    assert torch.equal(torch.isnan(into), torch.isnan(got)) and bool((into[1, 0, lens[1]:] == 1).all())
    every = attn_weight_sums(q, *rows, seq_lens=seq, causal=False)       # without the causal order it reaches all keys of its head
    assert bool(torch.isnan(every[1, 0, :130]).all()) and bool(torch.isfinite(every[1, 1]).all()) and bool((every[1, 0, 130:] == 0).all())


@pytest.mark.parametrize("T", [1, 12])
@pytest.mark.parametrize("q_size,cb_size,norm_size", [(1e-15, 1e-15, 1e8), (1e-15, 1e-15, 1e10), (1e-12, 1e-20, 1e11), (1e15, 1e-16, 1e-16), (1e-16, 1e15, 1e15)])
def test_sizes_far_apart(T, q_size, cb_size, norm_size):
    from omnistack_rs_b200.kernels.eviction import attn_weight_sums
    nib, qjl, norms, cb = packed(2, 2, 300, 3)
    norms, cb = norms * norm_size, cb * cb_size
    q = torch.randn(2, 4, T, 128, generator=torch.Generator(device=DEV).manual_seed(2), device=DEV) * q_size
    keys = dense.dequantized_keys(nib, qjl, norms, cb, [0, 0], True)
    got = attn_weight_sums(q, nib, qjl, norms, cb, seq_lens=torch.tensor([300, 77], device=DEV))
    dense.check_weights(got, q, keys, [300, 77], True, SCALE)
