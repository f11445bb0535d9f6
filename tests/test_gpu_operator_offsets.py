"""The prompt-side and eviction operators on tensors of more than 2^31 elements: the last users and prompts come out as on their own."""
import pytest
import torch

from tests import dense_reference as dense

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SCALE = 1.0 / 128 ** 0.5


@pytest.fixture(autouse=True)
def memory():
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB")
    yield
    torch.cuda.empty_cache()


def noise(seed, *shape, dtype=torch.bfloat16):
    out = torch.empty(shape, dtype=dtype, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(seed)
    return out.normal_(generator=g) if dtype.is_floating_point else out.random_(0, 256, generator=g)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_prompts_and_positions(dtype):
    from omnistack_rs_b200.kernels.position import qk_norm_rope
    from omnistack_rs_b200.kernels.prompt_attention import prompt_attn
    Hq, Hkv, n, each = 32, 8, 900, 610
    T = n * each + 77
    assert Hq * T * 128 > 2 ** 31
    q, k, v = noise(1, 1, Hq, T, 128, dtype=dtype), noise(2, 1, Hkv, T, 128, dtype=dtype), noise(3, 1, Hkv, T, 128, dtype=dtype)
    cu = (torch.arange(n + 1, device=DEV) * each).to(torch.int32)
    out = prompt_attn(q, k, v, cu_seqlens=cu)
    for first in (0, (n // 2) * each, (n - 1) * each):
        part = [x[:, :, first:first + each].contiguous() for x in (q, k, v)]
        assert torch.equal(out[:, :, first:first + each], prompt_attn(*part))
    assert bool((out[:, :, n * each:] == 0).all())
    del out, k, v
    positions, freq = torch.arange(T, device=DEV), 10000.0 ** (-torch.arange(64, device=DEV) / 64)
    y, _ = qk_norm_rope(q, None, positions, freq)
    assert torch.equal(y[:, -2:, -50:], qk_norm_rope(q[:, -2:, -50:].contiguous(), None, positions[-50:], freq)[0])


def test_padded_prompts_of_many_users():
    from omnistack_rs_b200.kernels.prompt_attention import prompt_attn
    B, Hq, T = 4500, 32, 130
    assert B * Hq * T * 128 > 2 ** 31
    q, k = noise(1, B, Hq, T, 128), noise(2, B, 8, T, 128)
    lens = torch.randint(0, T + 1, (B,), generator=torch.Generator().manual_seed(1))
    out = prompt_attn(q, k, k, seq_lens=lens.to(DEV))
    tail = [x[-3:].contiguous() for x in (q, k, k)]
    assert torch.equal(out[-3:], prompt_attn(*tail, seq_lens=lens[-3:].to(DEV)))


@pytest.mark.parametrize("T", [1, 16])
def test_weights_and_eviction(T):
    from omnistack_rs_b200.kernels.eviction import attn_weight_sums, evict_keys
    B, H, S = 70, 8, 65000
    assert B * H * S * 64 > 2 ** 31
    nib, qjl, norms = noise(1, B, H, S, 64, dtype=torch.uint8), noise(2, B, H, S, 8, dtype=torch.uint8), noise(3, B, H, S, dtype=torch.float32)
    cb, q = torch.sort(noise(4, H, 16, dtype=torch.float32), dim=1).values, noise(5, B, 2 * H, T, 128)
    lens = torch.full((B,), S, dtype=torch.int32, device=DEV)
    lens[-2], lens[-3] = 0, 31000
    sums = attn_weight_sums(q, nib, qjl, norms, cb, user_id=7, seq_lens=lens)
    for b in (0, B - 3, B - 1):
        keys = dense.dequantized_keys(nib[b:b + 1], qjl[b:b + 1], norms[b:b + 1], cb, [7], True)
        dense.check_weights(sums[b:b + 1], q[b:b + 1], keys, [int(lens[b])], True, SCALE)
        del keys
    v = noise(6, B, H, S, 64, dtype=torch.uint8)
    kept = evict_keys(sums, nib, qjl, norms, v, 5000, recent=10, seq_lens=lens, v_paired=True)
    last = evict_keys(*[x[-3:].contiguous() for x in (sums, nib, qjl, norms, v)], 5000, recent=10, seq_lens=lens[-3:], v_paired=True)
    assert all(torch.equal(x[-3:], y) for x, y in zip(kept, last) if x is not None)
