"""``prompt_attn`` on scores so large that one step of fp32 is many powers of two: nothing overflows, the largest score wins."""
import pytest
import torch

from tests import operator_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SCALE = 1.0 / 128 ** 0.5


@pytest.mark.parametrize("dtype,size", [(torch.float16, 300), (torch.float16, 1500), (torch.float16, 5000), (torch.float16, 12000), (torch.bfloat16, 5000),
                                        (torch.bfloat16, 1e8), (torch.bfloat16, 1e16), (torch.float32, 5000), (torch.float32, 1e16)])
@pytest.mark.parametrize("causal", [False, True])
def test_one_key_takes_all(dtype, size, causal):
    from omnistack_rs_b200.kernels.prompt_attention import prompt_attn
    T = 700
    g = torch.Generator(device=DEV).manual_seed(3)
    q, k, v = (torch.randn(1, h, T, 128, generator=g, device=DEV) for h in (8, 2, 2))
    q, k, v = (q * size).to(dtype), (k * size).to(dtype), v.to(dtype)
    assert bool(torch.isfinite(q).all()) and bool(torch.isfinite(k).all())
    out = prompt_attn(q, k, v, causal=causal)
    Q, K, V = q.double(), k.double().repeat_interleave(4, 1), v.double().repeat_interleave(4, 1)
    s, size = Q @ K.transpose(-1, -2) * SCALE, Q.abs() @ K.abs().transpose(-1, -2) * SCALE
    if causal:
        s, size = s + torch.full((T, T), float("-inf"), device=DEV, dtype=torch.float64).triu(1), size.tril()
    top = s.topk(2, -1)
    # 130 roundings of 2^-24 in each of two scores, and e^-40 for all others together
    sure = (top.values[..., 0] - top.values[..., 1]) > 2 * 130 * 2.0 ** -24 * size.amax(-1) + 40
    want = torch.gather(V, 2, top.indices[..., :1].expand(1, 8, T, 128))
    assert int(sure.sum()) > 0.9 * 8 * T
    assert bool(torch.isfinite(out).all())
    assert bool(((out.double() - want).abs() <= 2 * ref.half_step(dtype) * want.abs() + 2.0 ** -20)[sure].all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_large_scores_that_are_alike(dtype):
    """All keys of a prompt score alike, far from zero: the mean of the values, whatever the size."""
    from omnistack_rs_b200.kernels.prompt_attention import prompt_attn
    T = 300
    g = torch.Generator(device=DEV).manual_seed(4)
    v = torch.randn(1, 1, T, 128, generator=g, device=DEV).to(dtype)
    for size in (1.0, 40.0, 1000.0, 4096.0, 20000.0):
        for sign in (1.0, -1.0):
            q = torch.full((1, 2, T, 128), size, dtype=dtype, device=DEV)
            k = torch.full((1, 1, T, 128), sign * size, dtype=dtype, device=DEV)
            out = prompt_attn(q, k, v)
            want = v.double().cumsum(2) / torch.arange(1, T + 1, device=DEV)[:, None]
            mass = v.double().abs().cumsum(2) / torch.arange(1, T + 1, device=DEV)[:, None]
            # equal scores have equal weights exactly: rounded once (half a step, and of their sum not), added in fp32
            tol = (2 * ref.half_step(dtype) + 2 * T * 2.0 ** -24) * mass + ref.half_step(dtype) * want.abs() + 2.0 ** -20
            assert bool(((out.double() - want).abs() <= tol).all())
