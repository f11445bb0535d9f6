"""``prompt_attn`` with many more work items than SMs, so that a CTA goes on from item to item: hundreds of ragged prompts, heads that
fill a tile and heads that do not, rows in front of the first prompt and behind the last."""
import pytest
import torch

from tests import dense_reference as dense

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SCALE = 1.0 / 128 ** 0.5


def inputs(B, Hq, Hkv, T, dtype, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [(torch.randn(B, H, T, 128, generator=g, device=DEV) * s).to(dtype) for H, s in ((Hq, 1.5), (Hkv, 1.5), (Hkv, 1.0))]


def compare(out, want, tol):
    err = (out.double() - want).abs() - tol                              # rows of no prompt: zeros, exactly
    assert bool((err <= 0).all()), f"{float(err.max())} over the bound"


def ragged(n, longest, seed):
    """n lengths, a tenth of them zero and a tenth of them short of, at and past the 32 tokens of a tile of four heads."""
    g = torch.Generator().manual_seed(seed)
    lens = torch.randint(1, longest + 1, (n,), generator=g)
    lens[torch.randperm(n, generator=g)[:n // 10]] = 0
    edge = torch.randperm(n, generator=g)[:n // 10]
    lens[edge] = torch.tensor([1, 31, 32, 33, 64, 65, 127, 128, 129])[torch.arange(len(edge)) % 9].clamp(max=longest)
    return lens.tolist()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("Hq,Hkv,causal", [(32, 8, True), (32, 8, False), (17, 1, True), (12, 4, True)])
@pytest.mark.parametrize("n,longest", [(40, 400), (255, 60), (256, 60), (400, 50)])
def test_packed(dtype, Hq, Hkv, causal, n, longest):
    from omnistack_rs_b200.kernels.prompt_attention import prompt_attn
    lens = ragged(n, longest, seed=n)
    first, behind = 5, 77
    ends = torch.tensor([first] + lens).cumsum(0)
    T = int(ends[-1]) + behind
    q, k, v = inputs(1, Hq, Hkv, T, dtype, seed=n + Hq)
    out = prompt_attn(q, k, v, cu_seqlens=ends.to(device=DEV, dtype=torch.int32), causal=causal)
    spans = [(0, int(e) - m, m) for e, m in zip(ends[1:], lens)]
    compare(out, *dense.prompt(q, k, v, spans, causal, SCALE))
    assert torch.equal(out, prompt_attn(q, k, v, cu_seqlens=ends.to(device=DEV, dtype=torch.int32), causal=causal))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("causal", [True, False])
def test_padded(dtype, causal):
    from omnistack_rs_b200.kernels.prompt_attention import prompt_attn
    B, T = 40, 300
    lens = ragged(B, T, seed=3)
    q, k, v = inputs(B, 32, 8, T, dtype, seed=4)
    out = prompt_attn(q, k, v, seq_lens=torch.tensor(lens, device=DEV), causal=causal)
    compare(out, *dense.prompt(q, k, v, [(b, 0, n) for b, n in enumerate(lens)], causal, SCALE))


@pytest.mark.parametrize("order", ["long prompts first", "long prompts last"])
def test_long_among_short(order):
    """The ring of keys and the parities of its stages are carried over between items of one block and of many."""
    from omnistack_rs_b200.kernels.prompt_attention import prompt_attn
    lens = [2000, 1, 1300] + [7, 40, 0, 129] * 40
    if order == "long prompts last":
        lens = lens[::-1]
    ends = torch.tensor([0] + lens).cumsum(0)
    q, k, v = inputs(1, 16, 4, int(ends[-1]), torch.bfloat16, seed=6)
    out = prompt_attn(q, k, v, cu_seqlens=ends.to(device=DEV, dtype=torch.int32))
    compare(out, *dense.prompt(q, k, v, [(0, int(e) - m, m) for e, m in zip(ends[1:], lens)], True, SCALE))
