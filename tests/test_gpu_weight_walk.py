"""``attn_weight_sums`` over many tiles of keys per CTA: users of uneven lengths, some of them empty, several heads and users in one
CTA's share, tables and columns that change on the way; rotated queries, one round of columns and two, captured calls."""
import pytest
import torch

from tests import dense_reference as dense

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SCALE = 1.0 / 128 ** 0.5


def packed(B, H, S, seed, per_head=True):
    g = torch.Generator(device=DEV).manual_seed(seed)
    byte = lambda n: torch.randint(0, 256, (B, H, S, n), generator=g, device=DEV, dtype=torch.uint8)  # noqa: E731
    cb = torch.sort(torch.randn(H, 16, generator=g, device=DEV), dim=1).values
    return byte(64), byte(8), torch.rand(B, H, S, generator=g, device=DEV) + 0.5, cb if per_head else cb[0].contiguous()


def uneven(B, S, seed):
    lens = torch.randint(S // 2, S + 1, (B,), generator=torch.Generator().manual_seed(seed))
    lens[::7] = 0
    lens[3::11] = torch.tensor([1, 127, 128, 129])[torch.arange(len(lens[3::11])) % 4]
    lens[-1] = S
    return lens.tolist()


def tiles(lens, heads):
    return heads * sum((n + 127) // 128 for n in lens)


def run(B, H, G, T, S, dtype, per_head, causal=True, with_qjl=True, rotate=False, seed=1):
    from omnistack_rs_b200.kernels.eviction import attn_weight_sums
    from omnistack_rs_b200.kernels.hadamard import rotate_queries
    rows = packed(B, H, S, seed, per_head)
    lens = uneven(B, S, seed)
    q = (torch.randn(B, H * G, T, 128, generator=torch.Generator(device=DEV).manual_seed(seed + 1), device=DEV) * 1.5).to(dtype)
    ids = [(b % 5) * 333 for b in range(B)]
    call = lambda **more: attn_weight_sums(q, *rows, user_id=torch.tensor(ids, dtype=torch.int32, device=DEV), with_qjl=with_qjl,  # noqa: E731
                                           seq_lens=torch.tensor(lens, device=DEV), causal=causal, rotate_q=rotate, **more)
    got = call()
    turned = rotate_queries(q.float()) if rotate else q
    keys = dense.dequantized_keys(*rows, ids, with_qjl)
    dense.check_weights(got, turned, keys, lens, causal, SCALE)
    assert torch.equal(got, call())
    return call, got, lens


@pytest.mark.parametrize("dtype,rotate", [(torch.bfloat16, False), (torch.float32, False), (torch.float16, True)])
@pytest.mark.parametrize("per_head", [True, False])
@pytest.mark.parametrize("G,T", [(4, 1), (1, 8), (3, 1)])
def test_few_columns(dtype, rotate, per_head, G, T):
    """Two CTAs per SM: more than 1,500 tiles are five or more for each, with heads of a dozen."""
    B, H, S = 70, 4, 1500
    assert tiles(uneven(B, S, 1), H) > 5 * 296
    run(B, H, G, T, S, dtype, per_head, rotate=rotate)
    run(B, H, G, T, S, dtype, per_head, causal=False, with_qjl=False, rotate=rotate)


@pytest.mark.parametrize("dtype,rotate", [(torch.bfloat16, False), (torch.float32, False), (torch.bfloat16, True), (torch.float16, True)])
@pytest.mark.parametrize("per_head", [True, False])
@pytest.mark.parametrize("G,T", [(1, 9), (2, 12), (4, 32), (2, 70)])
def test_many_columns(dtype, rotate, per_head, G, T):
    """One CTA per SM: about 1,550 tiles are ten for each; 140 columns take two rounds."""
    B, H, S = 52, 4, 1500
    assert tiles(uneven(B, S, 1), H) > 9 * 148
    call, got, lens = run(B, H, G, T, S, dtype, per_head, rotate=rotate)
    run(B, H, G, T, S, dtype, per_head, causal=False, with_qjl=False, rotate=rotate)
    if G * T <= 128:                                                     # one round: a single addition
        into = torch.full_like(got, 3.0)
        call(into=into)
        assert torch.equal(into, 3 + got)


@pytest.mark.parametrize("T", [1, 40])
def test_long_caches(T):
    """Heads whose tiles are spread over many CTAs, one token's weights over more than 1,025 keys among them."""
    run(2, 2, 4, T, 20011, torch.bfloat16, True)
    run(1, 1, 4, T, 33000, torch.float32, False, rotate=True)


@pytest.mark.parametrize("rotate", [False, True])
def test_captured_calls_of_many_columns(rotate):
    from omnistack_rs_b200.kernels.eviction import attn_weight_sums
    B, H, G, T, S = 9, 2, 4, 20, 900
    rows = packed(B, H, S, 5)
    q = torch.randn(B, H * G, T, 128, generator=torch.Generator(device=DEV).manual_seed(6), device=DEV).to(torch.bfloat16)
    lens = torch.tensor(uneven(B, S, 7), dtype=torch.int32, device=DEV)
    first = attn_weight_sums(q, *rows, seq_lens=lens, rotate_q=rotate)
    into, summed = torch.zeros_like(first), torch.zeros_like(first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = attn_weight_sums(q, *rows, seq_lens=lens, rotate_q=rotate)
        attn_weight_sums(q, *rows, seq_lens=lens, rotate_q=rotate, into=into)
    graph.replay()
    summed += first
    assert torch.equal(out, first) and torch.equal(into, summed)
    lens.copy_(torch.tensor([900, 0, 3, 0, 640, 128, 900, 1, 77], dtype=torch.int32))
    q.mul_(-0.7)
    graph.replay()
    again = attn_weight_sums(q, *rows, seq_lens=lens, rotate_q=rotate)
    summed += again
    assert torch.equal(out, again) and torch.equal(into, summed)
