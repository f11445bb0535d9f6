"""``prompt_attn`` against its definition in 64 bits: head groups, lengths, packing, padding, strides, masked NaN."""
import pytest
import torch

from tests import operator_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SCALE = 1.0 / 128 ** 0.5


def spans_of(lens, T, packed):
    if packed:
        ends = torch.as_tensor(lens).cumsum(0).tolist()
        return [(0, e - n, n) for e, n in zip(ends, lens)]
    return [(b, 0, n) for b, n in enumerate(lens)]


def compare(out, q, k, v, spans, causal, scale=SCALE):
    want, mass, reach = ref.prompt(q.cpu(), k.cpu(), v.cpu(), spans, causal, scale)
    longest = max([n for _, _, n in spans] or [1])
    tol = ref.prompt_tolerance(q.dtype, mass, reach, want, longest)
    inside = torch.zeros(q.shape[0], q.shape[2], dtype=torch.bool)
    for b, r0, n in spans:
        inside[b, r0:r0 + n] = True
    got = out.cpu().double()
    err = torch.where(inside[:, None, :, None], (got - want).abs() - tol, got.abs())
    assert bool((err <= 0).all()), f"{float(err.max())} over the bound"


def inputs(B, Hq, Hkv, T, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(B, H, T, 128, generator=g).mul(s).to(dtype).to(DEV) for H, s in ((Hq, 1.5), (Hkv, 1.5), (Hkv, 1.0))]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (4, 1), (6, 2), (5, 1), (32, 1), (17, 1)])
@pytest.mark.parametrize("lens,causal", [([1], True), ([3, 1, 2], True), ([0, 65, 0, 64, 7], True), ([130, 33], False), ([257], True)])
def test_packed(dtype, Hq, Hkv, lens, causal):
    from omnistack_rs_b200.kernels.prompt_attention import prompt_attn
    T = sum(lens)
    q, k, v = inputs(1, Hq, Hkv, T, dtype, seed=Hq * 1000 + T)
    cu = torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32)
    out = prompt_attn(q, k, v, cu_seqlens=cu.to(DEV), causal=causal)
    assert out.shape == q.shape and out.dtype == dtype and out.is_contiguous()
    compare(out, q, k, v, spans_of(lens, T, True), causal)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("T,lens", [(1, None), (129, None), (200, [200, 1, 0, 77]), (64, [64, 63, 65, 5])])
def test_padded(dtype, causal, T, lens):
    from omnistack_rs_b200.kernels.prompt_attention import prompt_attn
    B = 2 if lens is None else len(lens)
    q, k, v = inputs(B, 8, 2, T, dtype, seed=T)
    out = prompt_attn(q, k, v, causal=causal, seq_lens=None if lens is None else torch.tensor(lens, device=DEV))
    compare(out, q, k, v, [(b, 0, T if lens is None else min(lens[b], T)) for b in range(B)], causal)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_long_rows_match_a_dense_product(dtype):
    """Lengths over many tiles, against a dense fp64 product on the device."""
    from omnistack_rs_b200.kernels.prompt_attention import prompt_attn
    T = 2500
    q, k, v = inputs(1, 2, 1, T, dtype, seed=9)
    q = q * 2                                                        # sharper rows: running maxima keep moving
    out = prompt_attn(q, k, v)
    Q, K, V = q.double(), k.double(), v.double()
    s = (Q @ K.transpose(-1, -2)) * SCALE
    p = torch.softmax(s + torch.full((T, T), float("-inf"), device=DEV, dtype=torch.float64).triu(1), -1)
    want, mass = p @ V, p @ V.abs()
    reach = (Q.abs() @ K.abs().transpose(-1, -2)).amax(-1) * SCALE
    tol = ref.prompt_tolerance(dtype, mass, reach, want, T)
    assert bool(((out.double() - want).abs() <= tol).all())


def test_rows_of_no_prompt_are_zero_and_reach_nothing():
    from omnistack_rs_b200.kernels.prompt_attention import prompt_attn
    for dtype in (torch.bfloat16, torch.float32):
        q, k, v = inputs(1, 4, 2, 300, dtype, seed=1)
        spans = [(0, 10, 90), (0, 100, 1), (0, 101, 130)]
        cu = torch.tensor([10, 100, 101, 231], dtype=torch.int32, device=DEV)
        for x in (q, k, v):
            x[:, :, :10] = float("nan")
            x[:, :, 231:] = float("inf")
        out = prompt_attn(q, k, v, cu_seqlens=cu)
        q, k, v = (torch.nan_to_num(x, posinf=0.0) for x in (q, k, v))
        compare(out, q, k, v, spans, True)
        compare(prompt_attn(q, k, v, cu_seqlens=cu[:1]), q, k, v, [], True)             # no prompt at all


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_nan_behind_a_query_stays_there(dtype):
    """A token's infinite or NaN key and value reach the queries from it on, and no earlier one; other prompts never see them."""
    from omnistack_rs_b200.kernels.prompt_attention import prompt_attn
    lens = [150, 40, 300]
    q, k, v = inputs(1, 4, 2, sum(lens), dtype, seed=2)
    cu = torch.tensor([0, 150, 190, 490], dtype=torch.int32, device=DEV)
    v[0, 0, 100, 5], v[0, 1, 149, 7], k[0, 0, 160], v[0, 1, 400, 3] = float("nan"), float("inf"), float("nan"), float("-inf")
    clean = [torch.nan_to_num(x, nan=0.0, posinf=0.0, neginf=0.0) for x in (q, k, v)]
    out = prompt_attn(q, k, v, cu_seqlens=cu)
    want, mass, reach = ref.prompt(*[x.cpu() for x in clean], spans_of(lens, 0, True), True, SCALE)
    tol = ref.prompt_tolerance(dtype, mass, reach, want, 300)
    touched = torch.zeros(out.shape, dtype=torch.bool)
    touched[0, :2, 100:150, 5] = True
    touched[0, 2:, 149, 7] = True
    touched[0, :2, 160:190] = True
    touched[0, 2:, 400:490, 3] = True
    got = out.cpu().double()
    assert not bool(torch.isfinite(got[touched]).any())
    assert bool(((got - want).abs() <= tol)[~touched].all())


def test_strides_scale_and_host_lengths():
    from omnistack_rs_b200.kernels.prompt_attention import prompt_attn
    g = torch.Generator().manual_seed(7)
    proj = torch.randn(2, 90, 4 + 2 + 2, 128, generator=g).to(torch.bfloat16).to(DEV)
    q, k, v = (proj[:, :, a:b].transpose(1, 2) for a, b in ((0, 4), (4, 6), (6, 8)))
    out = prompt_attn(q, k, v, scale=0.02, seq_lens=torch.tensor([90, 11]))
    compare(out, q, k, v, [(0, 0, 90), (1, 0, 11)], True, 0.02)
    assert torch.equal(out, prompt_attn(q.contiguous(), k.contiguous(), v.contiguous(), scale=0.02, seq_lens=torch.tensor([90, 11], device=DEV)))
    wide = torch.randn(1, 2, 70, 130, generator=g).to(torch.float16).to(DEV)     # rows off 16-byte boundaries are copied
    compare(prompt_attn(wide[..., 1:129], wide[..., 1:129], wide[..., 2:]), wide[..., 1:129], wide[..., 1:129], wide[..., 2:], [(0, 0, 70)], True)
    one = torch.randn(1, 1, 50, 128, generator=g).to(torch.bfloat16).to(DEV).expand(1, 3, 50, 128)   # shared by stride 0
    compare(prompt_attn(one, one, one), one, one, one, [(0, 0, 50)], True)
    flat = prompt_attn(q, k, v, scale=0.0)                                       # zero scale: the running mean of the values
    compare(flat, q, k, v, [(0, 0, 90), (1, 0, 90)], True, 0.0)
    for shape in ((0, 4, 5, 128), (1, 4, 0, 128)):
        x = torch.zeros(shape, dtype=torch.bfloat16, device=DEV)
        assert prompt_attn(x, x, x).shape == shape


def test_large_scores():
    """Scores of thousands: one key takes the whole weight, and nothing overflows."""
    from omnistack_rs_b200.kernels.prompt_attention import prompt_attn
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        q, k, v = inputs(1, 2, 1, 200, dtype, seed=3)
        q, k = q * 30, k * 30
        out = prompt_attn(q, k, v, causal=False)
        s = (q.double() @ k.double().transpose(-1, -2)) * SCALE
        top = s.topk(2, -1)
        sure = (top.values[..., 0] - top.values[..., 1]) > 30                    # the rest weighs less than e^-30 together
        want = torch.gather(v.double().expand(1, 2, 200, 128), 2, top.indices[..., :1].expand(1, 2, 200, 128))
        assert int(sure.sum()) > 100
        assert bool(((out.double() - want).abs() <= 2 * ref.half_step(dtype) * want.abs() + 2.0 ** -20)[sure].all())


def test_graph_replay_and_streams():
    """Captured, replayed on new contents, and run on two streams at once."""
    from omnistack_rs_b200.kernels.prompt_attention import prompt_attn
    q, k, v = inputs(1, 8, 2, 500, torch.bfloat16, seed=4)
    cu = torch.tensor([0, 200, 500], dtype=torch.int32, device=DEV)
    first = prompt_attn(q, k, v, cu_seqlens=cu)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = prompt_attn(q, k, v, cu_seqlens=cu)
    graph.replay()
    assert torch.equal(out, first)
    cu.copy_(torch.tensor([0, 350, 480], dtype=torch.int32))
    q.mul_(0.5)
    graph.replay()
    assert torch.equal(out, prompt_attn(q, k, v, cu_seqlens=cu)) and bool((out[:, :, 480:] == 0).all())
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append([prompt_attn(q, k, v, cu_seqlens=cu) for _ in range(5)])
    torch.cuda.synchronize()
    assert all(torch.equal(x, out) for xs in got for x in xs)
