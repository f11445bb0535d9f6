"""The way of a prompt into the cache and out of it again, as a serving loop runs it: norm and rotation, prompt attention, packing,
decoding, weights, eviction, decoding on what is left."""
import pytest
import torch

import oracle as orc
from tests import operator_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SCALE = 1.0 / 128 ** 0.5


def make_cache(pair_v, residual, n=3, H=2, max_len=160):
    from omnistack_rs_b200.serving import QuantizedKVCache
    cb = torch.sort(torch.randn(H, 16, generator=torch.Generator().manual_seed(0)), dim=1).values
    return QuantizedKVCache(n, H, max_len, cb, DEV, store_v_residual=residual, pair_v=pair_v)


@pytest.mark.parametrize("pair_v,residual,dtype", [(False, True, torch.bfloat16), (True, False, torch.float16), (True, True, torch.float32)])
def test_prompt_decode_observe_evict(pair_v, residual, dtype):
    from omnistack_rs_b200.kernels.fused_attention import omni_attn
    from omnistack_rs_b200.kernels.position import qk_norm_rope
    from omnistack_rs_b200.kernels.prompt_attention import prompt_attn
    from omnistack_rs_b200.kernels.quantize import quantize_heads
    g = torch.Generator(device=DEV).manual_seed(5)
    n, Hq, H, T = 3, 4, 2, 101
    lens = torch.tensor([101, 37, 64])
    proj = torch.randn(n, T, Hq + 2 * H, 128, generator=g, device=DEV).to(dtype)
    q, k, v = proj[:, :, :Hq].transpose(1, 2), proj[:, :, Hq:Hq + H].transpose(1, 2), proj[:, :, Hq + H:].transpose(1, 2)
    freq = 10000.0 ** (-torch.arange(64, device=DEV) / 64)
    q, k = qk_norm_rope(q, k, torch.arange(T, device=DEV), freq)
    cache = make_cache(pair_v, residual)
    out = cache.prefill(q, k, v, lens)
    assert torch.equal(out, prompt_attn(q, k, v, seq_lens=lens.to(DEV)))
    assert cache.lens.tolist() == lens.tolist() == cache.lens32.tolist()
    # the packed rows are those of the codec, V's in the layout that belongs to the lengths
    nib, qjl, norms = quantize_heads(k, cache.codebooks, cache.user_ids, rotate=True)
    v_nib = quantize_heads(v, cache.codebooks, cache.user_ids, rotate=True)[0].cpu()
    stored = ref.pair_rows(v_nib, lens) if pair_v else v_nib
    for b, m in enumerate(lens.tolist()):
        assert torch.equal(cache.k_nib[b, :, :m], nib[b, :, :m]) and torch.equal(cache.k_qjl[b, :, :m], qjl[b, :, :m])
        assert torch.equal(cache.k_norms[b, :, :m], norms[b, :, :m]) and torch.equal(cache.v_nib[b, :, :m].cpu(), stored[b, :, :m])
    # a few decoding steps: append, attend, observe
    for step in range(9):
        tok = torch.randn(n, 1, Hq + 2 * H, 128, generator=g, device=DEV).to(dtype)
        qs, ks = qk_norm_rope(tok[:, :, :Hq].transpose(1, 2), tok[:, :, Hq:Hq + H].transpose(1, 2), cache.lens[:, None], freq)
        cache.append(ks, tok[:, :, Hq + H:].transpose(1, 2))
        before = None if cache.weight_sums is None else cache.weight_sums.clone()
        cache.attend(qs, rotate_q=True, unrotate_out=True)
        sums = cache.observe(qs, rotate_q=True)
        for b, m in enumerate(cache.lens.tolist()):                              # every head's weights add up to its queries
            added = sums[b, :, :m] - (0 if before is None else before[b, :, :m])
            assert bool(((added.sum(-1) - Hq // H).abs() < 1e-4).all())
    total = cache.lens.tolist()
    assert total == [110, 46, 73]
    # evict, and decode on what is left: the same as attention over the kept rows alone
    old = {name: getattr(cache, name).clone() for name in ("k_nib", "k_qjl", "k_norms", "weight_sums")}
    v_rows = ref.pair_rows(cache.v_nib.cpu(), total) if pair_v else cache.v_nib.cpu()
    index = cache.evict(50, recent=8, max_len=70)
    assert cache.lens.tolist() == [50, 46, 50] == cache.lens32.tolist() and cache.k_nib.shape == (n, H, 70, 64) and cache.max_len == 70
    assert torch.equal(index[1, :, :46].cpu(), torch.arange(46, dtype=torch.int32).expand(H, 46)) and bool((index[1, :, 46:] == -1).all())
    for h in range(H):
        for b in (0, 2):
            assert index[b, h].tolist() == ref.kept_positions(old["weight_sums"][b, h].tolist(), total[b], 50, 8)
            assert torch.equal(cache.weight_sums[b, h, :50], old["weight_sums"][b, h, index[b, h].long()])
    qs = torch.randn(n, Hq, 1, 128, generator=g, device=DEV).to(dtype)
    out = cache.attend(qs)
    kept = [torch.stack([torch.stack([x[b, h, index[b, h].clamp(min=0).long().to(x.device)] for h in range(H)]) for b in range(n)])
            for x in (old["k_nib"], old["k_qjl"], old["k_norms"], v_rows.to(DEV))]
    want = omni_attn(qs, *kept, cache.codebooks, user_id=cache.user_ids, seq_lens=cache.lens32)
    assert torch.allclose(out, want, atol=1e-6, rtol=0)
    for b in range(n):                                                           # and against the oracle
        m = cache.lens.tolist()[b]
        dense = orc.decode_attention(qs[b:b + 1].cpu(), *[x[b:b + 1, :, :m].cpu() for x in kept], cache.codebooks.cpu(), int(cache.user_ids[b]))
        assert float((out[b:b + 1].cpu() - dense).abs().max()) <= 3e-3
    cache.append(ks, tok[:, :, Hq + H:].transpose(1, 2))                         # the smaller cache goes on
    assert cache.lens.tolist() == [51, 47, 51]


def test_prefill_refusals_and_defaults():
    cache = make_cache(True, False)
    x = torch.randn(3, 2, 20, 128, device=DEV)
    with pytest.raises(ValueError, match="prompt_lens"):
        cache.prefill(x, x, x, torch.tensor([1, 2]))
    with pytest.raises(ValueError, match="lie in"):
        cache.prefill(x, x, x, torch.tensor([1, 21, 0]))
    cache.prefill(x, x, x)
    assert cache.lens.tolist() == [20, 20, 20]
    with pytest.raises(ValueError, match="already holds"):
        cache.prefill(x, x, x)
    index = cache.evict(7)                                                       # nothing observed: the first keys stay
    assert cache.weight_sums is None and index.cpu().tolist() == [[list(range(7))] * 2] * 3 and cache.max_len == 160
    with pytest.raises(ValueError, match="budget"):
        cache.evict(8, recent=9)
    big = make_cache(False, True, max_len=10)
    with pytest.raises(ValueError, match="capacity"):
        big.prefill(x, x, x)


@pytest.mark.parametrize("pair_v", [False, True])
@pytest.mark.parametrize("T", [1, 33])
def test_padding_of_a_prompt_reaches_nothing(pair_v, T):
    """Rows behind a prompt may hold anything: the packed rows they leave behind the length are never attended to.  The prompt's own
    rows beside infinities or NaN are computed again with unrounded weights, the others with weights rounded to bf16: half a step,
    2^-8, of each weight and so at most of max |v| in the result, and each result is rounded once, 2^-8 of at most max |v| each."""
    g = torch.Generator(device=DEV).manual_seed(2)
    x = [torch.randn(3, h, 40, 128, generator=g, device=DEV, dtype=torch.bfloat16) for h in (4, 2, 2)]
    lens = torch.tensor([40, 13, 0])
    top = float(x[2].float().abs().max())
    results = []
    for fill in (0.0, float("nan"), float("inf")):
        rows = [t.clone() for t in x]
        for b, m in enumerate(lens.tolist()):
            for t in rows:
                t[b, :, m:] = fill
        cache = make_cache(pair_v, True)
        out = cache.prefill(*rows, lens)
        q = torch.randn(3, 4, T, 128, generator=torch.Generator(device=DEV).manual_seed(3), device=DEV, dtype=torch.bfloat16)
        got = [out, cache.attend(q), cache.observe(q).clone()]
        index = cache.evict(9, recent=2)
        results.append(got + [index, cache.k_nib, cache.v_nib, cache.k_norms, cache.weight_sums, cache.attend(q)])
    for got in results:
        assert all(bool(torch.isfinite(t.float()).all()) for t in got)
        assert all(torch.equal(a, b) for a, b in zip(got[1:], results[0][1:]))
        assert float((got[0].float() - results[0][0].float()).abs().max()) <= 3 * 2 ** -8 * 1.001 * top
        assert all(bool((got[0][b, :, m:] == 0).all()) for b, m in enumerate(lens.tolist()))
    assert bool((results[0][0][2] == 0).all()) and bool((results[0][2][2] == 0).all())


def test_empty_prompts():
    cache = make_cache(True, True)
    x = torch.randn(3, 2, 0, 128, device=DEV)
    assert cache.prefill(x, x, x).shape == (3, 2, 0, 128) and cache.lens.tolist() == [0, 0, 0]
    assert bool((cache.evict(4) == -1).all())
    q = torch.randn(3, 4, 1, 128, device=DEV)
    assert bool((cache.observe(q) == 0).all())


def test_captures():
    g = torch.Generator(device=DEV).manual_seed(4)
    x = torch.randn(3, 2, 40, 128, generator=g, device=DEV, dtype=torch.bfloat16)
    q = torch.randn(3, 4, 1, 128, generator=g, device=DEV, dtype=torch.bfloat16)
    cache, plain = make_cache(True, False), make_cache(True, False)
    for c in (cache, plain):
        c.prefill(x, x, x)
    plain.observe(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="before the capture"):
            cache.observe(q)
        with pytest.raises(RuntimeError, match="cannot be captured"):
            cache.evict(8)
    assert cache.weight_sums is None and cache.max_len == 160
    cache.observe(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.observe(q)
    for _ in range(3):
        graph.replay()
        plain.observe(q)
    assert torch.equal(cache.weight_sums, plain.weight_sums)
    assert torch.equal(cache.evict(8, recent=2), plain.evict(8, recent=2))
