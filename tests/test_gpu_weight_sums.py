"""``attn_weight_sums`` against its definition in 64 bits over the dequantised keys."""
import pytest
import torch

from tests import operator_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SCALE = 1.0 / 128 ** 0.5


def packed(B, H, S, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    byte = lambda n: torch.randint(0, 256, (B, H, S, n), generator=g, dtype=torch.uint8)  # noqa: E731
    cb = torch.sort(torch.randn(H, 16, generator=g) * spread, dim=1).values
    return byte(64), byte(8), torch.rand(B, H, S, generator=g) + 0.5, cb


def check(got, q, rows, cb, ids, lens, with_qjl, causal, scale=SCALE, extra=0.0):
    keys = ref.dequantized_keys(*[r.cpu() for r in rows], cb.cpu(), ids, with_qjl)
    want, reach = ref.weight_sums(q.cpu(), keys, lens, scale, causal)
    # Scores: centroids and queries may be split in two 11-bit parts (2^-22 each), 192 products and two factors in fp32
    # (200 * 2^-24): |ds| <= 52 * 2^-22 * reach; the exponential adds 2^-22 and the normaliser the same again.  Adding up S
    # weights of one column and the columns in fp32: (S + columns) * 2^-24.
    S, cols = want.shape[2], q.shape[1] // want.shape[1] * q.shape[2]
    rel = 4 * (52 * 2.0 ** -22 * reach[..., None] + 2.0 ** -22) + (S + cols) * 2.0 ** -24 + extra
    err = (got.cpu().double() - want).abs()
    assert bool((err <= rel * want + 1e-30).all()), float((err / (rel * want + 1e-30)).max())
    for b, n in enumerate(lens):
        assert bool((got[b, :, int(n):] == 0).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,Hq,Hkv,T,S,lens", [(1, 1, 1, 1, 1, None), (2, 8, 2, 1, 300, [300, 17]), (3, 6, 3, 4, 140, [0, 2, 140]), (1, 4, 1, 9, 129, None),
                                               (2, 10, 2, 1, 1025, [1025, 513]), (1, 3, 1, 32, 70, [33]), (2, 16, 1, 1, 64, None),
                                               (1, 8, 1, 40, 700, [690]), (1, 4, 2, 20, 1300, None)])
def test_against_definition(dtype, B, Hq, Hkv, T, S, lens):
    from omnistack_rs_b200.kernels.eviction import attn_weight_sums
    nib, qjl, norms, cb = packed(B, Hkv, S, seed=S + T)
    q = (torch.randn(B, Hq, T, 128, generator=torch.Generator().manual_seed(T)) * 1.5).to(dtype)
    ids = torch.tensor([7, 2000, 1023][:B], dtype=torch.int32)
    host = [S] * B if lens is None else lens
    dev = [x.to(DEV) for x in (q, nib, qjl, norms, cb)]
    seq = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=DEV)
    for causal in (True, False):
        for with_qjl in (True, False):
            got = attn_weight_sums(*dev, user_id=ids.to(DEV), with_qjl=with_qjl, seq_lens=seq, causal=causal)
            assert got.shape == (B, Hkv, S) and got.dtype is torch.float32
            check(got, q, (nib, qjl, norms), cb, ids, host, with_qjl, causal)
    again = attn_weight_sums(*dev, user_id=ids.to(DEV), seq_lens=seq)
    assert torch.equal(again, attn_weight_sums(*dev, user_id=ids.to(DEV), seq_lens=seq))


def test_into_adds_and_leaves_the_rest():
    from omnistack_rs_b200.kernels.eviction import attn_weight_sums
    nib, qjl, norms, cb = packed(2, 2, 50, seed=1)
    dev = [x.to(DEV) for x in (torch.randn(2, 4, 1, 128, generator=torch.Generator().manual_seed(0)), nib, qjl, norms, cb[0])]
    lens = torch.tensor([50, 20], device=DEV)
    once = attn_weight_sums(*dev, seq_lens=lens)
    into = torch.full((2, 2, 50), 3.0, device=DEV)
    assert attn_weight_sums(*dev, seq_lens=lens, into=into) is into
    assert torch.equal(into[0], 3 + once[0]) and torch.equal(into[1, :, :20], 3 + once[1, :, :20]) and bool((into[1, :, 20:] == 3).all())
    none = attn_weight_sums(dev[0][:, :, :0], *dev[1:])
    assert bool((none == 0).all())


def test_rotation_wide_codebooks_and_scale():
    """A query rotated in the call equals one rotated before it; codebooks of any finite size are served."""
    from omnistack_rs_b200.kernels.eviction import attn_weight_sums
    from omnistack_rs_b200.kernels.hadamard import rotate_queries
    for spread, scale in ((1.0, SCALE), (30.0, 0.003), (1e-4, 500.0)):
        nib, qjl, norms, cb = packed(2, 2, 200, seed=5, spread=spread)
        norms = norms * spread
        q = torch.randn(2, 8, 1, 128, generator=torch.Generator().manual_seed(1))
        rows = [x.to(DEV) for x in (nib, qjl, norms, cb)]
        turned = rotate_queries(q.to(DEV))
        got = attn_weight_sums(turned, *rows, user_id=3, scale=scale)
        check(got, turned, (nib, qjl, norms), cb, [3, 3], [200, 200], True, True, scale)
        check(attn_weight_sums(q.to(DEV), *rows, user_id=3, scale=scale, rotate_q=True), turned, (nib, qjl, norms), cb, [3, 3], [200, 200], True, True, scale)


@pytest.mark.parametrize("scale", [0.0, -0.3])
def test_scales_without_a_sign_of_their_own(scale):
    """A zero scale weighs every key alike, a negative one prefers the smallest products; for few and many columns."""
    from omnistack_rs_b200.kernels.eviction import attn_weight_sums
    nib, qjl, norms, cb = packed(1, 1, 150, seed=11)
    for T in (1, 12):
        q = torch.randn(1, 2, T, 128, generator=torch.Generator().manual_seed(T))
        got = attn_weight_sums(*[x.to(DEV) for x in (q, nib, qjl, norms, cb)], user_id=5, scale=scale, seq_lens=torch.tensor([140]))
        check(got, q, (nib, qjl, norms), cb, [5], [140], True, True, scale)


def test_few_tiles_for_many_ctas():
    """Most users empty, the others short: more CTAs than tiles.  Scratch memory holds whatever it held before."""
    from omnistack_rs_b200.kernels.eviction import attn_weight_sums
    nib, qjl, norms, cb = packed(12, 2, 600, seed=21)
    lens = [0, 0, 130, 0, 1, 0, 0, 0, 600, 0, 3, 0]
    dev = [x.to(DEV) for x in (nib, qjl, norms, cb)]
    for T in (1, 12):
        q = torch.randn(12, 4, T, 128, generator=torch.Generator().manual_seed(T))
        for fill in (1e30, float("nan")):
            torch.cuda.synchronize()
            trash = [torch.full((1 << 20,), fill, device=DEV) for _ in range(16)]
            del trash
            got = attn_weight_sums(q.to(DEV), *dev, user_id=9, seq_lens=torch.tensor(lens, device=DEV))
            check(got, q, (nib, qjl, norms), cb, [9] * 12, lens, True, True)


def test_nan_behind_the_length_is_not_read():
    from omnistack_rs_b200.kernels.eviction import attn_weight_sums
    nib, qjl, norms, cb = packed(1, 1, 100, seed=6)
    norms[0, 0, 60:] = float("nan")
    q = torch.randn(1, 2, 1, 128, generator=torch.Generator().manual_seed(1))
    dev = [x.to(DEV) for x in (q, nib, qjl, norms, cb)]
    check(attn_weight_sums(*dev, seq_lens=torch.tensor([60])), q, (nib, qjl, torch.nan_to_num(norms)), cb, [0], [60], True, True)
    assert bool(torch.isnan(attn_weight_sums(*dev, seq_lens=torch.tensor([61]))[0, 0, :61]).all())       # a NaN key makes its head's weights NaN


def test_graph_replay():
    from omnistack_rs_b200.kernels.eviction import attn_weight_sums
    nib, qjl, norms, cb = packed(4, 2, 700, seed=8)
    q = torch.randn(4, 8, 1, 128, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    dev = [x.to(DEV) for x in (q, nib, qjl, norms, cb)]
    lens = torch.tensor([700, 5, 333, 0], dtype=torch.int32, device=DEV)
    first = attn_weight_sums(*dev, seq_lens=lens)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = attn_weight_sums(*dev, seq_lens=lens)
    graph.replay()
    assert torch.equal(out, first)
    lens.copy_(torch.tensor([1, 700, 0, 64], dtype=torch.int32))
    graph.replay()
    assert torch.equal(out, attn_weight_sums(*dev, seq_lens=lens))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,per_head", [(1, True), (12, False), (70, True)])
def test_many_short_caches_per_cta(dtype, T, per_head):
    """More tiles than CTAs, so that a CTA walks over several heads and users, some of them empty, and changes columns and centroid
    tables on its way; 140 columns take two rounds."""
    from omnistack_rs_b200.kernels.eviction import attn_weight_sums
    B, H, S = 44, 4, 300
    nib, qjl, norms, cb = packed(B, H, S, seed=31)
    if not per_head:
        cb = cb[0]
    g = torch.Generator().manual_seed(2)
    lens = torch.randint(0, S + 1, (B,), generator=g).tolist()
    lens[:9] = [300, 0, 1, 128, 0, 0, 129, 256, 2]
    q = torch.randn(B, 2 * H, T, 128, generator=g).to(dtype)
    ids = torch.arange(B, dtype=torch.int32) * 37
    dev = [x.to(DEV) for x in (q, nib, qjl, norms, cb)]
    seq = torch.tensor(lens, device=DEV)
    for with_qjl in (True, False):
        got = attn_weight_sums(*dev, user_id=ids.to(DEV), with_qjl=with_qjl, seq_lens=seq)
        check(got, q, (nib, qjl, norms), cb if per_head else cb.expand(H, 16), ids, lens, with_qjl, True)
        assert torch.equal(got, attn_weight_sums(*dev, user_id=ids.to(DEV), with_qjl=with_qjl, seq_lens=seq))
        if T < 70:                                                               # one round: a single addition
            into = torch.full((B, H, S), 3.0, device=DEV)
            attn_weight_sums(*dev, user_id=ids.to(DEV), with_qjl=with_qjl, seq_lens=seq, into=into)
            assert torch.equal(into, 3 + got)
