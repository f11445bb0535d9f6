"""A resident cache whose lengths are set back: its weight sums belong to the keys it holds, not to those that stood there before."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
N, HQ, H, MAX = 3, 4, 2, 96


def make_cache(pair_v=False, residual=True):
    from omnistack_rs_b200.serving import QuantizedKVCache
    cb = torch.sort(torch.randn(H, 16, generator=torch.Generator().manual_seed(0)), dim=1).values
    return QuantizedKVCache(N, H, MAX, cb, DEV, store_v_residual=residual, pair_v=pair_v)


def rows(heads, T, seed, dtype=torch.bfloat16):
    return torch.randn(N, heads, T, 128, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dtype)


def set_lens(cache, lens):
    cache.lens.copy_(torch.tensor(lens))
    cache.lens32.copy_(cache.lens)


@pytest.mark.parametrize("pair_v,residual", [(False, True), (True, False)])
@pytest.mark.parametrize("values", [torch.bfloat16, torch.float32])       # (values of another type than the keys take the general path)
def test_another_continuation(pair_v, residual, values):
    k0, v0, q = rows(H, 40, 1), rows(H, 40, 2, values), rows(HQ, 1, 3)
    first, second = (rows(H, 30, 4), rows(H, 30, 5, values)), (rows(H, 20, 6), rows(H, 20, 7, values))
    cache, fresh = make_cache(pair_v, residual), make_cache(pair_v, residual)
    for c in (cache, fresh):
        c.append(k0, v0)
    set_lens(cache, [40, 8, 0])
    set_lens(fresh, [40, 8, 0])
    cache.append(*first)
    cache.observe(q)
    set_lens(cache, [40, 8, 0])                                           # back to where the continuation began
    cache.append(*second)
    fresh.append(*second)
    cache.observe(q)
    fresh.observe(q)
    for b, n in enumerate([40, 8, 0]):
        assert torch.equal(cache.weight_sums[b, :, n:n + 20], fresh.weight_sums[b, :, n:n + 20])
        assert n == 0 or bool((cache.weight_sums[b, :, :n] > fresh.weight_sums[b, :, :n]).all())   # these keys saw both
    cache.append(*second)                                                 # and new keys after any of it begin with nothing
    for b, n in enumerate([60, 28, 20]):
        assert bool((cache.weight_sums[b, :, n:n + 20] == 0).all())


def test_another_prompt():
    q = rows(HQ, 1, 3)
    old, new = [rows(h, 50, 10 + h) for h in (HQ, H, H)], [rows(h, 45, 20 + h) for h in (HQ, H, H)]
    cache, fresh = make_cache(), make_cache()
    cache.prefill(*old)
    cache.observe(q)
    set_lens(cache, [0, 0, 0])
    for c in (cache, fresh):
        c.prefill(*new, torch.tensor([45, 3, 20]))
        c.observe(q)
        c.append(rows(H, 9, 30), rows(H, 9, 31))
        c.observe(q)
    for b, n in enumerate([54, 12, 29]):
        assert torch.equal(cache.weight_sums[b, :, :n], fresh.weight_sums[b, :, :n])
    assert torch.equal(cache.evict(7, recent=2), fresh.evict(7, recent=2))


def test_a_refused_append_changes_no_sums():
    cache = make_cache()
    cache.append(rows(H, 80, 1), rows(H, 80, 2))
    before = cache.observe(rows(HQ, 1, 3)).clone()
    with pytest.raises(ValueError, match="capacity"):
        cache.append(rows(H, 20, 4), rows(H, 20, 5))
    assert torch.equal(cache.weight_sums, before) and bool((before[:, :, :80] > 0).all())


def test_clearing_stays_inside_the_rows():
    """Lengths at, near and past both ends: nothing outside a head's S entries is touched."""
    from omnistack_rs_b200 import _lib
    lib, B, S, T = _lib.load(), 7, 10, 4
    guard = torch.full((2 + B * H, S), 5.0, device=DEV)
    lens = torch.tensor([0, 3, 6, 8, 10, 1 << 40, -2], device=DEV)
    _lib.check(lib.omni_clear_new_sums(guard[1:].data_ptr(), lens.data_ptr(), B, H, S, T, _lib.stream_ptr(guard.device)))
    want = torch.full((2 + B * H, S), 5.0)
    for b, n in enumerate(lens.tolist()):
        for s in range(max(n, 0), min(n + T, S)):
            want[1 + b * H:1 + (b + 1) * H, s] = 0
    assert torch.equal(guard.cpu(), want)
    assert lib.omni_clear_new_sums(None, lens.data_ptr(), B, H, S, T, None) == _lib.ERR_ARG
    assert lib.omni_clear_new_sums(None, None, B, -1, S, T, None) == _lib.ERR_ARG and lib.omni_clear_new_sums(None, None, B, H, S, 0, None) == _lib.OK


@pytest.mark.parametrize("pair_v", [False, True])
def test_prompts_that_fit_although_their_padding_does_not(pair_v):
    """What counts is the longest prompt, not the padded length; what does not fit is refused before anything is done."""
    x = [rows(h, MAX + 40, h, torch.float16) for h in (HQ, H, H)]
    lens = torch.tensor([MAX, 13, 0])
    cache, narrow = make_cache(pair_v), make_cache(pair_v)
    out = cache.prefill(*x, lens)
    want = narrow.prefill(*[t[:, :, :MAX] for t in x], lens)
    assert out.shape == x[0].shape and torch.equal(out[:, :, :MAX], want) and bool((out[:, :, MAX:] == 0).all())
    assert cache.lens.tolist() == lens.tolist() == cache.lens32.tolist()
    for b, n in enumerate(lens.tolist()):
        for name in ("k_nib", "k_qjl", "k_norms", "v_nib", "v_qjl", "v_norms"):
            assert torch.equal(getattr(cache, name)[b, :, :n], getattr(narrow, name)[b, :, :n]), name
    q = rows(HQ, 1, 9)
    assert torch.equal(cache.attend(q), narrow.attend(q))
    over = make_cache(pair_v)
    with pytest.raises(ValueError, match="capacity"):
        over.prefill(*x, torch.tensor([1, MAX + 1, 0]))
    with pytest.raises(ValueError, match="capacity"):
        over.prefill(*x)
    assert over.lens.tolist() == [0, 0, 0] and bool((over.k_nib == 0).all())
    none = over.prefill(*x, torch.zeros(N, dtype=torch.int64))            # prompts without a token
    assert bool((none == 0).all()) and over.lens.tolist() == [0, 0, 0]


def test_sums_that_are_not_the_cache_s_own_kind():
    """A user may bring sums of their own, from a file for instance: of the cache's shape, on its device."""
    cache = make_cache()
    x = rows(H, 5, 1)
    cache.append(x, x)
    good = torch.ones(N, H, MAX, device=DEV)
    for bad, error in ((good.cpu(), RuntimeError), (good[:, :, :50], ValueError), (good.double(), ValueError), (good.transpose(0, 1).contiguous().transpose(0, 1), ValueError)):
        cache.weight_sums = bad
        with pytest.raises(error):
            cache.append(x, x)
        assert cache.lens.tolist() == [5] * N
    cache.weight_sums = good
    cache.append(x, x)
    assert cache.lens.tolist() == [10] * N
    assert bool((good[:, :, 5:10] == 0).all()) and bool((good[:, :, :5] == 1).all()) and bool((good[:, :, 10:] == 1).all())
