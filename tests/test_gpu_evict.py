"""``evict_keys``: the kept positions against plain sorting, and every array's rows bit for bit."""
import pytest
import torch

from tests import operator_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def arrays(B, H, S, seed, residual):
    g = torch.Generator().manual_seed(seed)
    byte = lambda n: torch.randint(0, 256, (B, H, S, n), generator=g, dtype=torch.uint8)  # noqa: E731
    real = lambda: torch.randn(B, H, S, generator=g)  # noqa: E731
    return byte(64), byte(8), real(), byte(64), byte(8) if residual else None, real() if residual else None


def check(sums, rows, lens, budget, recent, paired, capacity=None):
    from omnistack_rs_b200.kernels.eviction import evict_keys
    B, H, S = sums.shape
    k_nib, k_qjl, k_norms, v_nib, v_qjl, v_norms = rows
    stored = ref.pair_rows(v_nib, lens) if paired else v_nib
    dev = [None if x is None else x.to(DEV) for x in (sums, k_nib, k_qjl, k_norms, stored, v_qjl, v_norms)]
    before = [None if x is None else x.clone() for x in dev]
    got = evict_keys(*dev[:5], budget, recent=recent, seq_lens=torch.tensor(lens, device=DEV), v_qjl=dev[5], v_norms=dev[6], v_paired=paired,
                     capacity=capacity)
    same = lambda x, y: (x is None and y is None) or torch.equal(x.nan_to_num(nan=-7.0), y.nan_to_num(nan=-7.0))  # noqa: E731
    assert all(same(x, y) for x, y in zip(dev, before))                          # what was given is not changed
    cap = capacity or budget
    new = [min(n, budget) for n in lens]
    assert got.seq_lens.tolist() == new and got.seq_lens.dtype is torch.int32
    want = [None if x is None else torch.zeros(B, H, cap, *x.shape[3:], dtype=x.dtype) for x in (sums, *rows)]
    index = torch.full((B, H, budget), -1, dtype=torch.int32)
    for b in range(B):
        for h in range(H):
            kept = ref.kept_positions(sums[b, h].tolist(), lens[b], budget, recent)
            index[b, h, :len(kept)] = torch.tensor(kept, dtype=torch.int32)
            for w, x in zip(want, (sums, *rows)):
                if w is not None:
                    w[b, h, :len(kept)] = x[b, h, kept]
    if paired:
        want[4] = ref.pair_rows(want[4], new)
    assert torch.equal(got.index.cpu(), index)
    for name, w, x in zip(("sums", "k_nib", "k_qjl", "k_norms", "v_nib", "v_qjl", "v_norms"), want, got[2:]):
        assert same(w, None if x is None else x.cpu()), name


@pytest.mark.parametrize("paired,residual", [(False, True), (True, False)])
@pytest.mark.parametrize("S,lens,budget,recent", [(1, [1, 0], 1, 0), (40, [40, 9], 8, 3), (41, [41, 16], 17, 17), (1500, [1500, 1031], 100, 0),
                                                  (1025, [1024, 1025], 1023, 5), (300, [299, 8], 256, 64), (64, [64, 10], 64, 0), (30, [30, 12], 50, 10),
                                                  (20000, [20000, 8193], 8000, 100), (8200, [8192, 8200], 4000, 0)])
def test_against_sorting(paired, residual, S, lens, budget, recent):
    rows = arrays(2, 3, S, seed=S + budget, residual=residual)
    g = torch.Generator().manual_seed(budget)
    sums = torch.exp(2 * torch.randn(2, 3, S, generator=g))
    check(sums, rows, lens, budget, recent, paired)
    check(sums, rows, lens, budget, recent, paired, capacity=budget + 13)


@pytest.mark.parametrize("kind", ["equal", "few", "special"])
def test_ties_and_special_values(kind):
    """Equal sums go to the earlier key; -0 equals +0; infinities and NaN have their place in the order."""
    S = 2100
    rows = arrays(2, 2, S, seed=1, residual=False)
    g = torch.Generator().manual_seed(2)
    sums = torch.randint(0, 3, (2, 2, S), generator=g).float()
    if kind == "equal":
        sums = torch.full((2, 2, S), 0.25)
    if kind == "special":
        values = torch.tensor([float("nan"), float("inf"), float("-inf"), 0.0, -0.0, -1.0, 1e-40, 2.0])
        sums = values[torch.randint(0, 8, (2, 2, S), generator=g)]
    for budget in (1, 700, 2099):
        check(sums, rows, [S, 1800], budget, min(budget, 40), True)


def test_empty_arrays_and_host_lengths():
    from omnistack_rs_b200.kernels.eviction import evict_keys
    z = lambda *s: torch.zeros(*s, dtype=torch.uint8, device=DEV)  # noqa: E731
    for B, H, S in ((0, 2, 5), (2, 2, 0)):
        f = torch.zeros(B, H, S, device=DEV)
        got = evict_keys(f, z(B, H, S, 64), z(B, H, S, 8), f, z(B, H, S, 64), 3)
        assert got.k_nibbles.shape == (B, H, 3, 64) and bool((got.k_nibbles == 0).all()) and bool((got.index == -1).all()) and bool((got.seq_lens == 0).all())
    f = torch.rand(1, 1, 9, device=DEV)
    got = evict_keys(f, z(1, 1, 9, 64), z(1, 1, 9, 8), f, z(1, 1, 9, 64), 4, seq_lens=torch.tensor([7]))
    assert got.index.cpu()[0, 0].tolist() == ref.kept_positions(f[0, 0].tolist(), 7, 4, 0)
