"""``qk_norm_rope`` against its definition in 64 bits."""
import pytest
import torch

from tests import operator_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def check(q, k, positions, inv_freq, qw, kw, eps, axis_pairs, interleaved):
    from omnistack_rs_b200.kernels.position import qk_norm_rope
    args = [None if x is None else x.to(DEV) for x in (positions, inv_freq, qw, kw)]
    got = qk_norm_rope(q, k, args[0], args[1], q_weight=args[2], k_weight=args[3], eps=eps, axis_pairs=axis_pairs, interleaved=interleaved)
    B, T = q.shape[0], q.shape[2]
    pairs = axis_pairs or (inv_freq.numel(),)
    pos = (positions if axis_pairs else positions[None])
    pos = (pos[:, None] if pos.dim() == 2 else pos).expand(len(pairs), B, T)
    for x, w, y in ((q, qw, got[0]), (k, kw, got[1])):
        if x is None:
            assert y is None
            continue
        assert y.shape == x.shape and y.dtype == x.dtype and y.is_contiguous()
        want, size = ref.norm_rope(x.cpu(), pos, inv_freq, w, eps, pairs, interleaved)
        # the norm: 128 squares (relative 2^-24 each, half of it in the root), the root and two products; cos and sin 2^-22
        # with their argument's rounding; two products and a sum: less than 80 * 2^-24 of the pair's size
        tol = 80 * 2.0 ** -24 * size + ref.half_step(x.dtype) * (want.abs() + 80 * 2.0 ** -24 * size) + 2.0 ** -25
        err = (y.cpu().double() - want).abs()
        assert bool((err <= tol).all()), float((err - tol).max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,Hq,Hkv,T,P,interleaved", [(1, 1, 1, 1, 64, False), (3, 8, 2, 5, 64, True), (2, 3, 1, 33, 32, False), (2, 5, 5, 7, 16, True),
                                                      (1, 4, 2, 130, 8, False), (2, 2, 1, 9, 20, False), (1, 2, 2, 3, 1, False), (1, 2, 1, 3, 63, False),
                                                      (1, 7, 1, 2, 5, True), (2, 2, 1, 3, 0, False)])
def test_against_definition(dtype, B, Hq, Hkv, T, P, interleaved):
    g = torch.Generator().manual_seed(B * 100 + T)
    q, k = (torch.randn(B, H, T, 128, generator=g).mul(3).to(dtype).to(DEV) for H in (Hq, Hkv))
    positions = torch.randint(0, 40000, (B, T), generator=g)
    inv_freq = 10000.0 ** (-torch.arange(P) / max(P, 1))
    qw, kw = 1 + 0.3 * torch.randn(128, generator=g), (1 + 0.3 * torch.randn(128, generator=g)).to(dtype)
    check(q, k, positions, inv_freq, qw, kw, 1e-6, None, interleaved)
    check(q, k, positions.int()[0], inv_freq.double(), None, None, 1e-5, None, interleaved)
    check(q, None, positions, inv_freq, None, None, None, None, interleaved)


@pytest.mark.parametrize("axis_pairs", [(64,), (16, 24, 24), (0, 1, 62, 1), (32, 32)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_axes(axis_pairs, interleaved):
    g = torch.Generator().manual_seed(3)
    q, k = (torch.randn(2, H, 11, 128, generator=g).to(torch.bfloat16).to(DEV) for H in (4, 2))
    inv_freq = 500000.0 ** (-torch.arange(64) / 64)
    for shape in ((len(axis_pairs), 2, 11), (len(axis_pairs), 11)):
        check(q, k, torch.randint(-50, 5000, shape, generator=g), inv_freq, torch.randn(128, generator=g), None, 1e-6, axis_pairs, interleaved)


def test_far_positions():
    """Past 2^24 a position times a frequency needs 64 bits, and int64 positions past 2^31 are taken as they are."""
    g = torch.Generator().manual_seed(4)
    q = torch.randn(1, 2, 6, 128, generator=g).to(DEV)
    positions = torch.tensor([[0, 2 ** 24 + 1, 2 ** 31 - 1, 2 ** 31 + 7, 2 ** 40 + 3, -5]])
    # the product of position and frequency is rounded to 53 bits: at 2^40 radians that is 2^-13 of a radian
    check(q[:, :, :4], None, positions[:, :4], 10000.0 ** (-torch.arange(64) / 64), None, None, 1e-6, None, False)
    check(q, None, positions, torch.full((64,), 2.0 ** -20), None, None, 1e-6, None, False)


def test_strided_views_and_zero_sizes():
    from omnistack_rs_b200.kernels.position import qk_norm_rope
    g = torch.Generator().manual_seed(5)
    proj = torch.randn(2, 7, 12, 128, generator=g).to(torch.bfloat16).to(DEV)
    positions, inv_freq = torch.arange(7)[None].expand(2, 7), 10000.0 ** (-torch.arange(64) / 64)
    w = torch.randn(128, generator=g)
    before = proj.clone()
    check(proj[:, :, :8].transpose(1, 2), proj[:, :, 8:10].transpose(1, 2), positions, inv_freq, w, w, 1e-6, None, False)
    assert torch.equal(proj, before)
    odd = torch.randn(2, 4, 7, 129, generator=g).to(DEV)                         # rows that start off a 16-byte boundary are copied
    check(odd[..., 1:], odd[:, :2, :, 1:], positions, inv_freq, w, None, 1e-6, None, True)
    check(torch.randn(1 + 2 * 4 * 7 * 128, generator=g).to(DEV)[1:].view(2, 4, 7, 128), None, positions, inv_freq, w, None, 1e-6, None, True)
    check(proj[:1, :, :1].transpose(1, 2).expand(2, 3, 7, 128), None, positions, inv_freq, w, None, 1e-6, None, False)
    for shape in ((0, 2, 3, 128), (2, 2, 0, 128)):
        x = torch.zeros(shape, device=DEV)
        y, none = qk_norm_rope(x, None, torch.zeros(shape[0], shape[2], dtype=torch.int64, device=DEV), inv_freq.to(DEV))
        assert y.shape == shape and none is None


def test_rows_stay_apart():
    """Infinities and NaN of one row reach no other row; zero rows stay zero."""
    from omnistack_rs_b200.kernels.position import qk_norm_rope
    x = torch.randn(1, 4, 5, 128, device=DEV, generator=torch.Generator(DEV).manual_seed(0))
    x[0, 1, 2, 3], x[0, 2, 2, 3], x[0, 3, 4] = float("nan"), float("inf"), 0.0
    pos, freq = torch.arange(5, device=DEV), 10000.0 ** (-torch.arange(32, device=DEV) / 32)
    y, _ = qk_norm_rope(x, None, pos, freq)
    bad = ~torch.isfinite(y).all(-1)
    assert bad[0, 1, 2] and bad[0, 2, 2] and int(bad.sum()) == 2
    assert bool((y[0, 3, 4] == 0).all())
    raw, _ = qk_norm_rope(x, None, pos, freq, eps=None)
    x[0, 1, 2, 100] = float("inf")                                               # behind the rotated dims: passes through alone
    raw2, _ = qk_norm_rope(x, None, pos, freq, eps=None)
    assert raw2[0, 1, 2, 100] == float("inf") and torch.equal(raw2[0, 1, 2, 64:100], raw[0, 1, 2, 64:100])
