"""What the prompt-side and eviction operators refuse, checked before anything reaches a GPU."""
import pytest
import torch

from omnistack_rs_b200 import _lib, build
from omnistack_rs_b200.kernels import eviction, position, prompt_attention
from omnistack_rs_b200.kernels.eviction import attn_weight_sums, evict_keys
from omnistack_rs_b200.kernels.position import qk_norm_rope
from omnistack_rs_b200.kernels.prompt_attention import prompt_attn

Z = torch.zeros


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


@pytest.mark.parametrize("change,error,match", [
    (dict(q=Z(1, 2, 3, 64)), ValueError, "head_dim"), (dict(k=Z(1, 1, 4, 128)), ValueError, "like q"), (dict(k=Z(1, 1, 3, 64)), ValueError, "like q"),
    (dict(q=Z(2, 3, 128)), ValueError, "n_heads"), (dict(q=Z(1, 2, 3, 128, dtype=torch.float64)), TypeError, "dtype"),
    (dict(k=Z(1, 1, 3, 128, dtype=torch.float16)), TypeError, "different dtypes"), (dict(inv_freq=Z(65)), ValueError, "inv_freq"),
    (dict(inv_freq=Z(64, dtype=torch.bfloat16)), TypeError, "inv_freq"), (dict(positions=Z(1, 3)), TypeError, "positions"),
    (dict(positions=Z(4, dtype=torch.int64)), ValueError, "positions"), (dict(positions=Z(2, 1, 3, dtype=torch.int64)), ValueError, "positions"),
    (dict(axis_pairs=(32, 31)), ValueError, "axis_pairs"), (dict(axis_pairs=(16, 16, 16, 8, 8)), ValueError, "axis_pairs"),
    (dict(axis_pairs=(80, -16)), ValueError, "axis_pairs"), (dict(axis_pairs=(32, 32)), ValueError, "positions"),
    (dict(q_weight=Z(64)), ValueError, "q_weight"), (dict(eps=None, q_weight=Z(128)), ValueError, "eps=None"),
    (dict(), RuntimeError, "no CPU fallback"),
])
def test_norm_rope_refusals(change, error, match):
    args = dict(q=Z(1, 2, 3, 128), k=Z(1, 1, 3, 128), positions=Z(1, 3, dtype=torch.int64), inv_freq=Z(64)) | change
    with pytest.raises(error, match=match):
        qk_norm_rope(args.pop("q"), args.pop("k"), args.pop("positions"), args.pop("inv_freq"), **args)


I32 = dict(dtype=torch.int32)


@pytest.mark.parametrize("change,error,match", [
    (dict(q=Z(1, 4, 6, 64)), ValueError, "head_dim"), (dict(k=Z(1, 2, 5, 128)), ValueError, "like q"), (dict(v=Z(1, 1, 6, 128)), ValueError, "like q"),
    (dict(q=Z(1, 3, 6, 128)), ValueError, "multiple"), (dict(q=Z(1, 4, 6, 128, dtype=torch.float64)), TypeError, "dtype"),
    (dict(v=Z(1, 2, 6, 128, dtype=torch.bfloat16)), TypeError, "different dtypes"),
    (dict(cu_seqlens=Z(2, **I32), seq_lens=Z(1, **I32)), ValueError, "not both"), (dict(seq_lens=Z(2, **I32)), ValueError, "seq_lens"),
    (dict(seq_lens=torch.tensor([7])), ValueError, "lie in"), (dict(seq_lens=torch.tensor([-1])), ValueError, "lie in"),
    (dict(cu_seqlens=torch.tensor([0, 4, 3, 6])), ValueError, "ascend"), (dict(cu_seqlens=torch.tensor([0, 7])), ValueError, "lie in"),
    (dict(cu_seqlens=Z(0, **I32)), ValueError, "cu_seqlens"), (dict(cu_seqlens=torch.tensor([0.0, 6.0])), TypeError, "cu_seqlens"),
    (dict(q=Z(2, 4, 6, 128), k=Z(2, 2, 6, 128), v=Z(2, 2, 6, 128), cu_seqlens=torch.tensor([0, 6])), ValueError, "one user"),
    (dict(), RuntimeError, "no CPU fallback"),
])
def test_prompt_refusals(change, error, match):
    args = dict(q=Z(1, 4, 6, 128), k=Z(1, 2, 6, 128), v=Z(1, 2, 6, 128)) | change
    with pytest.raises(error, match=match):
        prompt_attn(args.pop("q"), args.pop("k"), args.pop("v"), **args)


U8 = dict(dtype=torch.uint8)


def cache(B=2, H=2, S=5):
    return dict(k_nibbles=Z(B, H, S, 64, **U8), k_qjl=Z(B, H, S, 8, **U8), k_norms=Z(B, H, S))


@pytest.mark.parametrize("change,error,match", [
    (dict(q=Z(2, 4, 1, 64)), ValueError, "head_dim"), (dict(q=Z(3, 4, 1, 128)), ValueError, "users"), (dict(q=Z(2, 3, 1, 128)), ValueError, "multiple"),
    (dict(q=Z(2, 4, 1, 128, dtype=torch.float64)), TypeError, "dtype"), (dict(k_qjl=Z(2, 2, 5, 4, **U8)), ValueError, "k_qjl"),
    (dict(k_norms=Z(2, 2, 5, dtype=torch.float64)), ValueError, "k_norms"), (dict(k_nibbles=Z(2, 2, 5, 64)), ValueError, "k_nibbles"),
    (dict(into=Z(2, 2, 4)), ValueError, "into"), (dict(into=Z(2, 5, 2).transpose(1, 2)), ValueError, "contiguous"),
    (dict(), RuntimeError, "no CPU fallback"),
])
def test_weight_sums_refusals(change, error, match):
    args = dict(q=Z(2, 4, 1, 128), codebooks=Z(16)) | cache() | change
    with pytest.raises(error, match=match):
        attn_weight_sums(args.pop("q"), args.pop("k_nibbles"), args.pop("k_qjl"), args.pop("k_norms"), args.pop("codebooks"), **args)


@pytest.mark.parametrize("change,error,match", [
    (dict(budget=0), ValueError, "budget"), (dict(recent=4), ValueError, "budget"), (dict(recent=-1), ValueError, "budget"),
    (dict(capacity=2), ValueError, "budget"), (dict(sums=Z(2, 2, 6)), ValueError, "sums"), (dict(sums=Z(2, 2, 5, dtype=torch.float16)), ValueError, "sums"),
    (dict(v_qjl=Z(2, 2, 5, 8, **U8)), ValueError, "both"), (dict(v_nibbles=Z(2, 2, 4, 64, **U8)), ValueError, "v_nibbles"),
    (dict(), RuntimeError, "no CPU fallback"),
])
def test_evict_refusals(change, error, match):
    args = dict(sums=Z(2, 2, 5), v_nibbles=Z(2, 2, 5, 64, **U8), budget=3) | cache() | change
    with pytest.raises(error, match=match):
        evict_keys(args.pop("sums"), args.pop("k_nibbles"), args.pop("k_qjl"), args.pop("k_norms"), args.pop("v_nibbles"), args.pop("budget"), **args)


def test_c_entries_refuse_bad_arguments(lib):
    """Checks that need no device: they come before the first CUDA call of each entry."""
    assert lib.omni_qk_norm_rope(None, None) == _lib.ERR_ARG
    def norm_rope(q=16, heads=1, axes=1, pairs=0, end=0, stride=128, dtype=1):
        return lib.omni_qk_norm_rope(position._NORM_ROPE.pack(q, 0, 16, 0, 0, 0, 16, 16, 0, 0, stride, 0, 0, 0, 0, 0, 0, 1, 1, heads, 0, 0, 0, end, 0, 0, 0,
                                                              dtype, axes, pairs, 0, 0, 0, 1, 1e-6), None)
    assert norm_rope(q=0) == norm_rope(q=8) == norm_rope(heads=-1) == norm_rope(pairs=65, end=65) == norm_rope(pairs=8) == _lib.ERR_ARG
    assert norm_rope(stride=132) == norm_rope(dtype=7) == _lib.ERR_ARG and norm_rope(axes=5) == _lib.ERR_UNSUPPORTED and norm_rope(heads=0) == _lib.OK
    assert lib.omni_prompt_attn(None, None) == lib.omni_attn_weight_sums(None, None) == _lib.ERR_ARG
    prompt = lambda q=32, out=32, dt=1, stride=128, n=1, B=1, Hq=2, Hkv=1, T=4, cu=0: lib.omni_prompt_attn(prompt_attention._PROMPT.pack(  # noqa: E731
        q, 32, 32, out, cu, 0, 0, 0, 0, stride, 0, 0, 128, 0, 0, 128, n, B, T, dt, Hq, Hkv, 1, 1.0), None)
    assert prompt(q=0) == prompt(q=8) == prompt(out=16) == prompt(dt=3) == prompt(Hq=3, Hkv=2) == prompt(n=2) == _lib.ERR_ARG
    assert prompt(stride=130) == prompt(cu=32, B=2) == prompt(T=-1) == _lib.ERR_ARG
    assert prompt(T=1 << 31) == _lib.ERR_UNSUPPORTED and prompt(T=0) == _lib.OK
    assert lib.omni_attn_weight_sums_workspace_bytes(0, 4, 2, 1, 100) == 0
    sums = lambda q=16, Hq=4, Hkv=2, S=64, ws=0: lib.omni_attn_weight_sums(eviction._WEIGHT_SUMS.pack(  # noqa: E731
        q, 16, 16, 16, 16, 0, 0, 16, 16, 0, 1, S, ws, 1, 0, 0, Hq, Hkv, 1, 1, 0, 1, 0, 1.0), None)
    assert sums(q=0) == sums(Hq=3) == sums(ws=0) == _lib.ERR_ARG and sums(S=0) == _lib.OK
    assert sums(Hq=2048, Hkv=2048) == _lib.ERR_UNSUPPORTED
    assert lib.omni_evict_keys(None, None) == _lib.ERR_ARG
    evict = lambda capacity, nib=16, B=1: lib.omni_evict_keys(  # noqa: E731
        eviction._EVICT.pack(16, 0, nib, 16, 16, 16, 0, 0, 16, 16, 16, 16, 16, 0, 0, 16, 16, B, 8, 4, 0, capacity, 1, 0), None)
    assert evict(3) == evict(4, nib=0) == evict(4, nib=8) == evict(4, B=-1) == _lib.ERR_ARG and evict(4, B=0) == _lib.OK
