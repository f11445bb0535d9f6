"""Packed rows and queries of the key weights and of eviction start on 16-byte boundaries, sign bytes on 8: others are refused by the C
entries before anything is launched."""
import pytest

from omnistack_rs_b200 import _lib, build
from omnistack_rs_b200.kernels import eviction


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def test_misaligned_buffers_are_refused(lib):
    need = lib.omni_attn_weight_sums_workspace_bytes(1, 4, 2, 1, 64)
    sums = lambda q=16, nib=16, qjl=16, scratch=16: lib.omni_attn_weight_sums(eviction._WEIGHT_SUMS.pack(  # noqa: E731
        q, nib, qjl, 16, 16, 0, 0, scratch, 16, 0, 1, 64, need, 1, 0, 0, 4, 2, 1, 1, 0, 1, 0, 1.0), None)
    for change in (dict(q=24), dict(nib=24), dict(qjl=20), dict(scratch=24)):
        assert sums(**change) == _lib.ERR_ARG
        assert b"misaligned" in lib.omni_last_error()
    evict = lambda k=16, kq=16, v=16, out=16, oq=16: lib.omni_evict_keys(eviction._EVICT.pack(  # noqa: E731
        16, 0, k, kq, 16, v, 0, 0, 16, out, oq, 16, 16, 0, 0, 16, 16, 1, 8, 4, 0, 4, 1, 0), None)
    for change in (dict(k=24), dict(kq=20), dict(v=24), dict(out=24), dict(oq=20)):
        assert evict(**change) == _lib.ERR_ARG
        assert b"misaligned" in lib.omni_last_error()
