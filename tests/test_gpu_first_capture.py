"""A graph that holds the first call on a device does not own the device's status word."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def test_status_word_of_a_first_call_that_is_captured(monkeypatch):
    from omnistack_rs_b200 import _lib
    from omnistack_rs_b200.kernels.prompt_attention import prompt_attn
    q = torch.randn(1, 2, 50, 128, generator=torch.Generator(device=DEV).manual_seed(0), device=DEV, dtype=torch.bfloat16)
    want = prompt_attn(q, q, q)
    monkeypatch.setattr(_lib, "_status_words", {})                       # as in a process that has made no call yet
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = prompt_attn(q, q, q)
    _lib.check_device_status(DEV)                                        # nothing to report before the first replay
    graph.replay()
    assert torch.equal(out, want)
    _lib.status_word(DEV).fill_(4)                                       # what an expired wait of another call leaves
    graph.replay()
    with pytest.raises(RuntimeError, match="wait expired"):
        _lib.check_device_status(DEV)
    _lib.check_device_status(DEV)
    del graph, out
    torch.cuda.empty_cache()
    _lib.check_device_status(DEV)
