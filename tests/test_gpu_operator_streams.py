"""The prompt-side and eviction operators on several streams at once: the same bits as one after the other."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def work(seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    real = lambda *s, dt=torch.bfloat16: torch.randn(*s, generator=g, device=DEV).to(dt)  # noqa: E731
    byte = lambda *s: torch.randint(0, 256, s, generator=g, device=DEV, dtype=torch.uint8)  # noqa: E731
    B, H, S = 12, 4, 900 + 100 * seed
    rows = byte(B, H, S, 64), byte(B, H, S, 8), real(B, H, S, dt=torch.float32).abs()
    lens = torch.randint(0, S + 1, (B,), generator=g, device=DEV)
    cb = real(H, 16, dt=torch.float32)
    return dict(q=real(1, 16, 1500, 128), k=real(1, 4, 1500, 128), cu=torch.tensor([0, 300, 300, 1234, 1480], dtype=torch.int32, device=DEV),
                positions=torch.arange(1500, device=DEV) * (seed + 1), freq=10000.0 ** (-torch.arange(64, device=DEV) / 64),
                one=real(B, 8, 1, 128), many=real(B, 8, 30, 128), rows=rows, v=byte(B, H, S, 64), cb=cb, lens=lens.to(torch.int32))


def run(w):
    from omnistack_rs_b200.kernels.eviction import attn_weight_sums, evict_keys
    from omnistack_rs_b200.kernels.position import qk_norm_rope
    from omnistack_rs_b200.kernels.prompt_attention import prompt_attn
    q, k = qk_norm_rope(w["q"], w["k"], w["positions"], w["freq"])
    out = prompt_attn(q, k, w["k"], cu_seqlens=w["cu"])
    sums = attn_weight_sums(w["one"], *w["rows"], w["cb"], seq_lens=w["lens"])
    attn_weight_sums(w["many"], *w["rows"], w["cb"], seq_lens=w["lens"], rotate_q=True, into=sums)
    kept = evict_keys(sums, *w["rows"], w["v"], 400, recent=30, seq_lens=w["lens"], v_paired=True)
    return [q, k, out, sums, *[x for x in kept if x is not None]]


def test_streams_at_once():
    sets = [work(seed) for seed in range(3)]
    want = [run(w) for w in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for _ in range(6):
        for s, w in zip(streams, sets):
            with torch.cuda.stream(s):
                got.append(run(w))
    torch.cuda.synchronize()
    for i, xs in enumerate(got):
        assert all(torch.equal(x, y) for x, y in zip(xs, want[i % len(sets)]))


def test_captured_graphs_at_once():
    """Two graphs of the same operators share no scratch: replayed on two streams at once, each gives its own results."""
    sets = [work(seed) for seed in (3, 4)]
    want = [[x.clone() for x in run(w)] for w in sets]
    graphs, outs = [], []
    for w in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(run(w))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(5):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for xs, ys in zip(outs, want):
        assert all(torch.equal(x, y) for x, y in zip(xs, ys))
