"""Prompt-side and eviction operators around the packed cache: what they are, and calls of them over their real ranges.

Four kinds of work, one for each operator:

  position  ``qk_norm_rope``: per-head norm of queries and keys and their position rotation (one axis, or time/height/width)
  prompt    ``prompt_attn``: attention of whole prompts over themselves, grouped heads, packed or padded sequences
  weights   ``attn_weight_sums``: the softmax weight every cached key receives from a set of queries
  evict     ``evict_keys``: the heaviest and the latest keys of every head, gathered into a smaller cache

``own`` selects between the package's kernels and the plain form of the same definition in elementary torch operations.
"""
import functools
import math

import torch

own = False

HEAD_DIM = 128
PROJECTIONS = 64
QJL_COEF = math.sqrt(2.0 / math.pi) / HEAD_DIM
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
DTYPE_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
# 16-level Lloyd-Max levels of a unit Gaussian (what calibration of rotated N(0, 1) rows gives)
LEVELS = (-2.733, -2.069, -1.618, -1.256, -0.9424, -0.6568, -0.3881, -0.1284,
          0.1284, 0.3881, 0.6568, 0.9424, 1.256, 1.618, 2.069, 2.733)
IMAGE_AXES = (16, 24, 24)                 # pairs that follow time, height and width


def listed():
    return [
        # one decode step of 64 users: norm and rotation of one token's queries and keys at far positions (the smallest call)
        dict(kind="position", name="position_decode_64", users=64, q_heads=32, kv_heads=8, tokens=1, dtype="bf16", axes=1,
             start=900000, interleaved=False, rotated=128),
        # a prompt's queries and keys as views of the projection's output
        dict(kind="position", name="position_prompt_8x2048", users=8, q_heads=32, kv_heads=8, tokens=2048, dtype="bf16", axes=1,
             start=0, interleaved=False, rotated=128),
        # image tokens with three position axes, odd length, neighbouring pairs, half of the dims rotated in fp32
        dict(kind="position", name="position_axes_fp16_3x4095", users=3, q_heads=32, kv_heads=4, tokens=4095, dtype="fp16", axes=3,
             start=0, interleaved=False, rotated=128),
        dict(kind="position", name="position_partial_fp32_5x777", users=5, q_heads=8, kv_heads=8, tokens=777, dtype="fp32", axes=1,
             start=31000, interleaved=True, rotated=64),
        # the histories of one ranking query: 64 prompts of at most 50 tokens, packed
        dict(kind="prompt", name="prompt_packed_64x50", prompts=64, longest=50, shortest=1, q_heads=32, kv_heads=8, dtype="bf16",
             packed=True, causal=True),
        # a batch of ragged prompts, packed
        dict(kind="prompt", name="prompt_packed_16x2048", prompts=16, longest=2048, shortest=100, q_heads=32, kv_heads=8,
             dtype="bf16", packed=True, causal=True),
        # one long prompt (the largest call)
        dict(kind="prompt", name="prompt_long_16384", prompts=1, longest=16384, shortest=16384, q_heads=32, kv_heads=8,
             dtype="fp16", packed=False, causal=True),
        # fp32 check of a model on padded prompts without the causal mask, ungrouped heads
        dict(kind="prompt", name="prompt_full_fp32_4x611", prompts=4, longest=611, shortest=65, q_heads=8, kv_heads=8,
             dtype="fp32", packed=False, causal=False),
        # weights of one decoding step over the caches of a serving loop
        dict(kind="weights", name="weights_step_64x1500", users=64, q_heads=32, kv_heads=8, keys=1500, shortest=375, queries=1,
             dtype="bf16", per_head=True),
        # the last 32 tokens of long prompts decide what is kept of them
        dict(kind="weights", name="weights_window_32_16x8192", users=16, q_heads=32, kv_heads=8, keys=8192, shortest=1024,
             queries=32, dtype="bf16", per_head=False),
        # long prompts cut down to 1,024 keys per head
        dict(kind="evict", name="evict_64x8192_to_1024", users=64, kv_heads=8, keys=8192, shortest=600, budget=1024, recent=64,
             pair=True, residual=False),
        # a few users in the reference layout, V's sign bits and norms kept, odd sizes
        dict(kind="evict", name="evict_5x2047_to_777", users=5, kv_heads=4, keys=2047, shortest=500, budget=777, recent=33,
             pair=False, residual=True),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["position", "prompt", "prompt", "weights", "evict"])
    if kind == "position":
        kv_heads = rng.choice([1, 4, 8])
        q_heads = kv_heads * rng.choice([1, 3, 4])
        tokens = _log_int(rng, 1, 4096)
        axes = rng.choice([1, 1, 3])
        return dict(kind=kind, users=_log_int(rng, 1, max(1, min(64, 16384 * 40 // (tokens * (q_heads + kv_heads))))), q_heads=q_heads,
                    kv_heads=kv_heads, tokens=tokens, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), axes=axes,
                    start=rng.choice([0, 5000, 900000]), interleaved=rng.choice([False, True]),
                    rotated=128 if axes == 3 else rng.choice([128, 64, 32]))
    if kind == "prompt":
        longest = _log_int(rng, 1, 12000)
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"]) if longest <= 1500 else rng.choice(["bf16", "fp16"])
        kv_heads = rng.choice([1, 2, 8])
        q_heads = kv_heads * rng.choice([1, 3, 4, 8]) if kv_heads < 8 else rng.choice([8, 32])
        most = max(1, min(64, int(16384 ** 2 * 32 / (longest ** 2 * q_heads)), 65536 // longest))
        prompts = _log_int(rng, 1, most)
        return dict(kind=kind, prompts=prompts, longest=longest, shortest=_log_int(rng, 1, longest), q_heads=q_heads,
                    kv_heads=kv_heads, dtype=dtype, packed=rng.choice([True, True, False]), causal=rng.random() < 0.75)
    keys = _log_int(rng, 16, 8192)
    kv_heads = rng.choice([1, 4, 8])
    if kind == "weights":
        queries = rng.choice([1, 1, 1, 4, 16, 32])
        users = _log_int(rng, 1, max(1, min(256, 8 * 8192 * 64 // (keys * kv_heads))))
        return dict(kind=kind, users=users, q_heads=kv_heads * rng.choice([1, 2, 4]), kv_heads=kv_heads, keys=keys,
                    shortest=_log_int(rng, 1, keys), queries=queries, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                    per_head=rng.random() < 0.5)
    budget = _log_int(rng, 8, keys)
    return dict(kind=kind, users=_log_int(rng, 1, max(1, min(256, 8 * 8192 * 64 // (keys * kv_heads)))), kv_heads=kv_heads, keys=keys,
                shortest=_log_int(rng, 1, keys), budget=budget, recent=rng.randint(0, min(budget, 64)), pair=rng.random() < 0.5,
                residual=rng.random() < 0.5)


# ---- inputs ------------------------------------------------------------------------------------------------------------

def _lengths(shortest, longest, count):
    """The case's lengths: spread over [shortest, longest], the longest always among them (host values, as a scheduler has
    them).  They go by the case alone, and the seed gives their order, so that a case is the same work for every seed."""
    lens = torch.randint(shortest, longest + 1, (count,), generator=torch.Generator().manual_seed(longest * 1000 + count))
    lens[0] = longest
    return lens


def _shuffled(lens, seed):
    return lens[torch.randperm(lens.numel(), generator=torch.Generator().manual_seed(seed))]


@functools.lru_cache(maxsize=1)
def _sign_rows():
    """The codec's +-1 projections of all 1,024 seeds, (1024, 64, 128) int8 (one MT19937 stream per seed)."""
    rows = [torch.randint(0, 2, (PROJECTIONS, HEAD_DIM), generator=torch.Generator().manual_seed(s), dtype=torch.int8) for s in range(1024)]
    return torch.stack(rows) * 2 - 1


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    kind = case["kind"]
    if kind == "position":
        B, T, Hq, Hkv = case["users"], case["tokens"], case["q_heads"], case["kv_heads"]
        dtype = DTYPES[case["dtype"]]
        # queries and keys as the fused projection leaves them: one row per token, heads side by side
        proj = (torch.randn(B, T, Hq + 2 * Hkv, HEAD_DIM, generator=g, device=dev) * 1.7).to(dtype)
        q, k = proj[:, :, :Hq].transpose(1, 2), proj[:, :, Hq:Hq + Hkv].transpose(1, 2)
        weight = lambda: 1.0 + 0.2 * torch.randn(HEAD_DIM, generator=g, device=dev)  # noqa: E731
        pairs = case["rotated"] // 2
        inv_freq = 10000.0 ** (-torch.arange(pairs, dtype=torch.float64, device=dev) / pairs)
        first = torch.randint(0, 1000, (B, 1), generator=g, device=dev) + case["start"]
        step = torch.arange(T, device=dev)[None]
        if case["axes"] == 1:
            positions, axis_pairs = first + step, None
        else:                                                       # frames of 45 x 91 patches
            positions, axis_pairs = torch.stack([first + step // 4095, (step // 91) % 45 + 0 * first, step % 91 + 0 * first]), IMAGE_AXES
        return dict(case=case, q=q, k=k, positions=positions, inv_freq=inv_freq.float(), axis_pairs=axis_pairs,
                    q_weight=weight(), k_weight=weight())
    if kind == "prompt":
        Hq, Hkv, n = case["q_heads"], case["kv_heads"], case["prompts"]
        dtype = DTYPES[case["dtype"]]
        lens = _shuffled(_lengths(case["shortest"], case["longest"], n), seed)
        rows = int(lens.sum()) if case["packed"] else case["longest"]
        B = 1 if case["packed"] else n
        make = lambda H, scale: (torch.randn(B, H, rows, HEAD_DIM, generator=g, device=dev) * scale).to(dtype)  # noqa: E731
        state = dict(case=case, q=make(Hq, 1.5), k=make(Hkv, 1.5), v=make(Hkv, 1.0), longest=case["longest"],
                     lens=lens.to(device=dev, dtype=torch.int32), cu_seqlens=None)
        if case["packed"]:
            state["cu_seqlens"] = torch.cat([torch.zeros(1, dtype=torch.int64), lens.cumsum(0)]).to(device=dev, dtype=torch.int32)
        return state
    B, H, S = case["users"], case["kv_heads"], case["keys"]
    lens = _shuffled(_lengths(case["shortest"], S, B), seed).to(device=dev, dtype=torch.int32)
    row_bytes = lambda n: torch.randint(0, 256, (B, H, S, n), generator=g, device=dev, dtype=torch.uint8)  # noqa: E731
    norms = lambda: 1.0 + 0.1 * torch.randn(B, H, S, generator=g, device=dev)  # noqa: E731
    state = dict(case=case, lens=lens, k_nib=row_bytes(64), k_qjl=row_bytes(8), k_norms=norms())
    if kind == "weights":
        cb = torch.tensor(LEVELS, device=dev)
        if case["per_head"]:
            cb = cb * (1 + 0.05 * torch.arange(H, device=dev)[:, None])
        q = torch.randn(B, case["q_heads"], case["queries"], HEAD_DIM, generator=g, device=dev) * 1.5
        return dict(state, q=q.to(DTYPES[case["dtype"]]), codebooks=cb, user_ids=torch.arange(B, dtype=torch.int32, device=dev),
                    sign_rows=_sign_rows().to(dev))
    # weight sums are heavy-tailed, and keys that nothing ever attended to share the value zero
    sums = torch.exp(2.0 * torch.randn(B, H, S, generator=g, device=dev))
    sums = sums * (torch.rand(B, H, S, generator=g, device=dev) > 0.05)
    v_nib = row_bytes(64)
    return dict(state, sums=sums, v_nib=v_nib, v_qjl=row_bytes(8) if case["residual"] else None,
                v_norms=norms() if case["residual"] else None)


# ---- plain forms -------------------------------------------------------------------------------------------------------

def _norm_rope_plain(x, weight, cos, sin, interleaved):
    """cos and sin (B, 1, T, pairs) fp32."""
    y = x.float()
    y = y * torch.rsqrt(y.square().mean(dim=-1, keepdim=True) + 1e-6) * weight
    pairs = cos.shape[-1]
    turned, rest = y[..., :2 * pairs], y[..., 2 * pairs:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = turned[..., :pairs], turned[..., pairs:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([turned, rest], dim=-1).to(x.dtype)


def _angles(state):
    """(B, 1, T, pairs) fp64; the angles of far positions need more than 24 bits."""
    positions, inv_freq = state["positions"], state["inv_freq"].double()
    if state["axis_pairs"] is None:
        return positions[:, None, :, None].double() * inv_freq
    axis = torch.arange(len(state["axis_pairs"]), device=inv_freq.device).repeat_interleave(
        torch.tensor(state["axis_pairs"], device=inv_freq.device), output_size=inv_freq.numel())
    return positions.permute(1, 2, 0)[:, None, :, axis].double() * inv_freq


def _prompt_plain(state):
    """Every prompt on rows of its own (padded to the longest), one dense product for all of them."""
    case, lens = state["case"], state["lens"].long()
    L, Hkv = state["longest"], case["kv_heads"]
    G = case["q_heads"] // Hkv
    scale = 1.0 / math.sqrt(HEAD_DIM)
    step = torch.arange(L, device=lens.device)
    inside = step[None] < lens[:, None]                                         # (prompts, L)
    if case["packed"]:
        rows = (state["cu_seqlens"][:-1].long()[:, None] + step[None]).clamp(max=state["q"].shape[2] - 1)
        q, k, v = (state[n][0][:, rows].transpose(0, 1) for n in "qkv")         # (prompts, H, L, 128)
    else:
        q, k, v = state["q"], state["k"], state["v"]
    n = q.shape[0]
    scores = torch.matmul(q.float().reshape(n, Hkv, G * L, HEAD_DIM), k.float().transpose(-1, -2)).mul_(scale)
    scores = scores.view(n, Hkv, G, L, L)
    allowed = inside[:, None, :].expand(n, L, L)
    if case["causal"]:
        allowed = allowed & (step[None, None, :] <= step[None, :, None])
    scores.masked_fill_(~allowed[:, None, None], float("-inf"))
    scores.sub_(scores.amax(dim=-1, keepdim=True)).exp_()
    total = scores.sum(dim=-1, keepdim=True)
    out = torch.matmul(scores.view(n, Hkv, G * L, L), v.float()).view(n, Hkv, G, L, HEAD_DIM) / total
    out = out.reshape(n, Hkv * G, L, HEAD_DIM).to(state["q"].dtype)
    if case["packed"]:
        return out.transpose(1, 2)[inside].transpose(0, 1)[None].contiguous()
    return out * inside[:, None, :, None]


def _weights_plain(state):
    case, lens = state["case"], state["lens"].long()
    B, H, S, T = case["users"], case["kv_heads"], case["keys"], case["queries"]
    G, dev = case["q_heads"] // H, lens.device
    cb = state["codebooks"].expand(H, 16)
    byte = torch.arange(256, device=dev)
    pairs = torch.stack([cb[:, byte & 15], cb[:, byte >> 4]], dim=-1).view(H * 256, 2)     # the two centroids a byte stands for
    head = torch.arange(H, device=dev, dtype=torch.int32)
    k = pairs[state["k_nib"].int() + 256 * head[:, None, None]].view(B, H, S, HEAD_DIM)
    bits = (state["k_qjl"][..., None] >> torch.arange(8, device=dev, dtype=torch.uint8)) & 1
    signs = bits.view(B, H, S, PROJECTIONS).float() * 2 - 1
    rows = state["sign_rows"][((state["user_ids"].long()[:, None] % 1024) ^ head.long()[None])].float()
    k = k + torch.matmul(signs, rows) * (state["k_norms"] * QJL_COEF)[..., None]
    q = state["q"].float().reshape(B, H, G, T, HEAD_DIM)
    scores = torch.matmul(q.reshape(B, H, G * T, HEAD_DIM), k.transpose(-1, -2)).view(B, H, G, T, S) / math.sqrt(HEAD_DIM)
    step = torch.arange(S, device=dev)
    last = lens[:, None] - T + torch.arange(T, device=dev)[None]                            # the newest key query t may see
    allowed = (step <= last[..., None]) & (step < lens[:, None, None])
    scores = scores.masked_fill(~allowed[:, None, None], float("-inf"))
    top = scores.amax(dim=-1, keepdim=True)
    p = torch.exp(scores - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(dim=-1, keepdim=True)
    return torch.where(total > 0, p / total, torch.zeros_like(p)).sum(dim=(2, 3))


def _pair_rows(v, lens):
    """The pair layout of V's nibble rows, applied to every group of eight rows that lies completely below the length
    (applied twice, it gives the rows back)."""
    S = v.shape[2]
    at = torch.arange(S, device=v.device)
    other = v[:, :, (at ^ 3).clamp(max=S - 1)]
    first = ((at & 2) == 0)[:, None]
    changed = torch.where(first, (v & 15) | ((other & 15) << 4), (other >> 4) | (v & 240))
    whole = at[None] < (lens.long()[:, None] // 8) * 8
    return torch.where(whole[:, None, :, None], changed, v)


def _evict_plain(state):
    case, lens = state["case"], state["lens"].long()
    S, budget, dev = case["keys"], case["budget"], lens.device
    at = torch.arange(S, device=dev)
    inf = torch.full((), float("inf"), device=dev)
    key = torch.where((at[None] >= lens[:, None] - case["recent"])[:, None], inf, state["sums"])
    key = torch.where((at[None] >= lens[:, None])[:, None], -inf, key)
    index = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :budget].sort(dim=-1).values
    new_lens = lens.clamp(max=budget)
    valid = (torch.arange(budget, device=dev)[None] < new_lens[:, None])[:, None].expand_as(index)
    take = lambda x: None if x is None else torch.gather(  # noqa: E731
        x, 2, index.view(*index.shape, *([1] * (x.dim() - 3))).expand(*index.shape, *x.shape[3:])) * (
            valid if x.dim() == 3 else valid[..., None]).to(x.dtype)
    v_nib = take(_pair_rows(state["v_nib"], lens) if case["pair"] else state["v_nib"])
    return [torch.where(valid, index, -1).int(), new_lens.int(), take(state["sums"]), take(state["k_nib"]), take(state["k_qjl"]),
            take(state["k_norms"]), _pair_rows(v_nib, new_lens) if case["pair"] else v_nib, take(state["v_qjl"]), take(state["v_norms"])]


def run(state):
    case = state["case"]
    if own:
        return _run_own(state)
    if case["kind"] == "position":
        angles = _angles(state)
        cos, sin = torch.cos(angles).float(), torch.sin(angles).float()
        return [_norm_rope_plain(state["q"], state["q_weight"], cos, sin, case["interleaved"]),
                _norm_rope_plain(state["k"], state["k_weight"], cos, sin, case["interleaved"])]
    return {"prompt": _prompt_plain, "weights": _weights_plain, "evict": _evict_plain}[case["kind"]](state)


def _run_own(state):
    case = state["case"]
    if case["kind"] == "position":
        from omnistack_rs_b200.kernels.position import qk_norm_rope
        return list(qk_norm_rope(state["q"], state["k"], state["positions"], state["inv_freq"], q_weight=state["q_weight"],
                                 k_weight=state["k_weight"], eps=1e-6, axis_pairs=state["axis_pairs"],
                                 interleaved=case["interleaved"]))
    if case["kind"] == "prompt":
        from omnistack_rs_b200.kernels.prompt_attention import prompt_attn
        lengths = dict(cu_seqlens=state["cu_seqlens"]) if case["packed"] else dict(seq_lens=state["lens"])
        return prompt_attn(state["q"], state["k"], state["v"], causal=case["causal"], **lengths)
    if case["kind"] == "weights":
        from omnistack_rs_b200.kernels.eviction import attn_weight_sums
        return attn_weight_sums(state["q"], state["k_nib"], state["k_qjl"], state["k_norms"], state["codebooks"],
                                user_id=state["user_ids"], seq_lens=state["lens"])
    from omnistack_rs_b200.kernels.eviction import evict_keys
    return list(evict_keys(state["sums"], state["k_nib"], state["k_qjl"], state["k_norms"], state["v_nib"], case["budget"],
                           recent=case["recent"], seq_lens=state["lens"], v_qjl=state["v_qjl"], v_norms=state["v_norms"],
                           v_paired=case["pair"]))


# ---- what a pass cannot do without -------------------------------------------------------------------------------------

def work(case):
    if case["kind"] == "position":
        rows = case["users"] * case["tokens"] * (case["q_heads"] + case["kv_heads"])
        return {"bytes": 2 * rows * HEAD_DIM * DTYPE_BYTES[case["dtype"]] + 8 * case["axes"] * case["users"] * case["tokens"],
                "flops": 8 * rows * HEAD_DIM}
    if case["kind"] == "prompt":
        lens = _lengths(case["shortest"], case["longest"], case["prompts"])
        rows = int(lens.sum())
        written = rows if case["packed"] else case["prompts"] * case["longest"]
        pairs = int((lens * (lens + 1) // 2 if case["causal"] else lens * lens).sum())
        return {"bytes": (rows * (case["q_heads"] + 2 * case["kv_heads"]) + written * case["q_heads"]) * HEAD_DIM * DTYPE_BYTES[case["dtype"]],
                "flops": 4 * HEAD_DIM * case["q_heads"] * pairs}
    lens = _lengths(case["shortest"], case["keys"], case["users"])
    keys = case["kv_heads"] * int(lens.sum())
    heads = case["users"] * case["kv_heads"]
    if case["kind"] == "weights":
        columns = case["q_heads"] // case["kv_heads"] * case["queries"]
        return {"bytes": 76 * keys + 4 * heads * case["keys"] + heads * columns * HEAD_DIM * DTYPE_BYTES[case["dtype"]],
                "flops": 2 * (HEAD_DIM + PROJECTIONS) * columns * keys}
    kept = case["kv_heads"] * int(lens.clamp(max=case["budget"]).sum())
    row = 144 + (12 if case["residual"] else 0)
    return {"bytes": 4 * keys + row * kept + (row + 4) * heads * case["budget"], "flops": keys}


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------

def _exact_position(state, name):
    x, w = state[name].double(), state[name + "_weight"].double()
    case, pairs = state["case"], state["inv_freq"].numel()
    y = x / torch.sqrt((x * x).sum(-1, keepdim=True) / HEAD_DIM + 1e-6) * w
    out = y.clone()
    axes = state["axis_pairs"] or (pairs,)
    positions = state["positions"] if state["axis_pairs"] else state["positions"][None]
    i = 0
    for a, count in enumerate(axes):
        for _ in range(count):
            angle = (positions[a].double() * float(state["inv_freq"][i]))[:, None]
            first, second = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + pairs)
            out[..., first] = y[..., first] * torch.cos(angle) - y[..., second] * torch.sin(angle)
            out[..., second] = y[..., second] * torch.cos(angle) + y[..., first] * torch.sin(angle)
            i += 1
    return out


def _exact_prompt(state):
    case = state["case"]
    G = case["q_heads"] // case["kv_heads"]
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
    begin = 0
    for b, n in enumerate(state["lens"].tolist()):
        at, r0 = (0, begin) if case["packed"] else (b, 0)
        begin += n
        for h in range(case["q_heads"]):
            k, v = state["k"][at, h // G, r0:r0 + n].double(), state["v"][at, h // G, r0:r0 + n].double()
            for i in range(0, n, 4096):
                m = min(n, i + 4096)
                s = state["q"][at, h, r0 + i:r0 + m].double() @ k.T / math.sqrt(HEAD_DIM)
                if case["causal"]:
                    s += torch.full_like(s, -math.inf).triu(i + 1)
                out[at, h, r0 + i:r0 + m] = torch.softmax(s, dim=-1) @ v
    return out


def _exact_weights(state):
    case = state["case"]
    B, H, S, T = case["users"], case["kv_heads"], case["keys"], case["queries"]
    G = case["q_heads"] // H
    out = torch.zeros(B, H, S, dtype=torch.float64, device="cuda")
    shifts = torch.arange(8, device="cuda")
    for b, n in enumerate(state["lens"].tolist()):
        for h in range(H):
            cb = (state["codebooks"][h] if case["per_head"] else state["codebooks"]).double()
            nib = state["k_nib"][b, h, :n].long()
            k = torch.empty(n, HEAD_DIM, dtype=torch.float64, device="cuda")
            k[:, 0::2], k[:, 1::2] = cb[nib % 16], cb[nib // 16]
            sign = 2.0 * ((state["k_qjl"][b, h, :n].long()[..., None] >> shifts) % 2).reshape(n, PROJECTIONS).double() - 1.0
            seed = (int(state["user_ids"][b]) % 1024) ^ h
            k += state["k_norms"][b, h, :n, None].double() * QJL_COEF * (sign @ state["sign_rows"][seed].double())
            q = state["q"][b, h * G:(h + 1) * G].double()                        # (G, T, 128)
            for t in range(max(0, T - n), T):
                m = n - T + t + 1
                out[b, h, :m] += torch.softmax(q[:, t] @ k[:m].T / math.sqrt(HEAD_DIM), dim=-1).sum(0)
    return out


def exact(case, seed):
    if case["kind"] == "evict":
        return None                                                               # nothing is computed: rows are chosen and moved
    if case["kind"] == "weights" and case["users"] * case["kv_heads"] * case["queries"] > 20000:
        return None
    state = prepare(case, seed)
    if case["kind"] == "position":
        return [_exact_position(state, "q"), _exact_position(state, "k")]
    return _exact_prompt(state) if case["kind"] == "prompt" else _exact_weights(state)
