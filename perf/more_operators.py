"""The work a serving program gives the layers of bounded state of a hybrid decoder, and the step's answer.

Beside KDA layers a hybrid decoder has layers that keep a bounded state of another kind (linear attention with
a decay for each head; attention over a sliding window whose first tokens, the sinks, stay visible), and its step
ends in a token drawn from the logits. Every case is one call of a public wrapper
(``sgl_glm53_ascend_ops.ops``) on tensors that are already on the GPU:

* ``op = "recurrent"``: ``linear_varlen_recurrent``, ``requests`` of ``low`` to ``high`` tokens each, token by token on
  states of a slot pool; ``checkpoints``: the state after every token is written instead of the last one.
* ``op = "chunk"``: ``linear_varlen_chunk``, the same on prompts; ``track``: the state after a prefix of each request
  goes into a slot of its own; ``after`` tokens behind the last request belong to none.
* ``op = "sample"``: ``sample_tokens``, ``rows`` of ``vocab`` logits (``fp32`` or bf16), each with its own parameters:
  temperatures around 1 (every ``greedy``-th row 0), the largest ``top_k`` at most, a nucleus of ``top_p`` at least, and
  ``min_p`` of the largest weight at most (0 each: not used). The token and the log of its probability come back.
* ``op = "attention"``: ``paged_attention`` with a ``window`` and ``sinks`` first tokens that stay visible: ``q_low`` to
  ``q_high`` new tokens of each of ``requests`` requests over ``kv_low`` to ``kv_high`` earlier ones and themselves.

Lengths are drawn with ``lens_seed`` (part of the case). ``gated``: a log decay for each token and head, else one
for each head. ``fused``: q, k, v are slices of one projection. ``index64``: the metadata is int64 instead of
int32. Sizes are those of this repository's measured configurations (4, 16 or 32 heads of 64 or 128; 8192 and
16384 tokens; 256 sequences; contexts to 32 K) and generic ones.
"""

import math
import os
import random
import sys

import torch

own = False

DEV = "cuda"
FP8 = torch.float8_e4m3fn
FP8_MAX = 448.0
INF = float("inf")


def _linear(op, requests, low, high, heads, dim, **more):
    return dict(dict(op=op, requests=requests, low=low, high=high, heads=heads, dim=dim, gated=True, fp32=False, fused=False,
                     checkpoints=False, track=False, after=0, padding=0, lens_seed=0, index64=False), **more)


def _sample(rows, vocab, **more):
    return dict(dict(op="sample", rows=rows, vocab=vocab, fp32=False, greedy=0, top_k=0, top_p=0.0, min_p=0.0), **more)


def _attention(requests, q_low, q_high, kv_low, kv_high, heads, kv_heads, dim, page, window, sinks, **more):
    return dict(dict(op="attention", requests=requests, q_low=q_low, q_high=q_high, kv_low=kv_low, kv_high=kv_high,
                     heads=heads, kv_heads=kv_heads, dim=dim, page=page, window=window, sinks=sinks, fp8=False, fused=False,
                     cap=0.0, lens_seed=0, index64=False), **more)


def listed():
    return [
        # One request's next token on a 16-head shard: the smallest call, where latency counts.
        dict(_linear("recurrent", 1, 1, 1, 16, 128), name="recurrent_1"),
        # A speculative verify step: 64 requests' four drafted tokens, the state after each kept; constant decays.
        dict(_linear("recurrent", 64, 4, 4, 16, 128, gated=False, checkpoints=True, index64=True), name="recurrent_verify_64"),
        # A large decode step, a padded batch: every 16th request has no state of its own.
        dict(_linear("recurrent", 256, 1, 1, 32, 128, fused=True, padding=16), name="recurrent_256"),
        # A batch of prompts of any length, a prefix of each kept for reuse; heads of 64, constant decays, padded tokens.
        dict(_linear("chunk", 37, 1, 2000, 16, 64, gated=False, track=True, after=57, lens_seed=1), name="chunk_ragged"),
        # A long prompt on the 4 heads of one shard: the recurrence itself is what there is little of.
        dict(_linear("chunk", 1, 16001, 16001, 4, 128, fused=True), name="chunk_16k_4_heads"),
        # A long prompt on all heads: the largest.
        dict(_linear("chunk", 1, 8192, 8192, 32, 128), name="chunk_8k"),
        # One request's next token from the usual filters.
        dict(_sample(1, 131072, top_k=50, top_p=0.9), name="sample_1"),
        # A batch that only has temperatures, some rows greedy; fp32 logits of an odd vocabulary.
        dict(_sample(37, 32001, fp32=True, greedy=5), name="sample_37_fp32"),
        # A large batch with a nucleus and a floor but no top-k: the filters need the whole row's mass.
        dict(_sample(256, 150000, top_p=0.8, min_p=0.02), name="sample_256"),
        # One request's next token far into a long conversation.
        dict(_attention(1, 1, 1, 30000, 30000, 32, 8, 128, 16, 4096, 4), name="sinks_decode_1"),
        # A decode batch with contexts from nothing to 32 K on layers with a window.
        dict(_attention(256, 1, 1, 0, 32767, 32, 8, 128, 64, 2048, 16, lens_seed=2, index64=True), name="sinks_decode_256"),
        # A prefill step in chunks: several requests' new tokens over long cached prefixes.
        dict(_attention(6, 300, 2048, 1000, 30000, 32, 8, 128, 16, 1024, 64, lens_seed=3), name="sinks_chunks"),
    ]


def _log(rng, low, high):
    """A whole number between the two, spread over its logarithm."""
    return max(low, min(high, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["recurrent", "recurrent", "chunk", "chunk", "sample", "sample", "decode", "prefill"])
    more = dict(index64=rng.random() < 0.3, lens_seed=rng.randrange(1 << 20))
    if kind in ("recurrent", "chunk"):
        heads, dim = rng.choice([4, 8, 16, 32, 5]), rng.choice([64, 128, 128])
        more.update(gated=rng.random() < 0.6, fused=rng.random() < 0.4, padding=rng.choice([0, 0, 7]))
        if kind == "recurrent":
            steps = rng.choice([1, 1, 2, 4, 8])
            checkpoints = steps > 1 and rng.random() < 0.6
            n = _log(rng, 1, 8192 // heads // (steps if checkpoints else 1))
            return _linear("recurrent", min(n, 1024), rng.randint(1, steps), steps, heads, dim, checkpoints=checkpoints,
                           fp32=rng.random() < 0.3, **more)
        n = _log(rng, 1, 64)
        high = _log(rng, 16, (8192 * 32 * 128) // (n * heads * dim))
        return _linear("chunk", n, rng.choice([1, high]), min(high, 32768), heads, dim, track=rng.random() < 0.4,
                       after=rng.choice([0, 0, 33]), **more)
    if kind == "sample":
        vocab = rng.choice([32000, 65536, 131072, _log(rng, 100, 200000)])
        rows = _log(rng, 1, min(512, 256 * 150000 // vocab))
        return _sample(rows, vocab, fp32=vocab * rows * 2 <= 256 * 150000 and rng.random() < 0.4, greedy=rng.choice([0, 3]),
                       top_k=rng.choice([0, 0, _log(rng, 1, min(vocab, 1000)), _log(rng, 1, vocab)]),
                       top_p=rng.choice([0.0, 0.5, 0.9, 0.99]), min_p=rng.choice([0.0, 0.0, 0.001, 0.05]))
    heads, kv_heads = rng.choice([(16, 16), (32, 8), (64, 8), (24, 8), (32, 2), (40, 8), (7, 1)])
    more.update(fp8=rng.random() < 0.4, fused=rng.random() < 0.3, cap=rng.choice([0.0, 0.0, 30.0]))
    dim, page = rng.choice([64, 128, 128]), rng.choice([1, 16, 64, 100])
    window, sinks = _log(rng, 16, 4096), rng.choice([1, 4, 4, 64, _log(rng, 1, 300)])
    if kind == "decode":
        n = _log(rng, 1, 256)
        steps = rng.choice([1, 1, 4])
        window = min(window, 256 * 2048 * 8 * 128 // (n * kv_heads * dim) - 600)
        high = _log(rng, 16, min(65536, (3 << 28) // (n * kv_heads * dim) - steps))
        return _attention(n, steps, steps, rng.choice([0, high]), high, heads, kv_heads, dim, page, max(window, 1), sinks, **more)
    n = _log(rng, 1, 8)
    q = _log(rng, 64, 5000 * 32 // (n * max(heads, 16)))
    kv = _log(rng, 64, 32768)
    return _attention(n, rng.randint(1, q), q, rng.choice([0, kv]), kv, heads, kv_heads, dim, page, min(window, 1024), sinks, **more)


def _lengths(case):
    """Tokens of each request of a linear layer."""
    rng = random.Random(case["lens_seed"])
    return [rng.randint(case["low"], case["high"]) for _ in range(case["requests"])]


def _attention_lengths(case):
    """New tokens and keys (the new ones among them) of each request."""
    rng = random.Random(case["lens_seed"])
    new = [rng.randint(case["q_low"], case["q_high"]) for _ in range(case["requests"])]
    return new, [n + rng.randint(case["kv_low"], case["kv_high"]) for n in new]


def _prepare_linear(case, gen, randn, index):
    state = dict(case=case)
    lens = _lengths(case)
    N, H, D, T = case["requests"], case["heads"], case["dim"], sum(lens) + case["after"]
    dtype = torch.float32 if case["fp32"] else torch.bfloat16
    if case["fused"]:
        qkv = randn(1, T, 3 * H, D).to(dtype)
        state["q"], state["k"], state["v"] = qkv[:, :, :H], qkv[:, :, H:2 * H], qkv[:, :, 2 * H:]
    else:
        state["q"], state["k"], state["v"] = (randn(1, T, H, D).to(dtype) for _ in range(3))
    if case["gated"]:  # from hardly any decay to one within a token
        state["g"] = -torch.exp(randn(1, T, H) * 1.5 - 3.0)
    else:  # a geometric series over the heads
        state["g"] = -torch.pow(2.0, -8.0 * torch.arange(1, H + 1, device=DEV) / H)
    slots = 1 + N * (2 if case["track"] else 1)
    # slot 0 is the padding row; K contiguous
    state["pool"] = randn(slots, H, D, D).transpose(2, 3)
    state["pool"][0] = 0.0
    order = torch.randperm(slots - 1, generator=gen, device=DEV) + 1
    at = order[:N].clone()
    if case["padding"]:
        at[case["padding"] - 1::case["padding"]] = 0
    state["indices"] = at.to(index)
    state["cu_seqlens"] = torch.tensor([0] + lens, device=DEV).cumsum(0).to(index)
    state["scale"] = D ** -0.5
    if case["track"]:
        state["track_indices"] = order[N:].to(index)
        state["track_lens"] = (torch.rand(N, generator=gen, device=DEV) * (torch.tensor(lens, device=DEV) + 1)).long().to(index)
    if case["checkpoints"]:
        state["middle"] = torch.zeros(N, case["high"], H, D, D, device=DEV).transpose(3, 4)
    return state


def _prepare_sample(case, gen, randn):
    state = dict(case=case)
    N, V = case["rows"], case["vocab"]
    logits = randn(N, V) * 2.0
    some = min(V, 64)  # the tokens that fit the context, some rows sure of a few and others not
    at = torch.randint(V, (N, some), generator=gen, device=DEV)
    height = 4.0 + 8.0 * torch.rand(N, 1, generator=gen, device=DEV)
    logits.scatter_add_(1, at, height - 1.5 * torch.arange(1, some + 1, device=DEV).float().log() + randn(N, some) * 0.5)
    state["logits"] = logits.to(torch.float32 if case["fp32"] else torch.bfloat16)
    state["uniforms"] = torch.rand(N, generator=gen, device=DEV)
    row = torch.arange(N, device=DEV)
    t = 0.6 + 0.8 * torch.rand(N, generator=gen, device=DEV)
    state["temperature"] = torch.where(row % case["greedy"] == 1, 0.0, t) if case["greedy"] else t
    x = torch.rand(3, N, generator=gen, device=DEV)
    state["top_k"] = torch.exp(x[0] * math.log(case["top_k"])).round().int() if case["top_k"] else None
    state["top_p"] = case["top_p"] + (1.0 - case["top_p"]) * x[1] if case["top_p"] else None
    state["min_p"] = case["min_p"] * x[2] if case["min_p"] else None
    return state


def _prepare_attention(case, gen, randn, index):
    state = dict(case=case)
    KH, D, page, dtype = case["kv_heads"], case["dim"], case["page"], torch.bfloat16
    state["k_scale"] = state["v_scale"] = None
    if case["fp8"]:  # a scale per key head, from the range that its keys or values have
        state["k_scale"] = 0.01 + 0.005 * torch.rand(KH, generator=gen, device=DEV)
        state["v_scale"] = 0.01 + 0.005 * torch.rand(KH, generator=gen, device=DEV)

    def cache(pages, scale):
        if scale is None:
            return randn(pages, page, KH, D).to(dtype)
        return (randn(pages, page, KH, D) / scale[:, None]).clamp(-FP8_MAX, FP8_MAX).to(FP8)

    new, keys = _attention_lengths(case)
    T, H = sum(new), case["heads"]
    used = [-(-n // page) for n in keys]
    width, pages = max(1, max(used)), sum(used) + 2
    state["q"] = randn(1, T, H + 2 * KH, D).to(dtype)[:, :, :H] if case["fused"] else randn(1, T, H, D).to(dtype)
    state["k_cache"], state["v_cache"] = cache(pages, state["k_scale"]), cache(pages, state["v_scale"])
    order = torch.randperm(pages, generator=gen, device=DEV)
    counts = torch.tensor(used, device=DEV)
    first = counts.cumsum(0) - counts
    column = torch.arange(width, device=DEV)
    at = torch.minimum(first[:, None] + column[None, :], torch.tensor(pages - 1, device=DEV))
    state["page_table"] = torch.where(column[None, :] < counts[:, None], order[at], 0).to(index)
    state["kv_lens"] = torch.tensor(keys, device=DEV).to(index)
    state["cu_seqlens"] = torch.tensor([0] + new, device=DEV).cumsum(0).to(index)
    state["max_query_len"] = max(new)
    state["scale"] = D ** -0.5
    return state


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=DEV)

    if case["op"] == "sample":
        return _prepare_sample(case, gen, randn)
    index = torch.int64 if case["index64"] else torch.int32
    return (_prepare_attention if case["op"] == "attention" else _prepare_linear)(case, gen, randn, index)


def _run_own(state):
    case = state["case"]
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "01-glm53-ascend_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from sgl_glm53_ascend_ops import ops

    if case["op"] == "sample":
        tokens, logprobs = ops.sample_tokens(state["logits"], state["uniforms"], temperature=state["temperature"],
                                             top_k=state["top_k"], top_p=state["top_p"], min_p=state["min_p"])
        return {"tokens": tokens, "logprobs": logprobs}
    if case["op"] == "attention":
        return {"out": ops.paged_attention(
            state["q"], k_cache=state["k_cache"], v_cache=state["v_cache"], page_table=state["page_table"],
            kv_lens=state["kv_lens"], cu_seqlens=state["cu_seqlens"], scale=state["scale"],
            max_query_len=state["max_query_len"], window=case["window"], sink_tokens=case["sinks"], logit_cap=case["cap"],
            k_scale=state["k_scale"], v_scale=state["v_scale"])}
    args = dict(initial_state_source=state["pool"], initial_state_indices=state["indices"], cu_seqlens=state["cu_seqlens"],
                scale=state["scale"])
    if case["track"]:
        args.update(track_state_indices=state["track_indices"], track_state_lens=state["track_lens"])
    if case["op"] == "chunk":
        out = ops.linear_varlen_chunk(state["q"], state["k"], state["v"], state["g"], **args)
    else:
        if case["checkpoints"]:
            args["intermediate_state"] = state["middle"]
        out = ops.linear_varlen_recurrent(state["q"], state["k"], state["v"], state["g"], **args)
    return {"out": out, **({"middle": state["middle"]} if case["checkpoints"] else {"pool": state["pool"]})}


def _linear_plain(state):
    """All requests at once, padded to the longest: token by token, or 64 tokens at a time (chunk)."""
    case, pool = state["case"], state["pool"]
    N, H, D = case["requests"], case["heads"], case["dim"]
    cu, slots = state["cu_seqlens"].long(), state["indices"].long()
    T = state["q"].shape[1]
    lens = cu[1:] - cu[:-1]
    step = 64 if case["op"] == "chunk" else 1
    L = -(-max(_lengths(case)) // step) * step
    t = torch.arange(L, device=DEV)
    real = t[None, :] < lens[:, None]  # [N, L]
    token = torch.where(real, cu[:-1, None] + t[None, :], 0)

    def padded(x):
        return torch.where(real[:, None, :, None], x[0][token].float().transpose(1, 2), 0.0)  # [N, H, L, D]

    q, k, v = padded(state["q"]), padded(state["k"]), padded(state["v"])
    g = state["g"].double().expand(1, T, H)[0][token].transpose(1, 2)  # [N, H, L]
    g = torch.where(real[:, None, :], g, 0.0)
    S = pool[slots].clone()  # [N, H, K, V]; slot 0 holds zeros
    out = torch.empty(N, H, L, D, device=DEV)
    if case["track"]:  # the state after a prefix, from the definition's sum
        upto = state["track_lens"].long()
        total = g.cumsum(2)
        there = torch.where(t[None, :] < upto[:, None], 0.0, -INF)[:, None, :]
        end = torch.where((upto > 0)[:, None, None], total.gather(2, (upto - 1).clamp_min(0)[:, None, None].expand(N, H, 1)), 0.0)
        weight = torch.exp(end - total + there).float()
        tracked = torch.matmul((k * weight[..., None]).transpose(2, 3), v) + torch.exp(end).float()[..., None] * S
        pool[state["track_indices"].long()] = tracked
    for a in range(0, L, step):
        sum_g = g[:, :, a:a + step].cumsum(2)
        qa, ka, va = q[:, :, a:a + step], k[:, :, a:a + step], v[:, :, a:a + step]
        if step == 1:
            S = torch.exp(sum_g).float()[..., None] * S + ka.transpose(2, 3) * va
            out[:, :, a:a + 1] = torch.matmul(qa, S)
            if case["checkpoints"]:
                kept = (real[:, a] & (slots > 0)).nonzero()[:, 0]
                state["middle"][kept, a] = S[kept]
            continue
        apart = sum_g[..., :, None] - sum_g[..., None, :]
        seen = torch.ones(step, step, dtype=torch.bool, device=DEV).tril()
        weight = torch.exp(torch.where(seen, apart, -INF)).float()
        scores = torch.matmul(qa, ka.transpose(2, 3)) * weight
        out[:, :, a:a + step] = torch.matmul(scores, va) + torch.exp(sum_g).float()[..., None] * torch.matmul(qa, S)
        late = torch.exp(sum_g[..., -1:] - sum_g).float()
        S = torch.exp(sum_g[..., -1:]).float()[..., None] * S + torch.matmul((ka * late[..., None]).transpose(2, 3), va)
    result = torch.zeros(1, T, H, D, dtype=state["q"].dtype, device=DEV)
    result[0, token[real]] = (out * state["scale"]).transpose(1, 2)[real].to(result.dtype)
    if case["checkpoints"]:
        return {"out": result, "middle": state["middle"]}
    kept = (slots > 0).nonzero()[:, 0]
    pool[slots[kept]] = S[kept]
    return {"out": result, "pool": pool}


def _sample_plain(state):
    """In 64 bits: a token next to a border has to fall on its right side."""
    case, logits = state["case"], state["logits"].double()
    N, V = logits.shape
    t = state["temperature"].double()[:, None]
    top = logits.amax(1, keepdim=True)
    first = (logits == top).int().argmax(1)
    w = torch.exp((logits - top) / torch.where(t > 0, t, 1.0))
    if state["top_k"] is not None or state["top_p"] is not None:
        values, order = torch.sort(logits, dim=1, descending=True, stable=True)
        rank = torch.arange(V, device=DEV)
        w = w.gather(1, order)
        if state["top_k"] is not None:
            most = torch.where(state["top_k"] > 0, state["top_k"], V)
            w = torch.where(rank < most[:, None], w, 0.0)
        if state["top_p"] is not None:
            total = w.cumsum(1)
            before = total - w
            p = state["top_p"].double()[:, None]
            w = torch.where((p >= 1) | (before < p * total[:, -1:]) | (rank == 0), w, 0.0)
        w = torch.zeros_like(w).scatter_(1, order, w)
    if state["min_p"] is not None:
        w = torch.where(w >= state["min_p"].double()[:, None], w, 0.0)
    total = w.cumsum(1)
    token = (total > state["uniforms"].double()[:, None] * total[:, -1:]).int().argmax(1)
    logprob = torch.log(w.gather(1, token[:, None]) / total[:, -1:])[:, 0]
    return {"tokens": torch.where(t[:, 0] > 0, token, first), "logprobs": torch.where(t[:, 0] > 0, logprob, 0.0).float()}


def _attention_plain(state):
    """All requests at once, padded: the sinks and the keys from the first window's start, masked softmax, product."""
    case, q = state["case"], state["q"][0]
    table, lens, cu = state["page_table"].long(), state["kv_lens"].long(), state["cu_seqlens"].long()
    T, H, D = q.shape
    KH, page, N, Q = case["kv_heads"], case["page"], case["requests"], state["max_query_len"]
    G, window, sinks = H // KH, case["window"], case["sinks"]
    new = cu[1:] - cu[:-1]
    low = (lens - new - window + 1).clamp_min(0)  # the first key that a window holds
    longest = int(min(max(_attention_lengths(case)[1]), Q + window - 1))
    key = torch.cat([torch.arange(sinks, device=DEV).expand(N, sinks),
                     torch.maximum(low, torch.tensor(sinks, device=DEV))[:, None] + torch.arange(longest, device=DEV)], 1)
    held = key < lens[:, None]  # [N, L]
    L = key.shape[1]
    place = torch.where(held, key, 0)
    pages, offsets = table.gather(1, place // page), place % page
    t = torch.arange(Q, device=DEV)
    rows = torch.minimum(cu[:-1, None] + t[None, :], cu[1:, None] - 1)  # [N, Q]
    at = (lens - new)[:, None] + t[None, :]  # position of each new token
    out = torch.zeros(N, Q, H, D, device=DEV)
    some = max(1, (1 << 28) // (Q * G * L * N))  # key heads at a time
    for h in range(0, KH, some):
        hs = slice(h, min(h + some, KH))

        def gathered(cache, scale):
            flat = cache[:, :, hs][pages, offsets].float()  # [N, L, heads, D]
            return flat if scale is None else flat * scale[hs][:, None]

        k = gathered(state["k_cache"], state["k_scale"]).permute(0, 2, 3, 1).contiguous()
        x = q[rows].float().view(N, Q, KH, G, D)[:, :, hs].permute(0, 2, 1, 3, 4).reshape(N, -1, Q * G, D)
        s = torch.matmul(x, k) * state["scale"]
        if case["cap"]:
            s = case["cap"] * torch.tanh(s / case["cap"])
        seen = held[:, None, :] & (key[:, None, :] <= at[:, :, None])
        seen &= (key[:, None, :] > at[:, :, None] - window) | (key < sinks)[:, None, :]
        s = s.view(N, -1, Q, G, L).masked_fill_(~seen[:, None, :, None, :], -INF)
        p = torch.exp(s - s.amax(-1, keepdim=True))  # a token sees itself
        total = p.sum(-1, keepdim=True)
        v = gathered(state["v_cache"], state["v_scale"]).permute(0, 2, 1, 3).contiguous()
        o = torch.matmul(p.view(N, -1, Q * G, L), v).view(N, -1, Q, G, D) / total
        out.view(N, Q, KH, G, D)[:, :, hs] = o.permute(0, 2, 1, 3, 4)
    token = torch.arange(T, device=DEV)
    request = (token[:, None] >= cu[None, 1:]).sum(1)
    return {"out": out[request, token - cu[request]].to(q.dtype)[None]}


def run(state):
    if own:
        return _run_own(state)
    plain = {"recurrent": _linear_plain, "chunk": _linear_plain, "sample": _sample_plain, "attention": _attention_plain}
    return plain[state["case"]["op"]](state)


def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (4 if case["fp32"] else 2) + case["rows"] * 32, "flops": 4 * n}
    if case["op"] == "attention":
        KH, D = case["kv_heads"], case["dim"]
        x, i = 1 if case["fp8"] else 2, 8 if case["index64"] else 4
        keys = pairs = entries = 0
        new, lens = _attention_lengths(case)
        for m, n in zip(new, lens):
            low = max(0, n - m - case["window"] + 1)
            sinks = min(case["sinks"], low)
            keys += n - low + sinks
            entries += -(-(n - low + sinks) // case["page"])
            for p in range(n - m, n):
                a = max(0, p - case["window"] + 1)
                pairs += p + 1 - a + min(case["sinks"], a)
        size = sum(new) * case["heads"] * D * 4 + keys * KH * D * 2 * x + (entries + 2 * len(new) + 1) * i
        return {"bytes": size, "flops": 4 * D * case["heads"] * pairs}
    lens = _lengths(case)
    N, H, D, T = case["requests"], case["heads"], case["dim"], sum(lens) + case["after"]
    held = N - (N // case["padding"] if case["padding"] else 0)  # requests with a state of their own
    if case["checkpoints"]:
        kept = sum(n for i, n in enumerate(lens) if not case["padding"] or (i + 1) % case["padding"])
    else:
        kept = held + (N if case["track"] else 0)
    states = (held + kept) * H * D * D * 4
    size = 4 * T * H * D * (4 if case["fp32"] else 2) + (T if case["gated"] else 1) * H * 4
    return {"bytes": states + size + (2 * N + 1) * (8 if case["index64"] else 4), "flops": 5 * sum(lens) * H * D * D}


def _linear_exact(case, state):
    """Every output as one sum over the earlier tokens, request by request."""
    f = torch.float64
    lens, D, H = _lengths(case), case["dim"], case["heads"]
    pool = state["pool"].to(f)
    begin = pool.clone()
    middle = state["middle"].to(f) if case["checkpoints"] else None
    out = torch.zeros(state["q"].shape, dtype=f, device=DEV)
    at = 0
    slots = state["indices"].tolist()
    if case["track"]:
        to, upto = state["track_indices"].tolist(), state["track_lens"].tolist()
    for n, m in enumerate(lens):
        q, k, v = (state[x][0, at:at + m].to(f).permute(1, 0, 2).contiguous() for x in ("q", "k", "v"))  # [H, m, D]
        g = state["g"].to(f)[0, at:at + m].t() if case["gated"] else state["g"].to(f)[:, None].expand(H, m)
        G = torch.cumsum(g, 1)
        S = begin[slots[n]] if slots[n] > 0 else torch.zeros(H, D, D, dtype=f, device=DEV)

        def after(count):
            if count == 0:
                return S
            w = (G[:, count - 1:count] - G[:, :count]).exp()
            return G[:, count - 1].exp()[:, None, None] * S + (k[:, :count] * w[..., None]).transpose(1, 2).contiguous() @ v[:, :count]

        for h in range(H):
            for a in range(0, m, 4096):
                b = min(a + 4096, m)
                lag = G[h, a:b, None] - G[h, None, :b]
                hidden = torch.arange(b, device=DEV)[None, :] > torch.arange(a, b, device=DEV)[:, None]
                scores = (q[h, a:b] @ k[h, :b].t().contiguous()) * lag.masked_fill(hidden, -INF).exp()
                o = scores @ v[h, :b] + G[h, a:b].exp()[:, None] * (q[h, a:b] @ S[h])
                out[0, at + a:at + b, h] = o * state["scale"]
        if case["track"]:
            pool[to[n]] = after(upto[n])
        if case["checkpoints"]:
            if slots[n] > 0:
                for i in range(m):
                    middle[n, i] = after(i + 1)
        elif slots[n] > 0:
            pool[slots[n]] = after(m)
        at += m
    return {"out": out, **({"middle": middle} if case["checkpoints"] else {"pool": pool})}


def _sample_exact(case, state):
    """Row by row from the sorted logits."""
    tokens, logprobs = [], []
    for n in range(case["rows"]):
        x = state["logits"][n].to(torch.float64)
        if state["temperature"][n] == 0:
            tokens.append(int((x == x.max()).nonzero()[0]))
            logprobs.append(0.0)
            continue
        x = x / state["temperature"][n].to(torch.float64)
        order = torch.argsort(x, descending=True, stable=True)
        if state["top_k"] is not None and state["top_k"][n] > 0:
            order = order[:int(state["top_k"][n])]
        p = torch.softmax(x[order], 0)
        if state["top_p"] is not None and state["top_p"][n] < 1:
            most = int((torch.cumsum(p, 0) < state["top_p"][n].to(torch.float64)).sum()) + 1
            p, order = p[:most], order[:most]
        if state["min_p"] is not None:
            most = max(1, int((p >= state["min_p"][n].to(torch.float64) * p[0]).sum()))
            p, order = p[:most], order[:most]
        order, by_index = torch.sort(order)
        mass = torch.cumsum(p[by_index], 0)
        at = int((mass <= state["uniforms"][n].to(torch.float64) * mass[-1]).sum())
        at = min(at, len(order) - 1)
        tokens.append(int(order[at]))
        logprobs.append(math.log(float(p[by_index][at]) / float(mass[-1])))
    return {"tokens": torch.tensor(tokens, device=DEV), "logprobs": torch.tensor(logprobs, dtype=torch.float64, device=DEV)}


def _attention_exact(case, state):
    f = torch.float64
    new, keys = _attention_lengths(case)
    H, KH, D, page, window = case["heads"], case["kv_heads"], case["dim"], case["page"], case["window"]
    out = torch.zeros(state["q"].shape, dtype=f, device=DEV)
    start = 0
    for n, (m, length) in enumerate(zip(new, keys)):
        low = max(0, length - m - window + 1)
        j = torch.cat([torch.arange(min(case["sinks"], low), device=DEV), torch.arange(low, length, device=DEV)])
        where = state["page_table"][n].long()[j // page], j % page
        for h in range(KH):
            k = state["k_cache"][:, :, h][where].to(f)
            v = state["v_cache"][:, :, h][where].to(f)
            if case["fp8"]:
                k, v = k * state["k_scale"][h].to(f), v * state["v_scale"][h].to(f)
            k = k.t().contiguous()
            heads = slice(h * (H // KH), (h + 1) * (H // KH))
            for t0 in range(0, m, 1024):
                t1 = min(m, t0 + 1024)
                q = state["q"][0, start + t0:start + t1, heads].to(f)
                z = (q.reshape(-1, D) @ k).view(t1 - t0, -1, len(j)) * state["scale"]
                if case["cap"]:
                    z = case["cap"] * torch.tanh(z / case["cap"])
                p = torch.arange(length - m + t0, length - m + t1, device=DEV)[:, None, None]
                visible = (j <= p) & ((p - j < window) | (j < case["sinks"]))
                z = torch.softmax(z.masked_fill(~visible, -INF), -1)
                out[0, start + t0:start + t1, heads] = (z.flatten(0, 1) @ v).view(t1 - t0, -1, D)
        start += m
    return {"out": out}


def exact(case, seed):
    """The definitions in 64 bits, request by request and row by row."""
    state = prepare(case, seed)
    if case["op"] == "sample":
        return _sample_exact(case, state)
    return _attention_exact(case, state) if case["op"] == "attention" else _linear_exact(case, state)
