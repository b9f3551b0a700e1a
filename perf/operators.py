"""The work a serving program gives the operators of a decoder's full-attention layers and norms.

The KDA operators are one kind of layer of a hybrid decoder; these stand between and beside them. Every
case is one call of a public wrapper (``sgl_glm53_ascend_ops.ops``) on tensors that are already on the GPU:

* ``op = "norm"``: ``add_rms_norm`` (the output has the input's type) or, with ``out8``,
  ``add_rms_norm_fp8`` (8-bit floats with a scale per row, or per ``group`` columns). ``rows`` x ``width``,
  ``fp32`` or bf16, ``residual`` added and updated in place.
* ``op = "store"``: ``paged_kv_store``, the new tokens' keys and values into the pages of a cache, in bf16
  or (``fp8``) in 8 bits with a scale per head. ``tokens`` of ``kv_heads`` x ``dim``; k and v are slices of
  one fused projection where ``fused``; every ``padding``-th token has no slot.
* ``op = "attention"``: ``paged_attention`` of ``q_low`` to ``q_high`` new tokens of each of ``requests``
  requests over ``kv_low`` to ``kv_high`` earlier ones and themselves, the lengths drawn with ``lens_seed``
  (part of the case). ``heads`` query heads on ``kv_heads``, ``dim`` wide, pages of ``page`` tokens in
  shuffled order; ``window`` keys are visible (0: all), scores capped by ``cap`` * tanh (0: not).

``index64``: the metadata is int64 instead of int32. Sizes are those of this repository's measured
configurations (16, 32 or 64 heads of 64 or 128; 8192 tokens; 256 sequences) and generic ones.
"""

import os
import random
import sys

import torch

own = False

DEV = "cuda"
EPS = 1e-6
FP8 = torch.float8_e4m3fn
FP8_MAX = 448.0
MIN_SCALE = 1e-12


def _norm(rows, width, **more):
    return dict(dict(op="norm", rows=rows, width=width, fp32=False, residual=True, out8=False, group=0), **more)


def _store(tokens, kv_heads, dim, page, **more):
    return dict(dict(op="store", tokens=tokens, kv_heads=kv_heads, dim=dim, page=page, pages=2 * tokens // page + 2,
                     fp8=False, fused=False, padding=0, index64=False), **more)


def _attention(requests, q_low, q_high, kv_low, kv_high, heads, kv_heads, dim, page, **more):
    return dict(dict(op="attention", requests=requests, q_low=q_low, q_high=q_high, kv_low=kv_low, kv_high=kv_high,
                     heads=heads, kv_heads=kv_heads, dim=dim, page=page, fp8=False, fused=False, window=0, cap=0.0,
                     lens_seed=0, index64=False), **more)


def listed():
    return [
        # The hidden row of one request's next token: the smallest call, where latency counts.
        dict(_norm(1, 4096), name="norm_1"),
        # An fp32 hidden state of an odd width: no row is aligned like the next one.
        dict(_norm(1001, 5003, fp32=True), name="norm_fp32_odd"),
        # A small decode batch before an 8-bit projection, one scale a row, no residual yet (the first layer).
        dict(_norm(37, 2048, residual=False, out8=True), name="norm_fp8_37"),
        # A whole prefill step before an 8-bit projection with block scales.
        dict(_norm(8192, 8192, out8=True, group=128), name="norm_fp8_8k"),
        # One decode step's keys and values of 256 sequences; a padded batch, int64 slots.
        dict(_store(256, 8, 128, 16, padding=16, index64=True), name="store_256"),
        # A prefill step's keys and values, slices of the fused projection, into an 8-bit cache.
        dict(_store(8192, 8, 128, 64, fp8=True, fused=True), name="store_fp8_8k"),
        # One request's next token over a medium context: a single call's latency.
        dict(_attention(1, 1, 1, 4000, 4000, 32, 8, 128, 16), name="decode_1"),
        # A ragged decode batch, contexts from nothing to 32k.
        dict(_attention(64, 1, 1, 0, 32767, 64, 8, 128, 64, lens_seed=2, index64=True), name="decode_64_ragged"),
        # A large decode batch on an 8-bit cache managed token by token, 16 query heads a key head.
        dict(_attention(256, 1, 1, 6000, 8191, 32, 2, 128, 1, fp8=True, lens_seed=3), name="decode_256_fp8"),
        # Speculative verify on sliding-window layers with capped scores: 3 query heads a key head, heads of 64.
        dict(_attention(32, 4, 4, 500, 6000, 24, 8, 64, 16, window=1000, cap=30.0, lens_seed=4), name="verify_window_cap"),
        # A prefill step in chunks: several requests' new tokens over long cached prefixes.
        dict(_attention(6, 100, 512, 1000, 30000, 32, 8, 128, 16, lens_seed=5), name="chunks_over_30k"),
        # A long prompt's attention from its start: the largest product.
        dict(_attention(1, 8192, 8192, 0, 0, 32, 8, 128, 64, fused=True), name="prefill_8k"),
    ]


def _log(rng, low, high):
    """A whole number between the two, spread over its logarithm."""
    return max(low, min(high, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "store", "decode", "decode", "verify", "chunk", "prompts"])
    more = dict(index64=rng.random() < 0.3)
    if kind == "norm":
        width = rng.choice([_log(rng, 64, 16384), 128 * _log(rng, 1, 128), 2048, 4096, 8192])
        rows = _log(rng, 1, min(65536, 8192 * 8192 // width))
        out8 = rng.random() < 0.5
        return _norm(rows, width, fp32=rng.random() < 0.25, residual=rng.random() < 0.75, out8=out8,
                     group=128 if out8 and rng.random() < 0.5 else 0)
    heads, kv_heads = rng.choice([(16, 16), (8, 8), (32, 8), (64, 8), (16, 4), (24, 8), (32, 2), (40, 8), (64, 4), (7, 1)])
    dim, page, fp8 = rng.choice([64, 128, 128]), rng.choice([1, 16, 16, 64, 100, 128]), rng.random() < 0.4
    if kind == "store":
        return _store(_log(rng, 1, 16384), kv_heads, dim, page, fp8=fp8, fused=rng.random() < 0.5,
                      padding=rng.choice([0, 0, 7]), **more)
    more.update(fp8=fp8, lens_seed=rng.randrange(1 << 20), fused=rng.random() < 0.3,
                window=_log(rng, 16, 4096) if rng.random() < 0.25 else 0, cap=rng.choice([0.0, 0.0, 0.0, 20.0, 50.0]))
    if kind in ("decode", "verify"):
        n = _log(rng, 1, 256)
        steps = 1 if kind == "decode" else rng.randint(2, 8)
        high = _log(rng, 16, min(65536, (3 << 28) // (n * kv_heads * dim) - steps))
        return _attention(n, steps, steps, rng.choice([0, high // 2, high]), high, heads, kv_heads, dim, page, **more)
    if kind == "chunk":  # new tokens over cached prefixes
        n = _log(rng, 1, 16)
        q = _log(rng, 9, 2048 // n)
        kv = _log(rng, 64, min(32768, (1 << 30) // (n * max(heads, 16) * q) - q))
        return _attention(n, rng.randint(1, q), q, rng.randint(0, kv), kv, heads, kv_heads, dim, page, **more)
    n = _log(rng, 1, 16)  # prompts from their start
    q = _log(rng, 64, int(((1 << 30) // (n * heads)) ** 0.5))
    return _attention(n, rng.randint(1, q), q, 0, 0, heads, kv_heads, dim, page, **more)


def _lengths(case):
    """New tokens and keys (the new ones among them) of each request."""
    rng = random.Random(case["lens_seed"])
    new = [rng.randint(case["q_low"], case["q_high"]) for _ in range(case["requests"])]
    return new, [n + rng.randint(case["kv_low"], case["kv_high"]) for n in new]


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=DEV)

    state = dict(case=case)
    if case["op"] == "norm":
        dtype = torch.float32 if case["fp32"] else torch.bfloat16
        state["x"] = randn(case["rows"], case["width"]).to(dtype)
        if case["residual"]:
            state["residual"] = (randn(case["rows"], case["width"]) * 3.0).to(dtype)
        state["weight"] = (1.0 + 0.2 * randn(case["width"])).to(dtype)
        return state
    KH, D, page = case["kv_heads"], case["dim"], case["page"]
    index = torch.int64 if case["index64"] else torch.int32
    dtype = torch.bfloat16
    state["k_scale"] = state["v_scale"] = None
    if case["fp8"]:  # a scale per key head, from the range that its keys or values have
        state["k_scale"] = 0.01 + 0.005 * torch.rand(KH, generator=gen, device=DEV)
        state["v_scale"] = 0.01 + 0.005 * torch.rand(KH, generator=gen, device=DEV)

    def cache(pages, scale):
        if scale is None:
            return randn(pages, page, KH, D).to(dtype)
        return (randn(pages, page, KH, D) / scale[:, None]).clamp(-FP8_MAX, FP8_MAX).to(FP8)

    if case["op"] == "store":
        T, pages = case["tokens"], case["pages"]
        if case["fused"]:  # q, k, v of one projection, two query heads a key head
            qkv = randn(1, T, 4 * KH, D).to(dtype)
            state["k"], state["v"] = qkv[:, :, 2 * KH:3 * KH], qkv[:, :, 3 * KH:]
        else:
            state["k"], state["v"] = randn(1, T, KH, D).to(dtype), randn(1, T, KH, D).to(dtype)
        state["k_cache"], state["v_cache"] = cache(pages, state["k_scale"]), cache(pages, state["v_scale"])
        slots = torch.randperm(pages * page, generator=gen, device=DEV)[:T]
        if case["padding"]:
            slots[case["padding"] - 1::case["padding"]] = -1
        state["slots"] = slots.to(index)
        return state
    new, keys = _lengths(case)
    T, H = sum(new), case["heads"]
    width = max(1, max(-(-n // page) for n in keys))
    used = [-(-n // page) for n in keys]
    pages = sum(used) + 2
    if case["fused"]:
        state["q"] = randn(1, T, H + 2 * KH, D).to(dtype)[:, :, :H]
    else:
        state["q"] = randn(1, T, H, D).to(dtype)
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


def _run_own(state):
    case = state["case"]
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "01-glm53-ascend_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from sgl_glm53_ascend_ops import ops

    if case["op"] == "norm":
        more = dict(residual=state["residual"]) if case["residual"] else {}
        if case["out8"]:
            out, scale = ops.add_rms_norm_fp8(state["x"], state["weight"], EPS, group_size=case["group"], **more)
            return {"out": out, "scale": scale, **more}
        return {"out": ops.add_rms_norm(state["x"], state["weight"], EPS, **more), **more}
    if case["op"] == "store":
        ops.paged_kv_store(state["k"], state["v"], k_cache=state["k_cache"], v_cache=state["v_cache"],
                           slot_indices=state["slots"], k_scale=state["k_scale"], v_scale=state["v_scale"])
        return {"k_cache": state["k_cache"], "v_cache": state["v_cache"]}
    return {"out": ops.paged_attention(
        state["q"], k_cache=state["k_cache"], v_cache=state["v_cache"], page_table=state["page_table"],
        kv_lens=state["kv_lens"], cu_seqlens=state["cu_seqlens"], scale=state["scale"],
        max_query_len=state["max_query_len"], window=case["window"], logit_cap=case["cap"],
        k_scale=state["k_scale"], v_scale=state["v_scale"])}


def _norm_plain(state):
    case, result = state["case"], {}
    h = state["x"].float()
    if case["residual"]:
        h = h + state["residual"].float()
        state["residual"].copy_(h)
        result["residual"] = state["residual"]
    y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS) * state["weight"].float()
    if not case["out8"]:
        return {"out": y.to(state["x"].dtype), **result}
    rows, width = y.shape
    group = case["group"] or width
    groups = -(-width // group)
    padded = torch.zeros(rows, groups * group, device=DEV)
    padded[:, :width] = y
    padded = padded.view(rows, groups, group)
    scale = (padded.abs().amax(-1) / FP8_MAX).clamp_min(MIN_SCALE)
    out = (padded / scale[:, :, None]).view(rows, groups * group)[:, :width]
    return {"out": out.to(FP8), "scale": scale, **result}


def _store_plain(state):
    slots, page = state["slots"].long(), state["case"]["page"]
    pages = state["k_cache"].shape[0]
    valid = (slots >= 0) & (slots < pages * page)
    at = slots[valid]
    for x, cache, scale in ((state["k"], state["k_cache"], state["k_scale"]), (state["v"], state["v_cache"], state["v_scale"])):
        rows = x[0, valid]
        if scale is None:
            cache[at // page, at % page] = rows
        else:
            rows = (rows.float() / scale[:, None]).clamp(-FP8_MAX, FP8_MAX).to(FP8)
            cache.view(torch.uint8)[at // page, at % page] = rows.view(torch.uint8)
    return {"k_cache": state["k_cache"], "v_cache": state["v_cache"]}


def _attention_plain(state):
    """All requests at once, padded to the longest: scores, masked softmax and product in 32 bits."""
    case, q = state["case"], state["q"][0]
    table, lens, cu = state["page_table"].long(), state["kv_lens"].long(), state["cu_seqlens"].long()
    T, H, D = q.shape
    KH, page, N, Q = case["kv_heads"], case["page"], case["requests"], state["max_query_len"]
    G, L = H // KH, table.shape[1] * page
    t = torch.arange(Q, device=DEV)
    key = torch.arange(L, device=DEV)
    new = cu[1:] - cu[:-1]
    rows = torch.minimum(cu[:-1, None] + t[None, :], cu[1:, None] - 1)  # [N, Q]

    def gathered(cache, scale):
        flat = cache[table].view(N, L, KH, D).float()
        return flat if scale is None else flat.mul_(scale[:, None])

    k = gathered(state["k_cache"], state["k_scale"]).permute(0, 2, 3, 1).contiguous()  # [N, KH, D, L]
    x = q[rows].float().view(N, Q, KH, G, D).permute(0, 2, 1, 3, 4).reshape(N, KH, Q * G, D)
    s = torch.matmul(x, k).mul_(state["scale"])
    del k
    if case["cap"]:
        s = s.div_(case["cap"]).tanh_().mul_(case["cap"])
    at = (lens - new)[:, None] + t[None, :]  # position of each new token
    seen = (key[None, None, :] <= at[:, :, None]) & (key[None, None, :] < lens[:, None, None])
    if case["window"]:
        seen &= key[None, None, :] > at[:, :, None] - case["window"]
    s = s.view(N, KH, Q, G, L).masked_fill_(~seen[:, None, :, None, :], float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(top == float("-inf"), 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    v = gathered(state["v_cache"], state["v_scale"]).permute(0, 2, 1, 3).contiguous()
    o = torch.matmul(p.view(N, KH, Q * G, L), v).view(N, KH, Q, G, D)
    o = torch.where(total > 0, o / total, 0.0).permute(0, 2, 1, 3, 4).reshape(N, Q, H, D)
    token = torch.arange(T, device=DEV)
    request = (token[:, None] >= cu[None, 1:]).sum(1)
    return {"out": o[request, token - cu[request]].to(q.dtype)[None]}


def run(state):
    if own:
        return _run_own(state)
    return {"norm": _norm_plain, "store": _store_plain, "attention": _attention_plain}[state["case"]["op"]](state)


def _visible(case):
    """Keys that a request's new tokens see together, and (token, key) pairs, of each request."""
    union, pairs = [], []
    for m, n in zip(*_lengths(case)):
        w = case["window"] or n
        low = max(0, n - m - w + 1)
        union.append(n - low)
        # token at position p sees min(p + 1, w) keys
        a, b = n - m + 1, n
        full = max(0, b - max(a, w) + 1)
        ramp = (b - a + 1) - full
        pairs.append(full * w + ramp * a + ramp * (ramp - 1) // 2)
    return union, pairs


def work(case):
    if case["op"] == "norm":
        n, x = case["rows"] * case["width"], 4 if case["fp32"] else 2
        groups = -(-case["width"] // (case["group"] or case["width"])) if case["out8"] else 0
        size = n * (x + (2 * x if case["residual"] else 0) + (1 if case["out8"] else x)) + case["width"] * x
        return {"bytes": size + case["rows"] * groups * 4, "flops": n * (5 if case["residual"] else 4)}
    KH, D = case["kv_heads"], case["dim"]
    x, i = 1 if case["fp8"] else 2, 8 if case["index64"] else 4
    if case["op"] == "store":
        T = case["tokens"]
        kept = T - (T // case["padding"] if case["padding"] else 0)
        return {"bytes": kept * KH * D * 2 * (2 + x) + T * i, "flops": kept * KH * D * 2}
    new, _ = _lengths(case)
    union, pairs = _visible(case)
    T, N = sum(new), case["requests"]
    size = T * case["heads"] * D * 4 + sum(union) * KH * D * 2 * x + sum(-(-n // case["page"]) for n in union) * i
    return {"bytes": size + (2 * N + 1) * i, "flops": 4 * D * case["heads"] * sum(pairs)}


def exact(case, seed):
    """The definitions in 64 bits: an 8-bit output's value before its own rounding, attention request by request."""
    state = prepare(case, seed)
    f = torch.float64
    if case["op"] == "norm":
        x = state["x"].to(f)
        result = {}
        if case["residual"]:
            x += state["residual"].to(f)
            result["residual"] = x
        root = ((x ** 2).sum(1) / case["width"] + EPS).sqrt()
        y = x / root[:, None] * state["weight"].to(f)
        if not case["out8"]:
            return {"out": y, **result}
        out, scales = torch.empty_like(y), []
        step = case["group"] or case["width"]
        for c in range(0, case["width"], step):
            scales.append((y[:, c:c + step].abs().max(1).values / FP8_MAX).clamp(min=MIN_SCALE))
            out[:, c:c + step] = y[:, c:c + step] / scales[-1][:, None]
        return {"out": out, "scale": torch.stack(scales, 1), **result}
    if case["op"] == "store":
        result = {}
        slots = state["slots"].tolist()
        token = torch.tensor([t for t, s in enumerate(slots) if s >= 0], device=DEV)
        slot = torch.tensor([s for s in slots if s >= 0], device=DEV)
        for name in ("k", "v"):
            cache = state[name + "_cache"].to(f)
            x = state[name][0].to(f)
            if case["fp8"]:
                x = (x / state[name + "_scale"].to(f)[None, :, None]).clip(-FP8_MAX, FP8_MAX)
            cache.view(-1, case["kv_heads"], case["dim"])[slot] = x[token]
            result[name + "_cache"] = cache
        return result
    new, keys = _lengths(case)
    H, KH, D, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    out = torch.zeros(state["q"].shape, dtype=f, device=DEV)
    start = 0
    for n, (m, length) in enumerate(zip(new, keys)):
        low = max(0, length - m - case["window"] + 1) if case["window"] else 0
        j = torch.arange(low, length, device=DEV)
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
                z = (q.reshape(-1, D) @ k).view(t1 - t0, -1, length - low) * state["scale"]
                if case["cap"]:
                    z = case["cap"] * torch.tanh(z / case["cap"])
                p = torch.arange(length - m + t0, length - m + t1, device=DEV)[:, None, None]
                hidden = j > p
                if case["window"]:
                    hidden = hidden | (j <= p - case["window"])
                z = torch.softmax(z.masked_fill(hidden, float("-inf")), -1)
                out[0, start + t0:start + t1, heads] = (z.flatten(0, 1) @ v).view(t1 - t0, -1, D)
        start += m
    return {"out": out}
