"""A hybrid decoder served with this package: KDA layers and paged full attention side by side.

Every layer is: residual add and RMS norm in one call, projections, the mixer (KDA with its
slot-indexed states, or attention over the paged cache that ``paged_kv_store`` has just
written), a norm of the heads, the output projection. Prompts run as one ragged
prefill batch, then a decode step for all requests is captured in a HIP graph and
replayed token by token; only the contents of its input tensors change in between.

Weights are random: the example shows the calls and their bookkeeping.

    PYTHONPATH=01-glm53-ascend_amd python examples/hybrid_decoder.py [--fp8] [--tokens 32]

``--fp8`` keeps the cache in 8 bits and feeds the attention layers' first projection from
``add_rms_norm_fp8`` (8-bit weights, a scale per row and per output column).
"""

import argparse
import time
from dataclasses import dataclass

import torch

from sgl_glm53_ascend_ops import ops

EPS = 1e-6
FP8 = torch.float8_e4m3fn


@dataclass
class Config:
    width: int = 1024
    layers: str = "kkak"     # k: KDA, a: attention
    kda_heads: int = 4       # of 128
    heads: int = 8           # of the attention
    kv_heads: int = 2
    head_dim: int = 128
    vocab: int = 4096
    page_size: int = 64
    window: int = 0
    fp8: bool = False


@dataclass
class Step:
    """What one call of the model gets beside its tokens; all of it on the device."""

    cu_seqlens: torch.Tensor    # [N + 1] int32
    kv_lens: torch.Tensor       # [N] int32, the new tokens among them
    slots: torch.Tensor         # [T] int64: page * page_size + offset of each new token
    page_table: torch.Tensor    # [N, max_pages] int32
    state_slots: torch.Tensor   # [N] int32, > 0
    max_query_len: int


class Pages:
    """Pages and state slots of running requests, on the host."""

    def __init__(self, cfg, requests, max_len, device):
        self.cfg, self.device = cfg, device
        per = -(-max_len // cfg.page_size)
        self.table = torch.randperm(requests * per).view(requests, per).int()  # any page may be any request's
        self.lens = [0] * requests
        self.pages = requests * per

    def step(self, new):
        """The metadata of a call that adds ``new[n]`` tokens to request n."""
        size = self.cfg.page_size
        slots = []
        for n, m in enumerate(new):
            at = torch.arange(self.lens[n], self.lens[n] + m)
            slots.append(self.table[n].long()[at // size] * size + at % size)
            self.lens[n] += m
        on = lambda t, dtype: t.to(dtype).to(self.device)  # noqa: E731
        return Step(
            cu_seqlens=on(torch.tensor([0] + new).cumsum(0), torch.int32),
            kv_lens=on(torch.tensor(self.lens), torch.int32),
            slots=on(torch.cat(slots), torch.int64),
            page_table=on(self.table, torch.int32),
            state_slots=on(torch.arange(1, len(new) + 1), torch.int32),
            max_query_len=max(new),
        )


class HybridDecoder:
    def __init__(self, cfg, requests, pages, device="cuda", seed=0):
        self.cfg = cfg
        gen = torch.Generator(device=device).manual_seed(seed)

        def weight(*shape):
            return (torch.randn(*shape, device=device, generator=gen) * shape[0] ** -0.5).bfloat16()

        one = lambda n: torch.ones(n, device=device).bfloat16()  # noqa: E731
        self.embedding = torch.randn(cfg.vocab, cfg.width, device=device, generator=gen).bfloat16()
        self.head = weight(cfg.width, cfg.vocab)
        self.last_norm = one(cfg.width)
        self.layers = []
        for kind in cfg.layers:
            layer = {"kind": kind, "norm": one(cfg.width)}
            if kind == "k":
                H, K = cfg.kda_heads, 128
                layer.update(
                    first=weight(cfg.width, 4 * H * K + H), last=weight(H * K, cfg.width), head_norm=one(K),
                    A_log=torch.rand(H, device=device, generator=gen), dt_bias=torch.zeros(H * K, device=device),
                    # slot 0 is the padding row; K contiguous
                    state=torch.zeros(requests + 1, H, 128, K, device=device).transpose(2, 3),
                )
            else:
                H, KH, D = cfg.heads, cfg.kv_heads, cfg.head_dim
                cache = (pages, cfg.page_size, KH, D)
                dtype = FP8 if cfg.fp8 else torch.bfloat16
                first = weight(cfg.width, (H + 2 * KH) * D)
                layer.update(
                    first=first, last=weight(H * D, cfg.width), head_norm=one(D),
                    k_cache=torch.zeros(cache, device=device).to(dtype), v_cache=torch.zeros(cache, device=device).to(dtype),
                    scales={},
                )
                if cfg.fp8:
                    top = first.float().abs().amax(0, keepdim=True) / 448
                    layer["first8"] = (first.float() / top).t().contiguous().to(FP8)  # [N, K]
                    layer["first_scale"] = top
                    layer["scales"] = {s: torch.full((KH,), 0.05, device=device) for s in ("k_scale", "v_scale")}
            self.layers.append(layer)

    def kda(self, layer, x, residual, step):
        cfg, T = self.cfg, x.shape[0]
        H, K = cfg.kda_heads, 128
        y = ops.add_rms_norm(x, layer["norm"], EPS, residual=residual) @ layer["first"]
        q, k, v, a = (y[:, i * H * K:(i + 1) * H * K].contiguous().view(1, T, H, K) for i in range(4))
        args = dict(
            A_log=layer["A_log"], a=a, dt_bias=layer["dt_bias"], q=q, k=k, v=v, b=y[:, 4 * H * K:].contiguous().view(1, T, H),
            initial_state_source=layer["state"], initial_state_indices=step.state_slots,
            cu_seqlens=step.cu_seqlens, lower_bound=-5.0, scale=K ** -0.5,
        )
        if step.max_query_len > 1:
            out = ops.kda_varlen_chunk(prefill=True, **args)
        else:
            out = ops.kda_varlen_recurrent(**args)
        return ops.add_rms_norm(out, layer["head_norm"], EPS).reshape(T, H * K) @ layer["last"]

    def attention(self, layer, x, residual, step):
        cfg, T = self.cfg, x.shape[0]
        H, KH, D = cfg.heads, cfg.kv_heads, cfg.head_dim
        if cfg.fp8:
            x8, scale = ops.add_rms_norm_fp8(x, layer["norm"], EPS, residual=residual)
            qkv = torch._scaled_mm(x8, layer["first8"].t(), scale_a=scale, scale_b=layer["first_scale"],
                                   out_dtype=torch.bfloat16)
        else:
            qkv = ops.add_rms_norm(x, layer["norm"], EPS, residual=residual) @ layer["first"]
        qkv = qkv.view(1, T, H + 2 * KH, D)
        q, k, v = qkv[:, :, :H], qkv[:, :, H:H + KH], qkv[:, :, H + KH:]
        k = ops.add_rms_norm(k, layer["head_norm"], EPS)  # slices as they are
        q = ops.add_rms_norm(q, layer["head_norm"], EPS)
        ops.paged_kv_store(k, v, k_cache=layer["k_cache"], v_cache=layer["v_cache"], slot_indices=step.slots,
                           **layer["scales"])
        out = ops.paged_attention(
            q, k_cache=layer["k_cache"], v_cache=layer["v_cache"], page_table=step.page_table, kv_lens=step.kv_lens,
            cu_seqlens=step.cu_seqlens, scale=D ** -0.5, max_query_len=step.max_query_len, window=cfg.window,
            **layer["scales"],
        )
        return out.reshape(T, H * D) @ layer["last"]

    def hidden(self, tokens, step):
        """The normed hidden states of the new tokens ``[T, width]``."""
        x = self.embedding[tokens]
        residual = torch.zeros_like(x, dtype=torch.float32)  # the sum of all layers, in 32 bits
        for layer in self.layers:
            x = (self.kda if layer["kind"] == "k" else self.attention)(layer, x, residual, step)
        return ops.add_rms_norm(x, self.last_norm, EPS, residual=residual)

    def next_tokens(self, tokens, step):
        """The likeliest next token of every request."""
        last = self.hidden(tokens, step)[step.cu_seqlens[1:].long() - 1]
        return (last @ self.head).argmax(-1)


class DecodeGraph:
    """One decode step for all requests, captured; ``replay`` feeds it and returns the next tokens."""

    def __init__(self, model, tokens, step):
        self.step = step
        self.tokens = tokens.clone()
        saved = [{k: t.clone() for k, t in layer.items() if k in ("state", "k_cache", "v_cache")} for layer in model.layers]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            model.next_tokens(self.tokens, step)  # warms up the libraries; its writes are taken back below
        torch.cuda.current_stream().wait_stream(side)
        for layer, old in zip(model.layers, saved):
            for k, t in old.items():
                layer[k].copy_(t)
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph):
            self.next = model.next_tokens(self.tokens, step)

    def replay(self, tokens, step):
        self.tokens.copy_(tokens)
        self.step.kv_lens.copy_(step.kv_lens)
        self.step.slots.copy_(step.slots)
        self.graph.replay()
        return self.next.clone()


def generate(cfg, prompts, new_tokens, device="cuda"):
    """Greedy continuations ``[requests, new_tokens]`` of token lists, and seconds a decode step."""
    pages = Pages(cfg, len(prompts), max(map(len, prompts)) + new_tokens, device)
    model = HybridDecoder(cfg, len(prompts), pages.pages, device)
    tokens = torch.tensor([t for p in prompts for t in p], device=device)
    out = [model.next_tokens(tokens, pages.step([len(p) for p in prompts]))]
    graph = None
    for i in range(new_tokens - 1):
        step = pages.step([1] * len(prompts))
        if graph is None:
            graph = DecodeGraph(model, out[-1], step)
            torch.cuda.synchronize()
            begin = time.perf_counter()
        out.append(graph.replay(out[-1], step))
    torch.cuda.synchronize()
    seconds = (time.perf_counter() - begin) / (new_tokens - 1) if graph is not None else float("nan")
    return torch.stack(out, 1), seconds


def main():
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--fp8", action="store_true")
    parser.add_argument("--window", type=int, default=0)
    parser.add_argument("--requests", type=int, default=16)
    parser.add_argument("--tokens", type=int, default=32, help="new tokens of each request")
    args = parser.parse_args()
    torch.manual_seed(0)
    cfg = Config(fp8=args.fp8, window=args.window)
    prompts = [torch.randint(cfg.vocab, (int(n),)).tolist() for n in torch.randint(1, 700, (args.requests,))]
    out, seconds = generate(cfg, prompts, args.tokens)
    print(f"{args.requests} requests, prompts of {min(map(len, prompts))} to {max(map(len, prompts))} tokens")
    print(f"first request continues {out[0].tolist()}")
    print(f"{seconds * 1e6:.0f} us a decode step")


if __name__ == "__main__":
    main()
