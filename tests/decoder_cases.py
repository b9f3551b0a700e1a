"""Plain 64-bit forms of the decoder operators, with bounds on what a kernel may differ by.

Every bound follows from the roundings that the operators are documented to make:

* norms: fp32 arithmetic, then one rounding to the output type. The sum of squares
  adds positive terms, at most 32 in a thread one after another and then a tree:
  its relative error is below 48 * 2^-24, halved by the square root; a few
  roundings more give 4e-6 for everything before the last rounding.
* attention, per output element, with A = sum_j p_j |v_j|: weights rounded to bf16
  (2^-8 A), the output's own rounding (2^-8 |out|), and an error d of a score moves
  its weight by the factor e^d: 2 d A for numerator and denominator, where d is at most
  the fp32 accumulation error D 2^-24 sum |q k| scale, 2e-6 of the cap, and 1e-5 for
  exponentials, sums and the running maximum's factors.
"""

import random

import torch

FP8 = torch.float8_e4m3fn


def norm_exact(x, weight, eps, residual=None):
    """(h, y) in 64 bits."""
    h = x.double()
    if residual is not None:
        h = h + residual.double()
    y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + eps) * weight.double()
    return h, y


def norm_scales(y, group):
    """max|y| / 448 of every group, at least 1e-12, and the same spread over the columns."""
    width = y.shape[-1]
    group = group or width
    scales = torch.stack([(y[..., c:c + group].abs().amax(-1) / 448).clamp_min(1e-12)
                          for c in range(0, width, group)], -1)
    return scales, scales.repeat_interleave(group, -1)[..., :width]


def assert_within(got, want, bound, what):
    """|got - want| <= bound elementwise (64 bits, on want's device); NaN and infinities where want has them."""
    got, bound = got.double().to(want.device), bound.to(want.device)
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN elsewhere"
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), f"{what}: infinities"
    off = ((got - want).abs() - bound)[fine]
    assert off.numel() == 0 or off.max() <= 0, f"{what}: over its bound by {off.max():.3g}"


class Attention:
    """Inputs of one ``paged_attention`` call on the CPU, drawn from a seed."""

    def __init__(self, seed, new, keys, heads, kv_heads, dim, page, fp8=False, index64=False, extra_pages=3,
                 window=0, cap=0.0, before=0, after=0, spread=1.0):
        gen = torch.Generator().manual_seed(seed)
        self.new, self.keys, self.heads, self.kv_heads, self.dim, self.page = new, keys, heads, kv_heads, dim, page
        self.window, self.cap, self.fp8 = window, cap, fp8
        self.scale = dim ** -0.5
        T = before + sum(new) + after
        index = torch.int64 if index64 else torch.int32
        self.q = (torch.randn(1, T, heads, dim, generator=gen) * spread).bfloat16()
        used = [-(-k // page) for k in keys]
        pages = sum(used) + extra_pages
        self.k_scale = self.v_scale = None
        k = torch.randn(pages, page, kv_heads, dim, generator=gen)
        v = torch.randn(pages, page, kv_heads, dim, generator=gen)
        if fp8:
            self.k_scale = 0.015 + 0.01 * torch.rand(kv_heads, generator=gen)
            self.v_scale = 0.015 + 0.01 * torch.rand(kv_heads, generator=gen)
            k = (k / self.k_scale[:, None]).clamp(-448, 448).to(FP8)
            v = (v / self.v_scale[:, None]).clamp(-448, 448).to(FP8)
        else:
            k, v = k.bfloat16(), v.bfloat16()
        self.k_cache, self.v_cache = k, v
        order = torch.randperm(pages, generator=gen).tolist()
        width = max([1] + used)
        table = torch.zeros(len(new), width, dtype=index)
        at = 0
        for n, c in enumerate(used):
            table[n, :c] = torch.tensor(order[at:at + c], dtype=index)
            at += c
        self.unused = order[at:]
        self.page_table = table
        self.kv_lens = torch.tensor(keys, dtype=index)
        self.cu_seqlens = (before + torch.tensor([0] + new).cumsum(0)).to(index)
        self.max_query_len = max([0] + new)

    def slots_of(self, n):
        """(page, offset) of the request's keys; pages outside the pool are -1."""
        j = torch.arange(self.keys[n])
        p = self.page_table[n].long()[j // self.page]
        return torch.where((p >= 0) & (p < self.k_cache.shape[0]), p, -1), j % self.page

    def kwargs(self, dev, **over):
        move = lambda t: None if t is None else t.to(dev)  # noqa: E731
        a = dict(k_cache=move(self.k_cache), v_cache=move(self.v_cache), page_table=move(self.page_table),
                 kv_lens=move(self.kv_lens), cu_seqlens=move(self.cu_seqlens), scale=self.scale,
                 max_query_len=self.max_query_len, window=self.window, logit_cap=self.cap,
                 k_scale=move(self.k_scale), v_scale=move(self.v_scale))
        a.update(over)
        return a

    def exact(self):
        """(out, bound) in 64 bits; tokens of no request are 0 with bound 0."""
        out = torch.zeros(self.q.shape, dtype=torch.float64)
        bound = torch.zeros_like(out)
        G = self.heads // self.kv_heads
        for n, m in enumerate(self.new):
            L, start = self.keys[n], int(self.cu_seqlens[n])
            if m == 0 or L == 0:
                continue
            page, off = self.slots_of(n)
            real = (page >= 0)[:, None, None]
            k = torch.where(real, self.k_cache[page, off].double(), 0.0)  # [L, KH, D]
            v = torch.where(real, self.v_cache[page, off].double(), 0.0)
            if self.fp8:
                k, v = k * self.k_scale.double()[:, None], v * self.v_scale.double()[:, None]
            k, v = k.repeat_interleave(G, 1).permute(1, 2, 0), v.repeat_interleave(G, 1).permute(1, 0, 2)
            q = self.q[0, start:start + m].double().permute(1, 0, 2)  # [H, m, D]
            s = q @ k * self.scale
            d = self.dim * 2.0 ** -24 * (q.abs() @ k.abs()) * abs(self.scale) + 1e-5
            if self.cap:
                s = self.cap * torch.tanh(s / self.cap)
                d = d + 2e-6 * self.cap
            pos = torch.arange(L - m, L)[:, None]
            j = torch.arange(L)[None, :]
            seen = j <= pos
            if self.window:
                seen &= j > pos - self.window
            s = s.masked_fill(~seen, float("-inf"))
            top = s.amax(-1, keepdim=True)
            p = torch.exp(s - torch.where(top == float("-inf"), 0.0, top))
            total = p.sum(-1, keepdim=True)
            p = torch.where(total > 0, p / total, 0.0)
            o = p @ v
            A = p @ v.abs()
            worst = torch.where(seen, d, 0.0).amax(-1, keepdim=True)
            e = (2.0 ** -8 + 2 * worst) * A + 2.0 ** -8 * o.abs()
            out[0, start:start + m] = o.permute(1, 0, 2)
            bound[0, start:start + m] = e.permute(1, 0, 2) * 1.01
        return out, bound


def lengths(rng, n, most, empty=0.2):
    return [0 if rng.random() < empty else rng.choice([1, 2, rng.randint(1, most), most]) for _ in range(n)]


def random_attention(seed):
    """Heads, lengths and layouts drawn over what the operator takes, sizes small enough for the CPU."""
    rng = random.Random(seed)
    kv_heads, group = rng.choice([(1, 1), (2, 1), (1, 7), (2, 4), (3, 3), (2, 8), (1, 16), (2, 20), (1, 33), (1, 5)])
    n = rng.randint(1, 6)
    new = lengths(rng, n, rng.choice([1, 3, 9, 70, 150]))
    keys = [max(0, m + rng.choice([0, 0, 1, 17, rng.randint(0, 700), -rng.randint(0, 2)])) for m in new]
    return Attention(seed, new, keys, kv_heads * group, kv_heads, rng.choice([64, 128]),
                     rng.choice([1, 3, 16, 48, 64, 100]), fp8=rng.random() < 0.4, index64=rng.random() < 0.4,
                     window=rng.choice([0, 0, 1, 5, 64, 130]), cap=rng.choice([0.0, 0.0, 5.0, 30.0]),
                     before=rng.choice([0, 0, 2]), after=rng.choice([0, 0, 3]), spread=rng.choice([1.0, 4.0]))
