"""Linear attention in 64 bits, token by token, with bounds on what a kernel may differ by.

The same recurrence on absolute values gives, for every output and state element, the sum A of its terms'
sizes. Bounds relative to A:

* states: a term's decays and products are fp32. A decay's exponent of up to 87 is rounded to fp32 (2^-24 of
  it): 6e-6 in its exponential, 1e-6 for the exponential itself, and the sums over n tokens add 2^-24 for each
  token: 1e-5 + n 2^-24. Token by token a state is rounded three times a token (decay, product, sum)
  and each decay's exponential is within 2e-7: 1e-6 + n 4e-7.
* outputs: those of the state, D + 64 additions more (2^-24 each), in chunks scores and state in two bf16 parts (2^-17 each,
  with a second rounding 2^-16 together), and the output's own rounding, eps / 2 of the value and of what it
  is off by.
"""

import torch


class Linear:
    """Inputs of one call on the CPU, drawn from a seed; slot 0 of the pool is the padding row."""

    def __init__(self, seed, lens, heads, dim, gated=True, fp32=False, fused=False, index64=False, zero_slots=(),
                 before=0, after=0, track=None, g_mean=-2.0, g_spread=1.5):
        gen = torch.Generator().manual_seed(seed)
        self.lens, self.heads, self.dim, self.before = lens, heads, dim, before
        T, N = before + sum(lens) + after, len(lens)
        dtype = torch.float32 if fp32 else torch.bfloat16
        index = torch.int64 if index64 else torch.int32
        if fused:
            qkv = torch.randn(1, T, 3 * heads, dim, generator=gen).to(dtype)
            self.q, self.k, self.v = qkv[:, :, :heads], qkv[:, :, heads:2 * heads], qkv[:, :, 2 * heads:]
        else:
            self.q, self.k, self.v = (torch.randn(1, T, heads, dim, generator=gen).to(dtype) for _ in range(3))
        shape = (1, T, heads) if gated else (heads,)
        self.g = -torch.exp(torch.randn(*shape, generator=gen) * g_spread + g_mean)
        self.slots = 2 * N + 2
        self.pool = torch.randn(self.slots, heads, dim, dim, generator=gen).transpose(2, 3)
        order = torch.randperm(self.slots - 1, generator=gen) + 1
        at = order[:N].clone()
        for n in zero_slots:
            at[n] = 0
        self.indices = at.to(index)
        self.cu = (torch.tensor([0] + list(lens)).cumsum(0) + before).to(index)
        self.scale = dim ** -0.5
        self.track = None
        if track is not None:
            self.track = (order[N:2 * N].to(index), torch.tensor(track).to(index))

    def on(self, device):
        """The call's arguments on a device, strides kept."""
        def move(t):
            if t.dim() == 4 and not t.is_contiguous() and t is not self.pool:  # a slice of a fused projection
                whole = torch.empty(1, t.shape[1], 3 * self.heads, self.dim, dtype=t.dtype, device=device)
                part = whole[:, :, :self.heads]
                part.copy_(t)
                return part
            return t.to(device)

        args = dict(initial_state_source=self.pool.transpose(2, 3).contiguous().to(device).transpose(2, 3),
                    initial_state_indices=self.indices.to(device), cu_seqlens=self.cu.to(device), scale=self.scale)
        if self.track is not None:
            args.update(track_state_indices=self.track[0].to(device), track_state_lens=self.track[1].to(device))
        return (move(self.q), move(self.k), move(self.v), self.g.to(device)), args

    def exact(self, absolute=False, device="cpu"):
        """(out, pool, middle) in 64 bits; of the absolute values: the sums of the terms' sizes."""
        f = (lambda t: t.to(device).double().abs()) if absolute else (lambda t: t.to(device).double())
        q, k, v, pool = f(self.q[0]), f(self.k[0]), f(self.v[0]), f(self.pool)
        g = self.g.to(device).double().expand(1, self.q.shape[1], self.heads)[0]
        out = torch.zeros_like(q)
        longest = max(list(self.lens) + [1])
        middle = torch.zeros(len(self.lens), longest, self.heads, self.dim, self.dim, dtype=torch.float64, device=device)
        begin = pool.clone()
        t = self.before
        for n, m in enumerate(self.lens):
            slot = int(self.indices[n])
            S = begin[slot].clone() if slot > 0 else torch.zeros_like(begin[0])
            for i in range(m + 1):
                if self.track is not None and int(self.track[1][n]) == i:
                    pool[int(self.track[0][n])] = S
                if i == m:
                    break
                S = S * g[t].exp()[:, None, None] + k[t][:, :, None] * v[t][:, None, :]
                out[t] = (q[t][:, :, None] * S).sum(1) * self.scale
                middle[n, i] = S if slot > 0 else 0
                t += 1
            if slot > 0:
                pool[slot] = S
        return out, pool, middle


def bounds(case, chunk, device="cpu"):
    """Of (out, pool, middle), elementwise."""
    out, pool, middle = case.exact(absolute=True, device=device)
    n = max(list(case.lens) + [1])
    state = 1e-5 + n * 2.0 ** -24 if chunk else 1e-6 + n * 4e-7
    value = case.exact(device=device)[0].abs()
    half = 2.0 ** -8 if case.q.dtype == torch.bfloat16 else 2.0 ** -24
    off = out * (state + (case.dim + 64) * 2.0 ** -24 + (2.0 ** -16 if chunk else 0.0))
    return off + half * (value + off), pool * state, middle * state
