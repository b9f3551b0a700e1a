"""Paged attention over a window and the first tokens that stay visible, against the definition in 64 bits.

The bounds are those of ``decoder_cases`` for the same roundings.
"""

import random

import pytest
import torch

from tests import decoder_cases as C

pytestmark = pytest.mark.gpu

DEV = "cuda"
INF, NAN = float("inf"), float("nan")


@pytest.fixture(scope="module")
def ops(gpu_ops):
    from sgl_glm53_ascend_ops import ops

    return ops


class Sinks(C.Attention):
    """Inputs of one call with sinks."""

    def __init__(self, *args, sinks=0, **more):
        super().__init__(*args, **more)
        self.sinks = sinks

    def kwargs(self, dev, **over):
        return super().kwargs(dev, **{**dict(sink_tokens=self.sinks), **over})

    def seen(self, n):
        """[new tokens, keys] of request n."""
        pos = torch.arange(self.keys[n] - self.new[n], self.keys[n])[:, None]
        j = torch.arange(self.keys[n])[None, :]
        seen = j <= pos
        if self.window:
            seen &= (j > pos - self.window) | (j < self.sinks)
        return seen

    def exact(self):
        out = torch.zeros(self.q.shape, dtype=torch.float64)
        bound = torch.zeros_like(out)
        G = self.heads // self.kv_heads
        for n, m in enumerate(self.new):
            start = int(self.cu_seqlens[n])
            if m == 0 or self.keys[n] == 0:
                continue
            page, off = self.slots_of(n)
            real = (page >= 0)[:, None, None]
            k = torch.where(real, self.k_cache[page, off].double(), 0.0)
            v = torch.where(real, self.v_cache[page, off].double(), 0.0)
            if self.fp8:
                k, v = k * self.k_scale.double()[:, None], v * self.v_scale.double()[:, None]
            seen = self.seen(n)
            for h in range(self.heads):
                q, kh, vh = self.q[0, start:start + m, h].double(), k[:, h // G], v[:, h // G]
                s = q @ kh.t() * self.scale
                d = self.dim * 2.0 ** -24 * (q.abs() @ kh.t().abs()) * abs(self.scale) + 1e-5
                if self.cap:
                    s = self.cap * torch.tanh(s / self.cap)
                    d = d + 2e-6 * self.cap
                p = torch.where(seen.any(1, keepdim=True), torch.softmax(s.masked_fill(~seen, -INF), 1), 0.0)
                # a key that is not seen has no part in the sum, whatever its value
                o, A = torch.zeros(m, self.dim).double(), torch.zeros(m, self.dim).double()
                for i in range(m):
                    o[i], A[i] = p[i, seen[i]] @ vh[seen[i]], p[i, seen[i]] @ vh[seen[i]].abs()
                worst = torch.where(seen, d, 0.0).amax(1, keepdim=True)
                out[0, start:start + m, h] = o
                bound[0, start:start + m, h] = ((2.0 ** -8 + 2 * worst) * A + 2.0 ** -8 * o.abs()) * 1.01
        return out, bound


def check(ops, case, **over):
    out = ops.paged_attention(case.q.to(DEV), **case.kwargs(DEV, **over))
    assert out.shape == case.q.shape and out.dtype == torch.bfloat16
    want, bound = case.exact()
    C.assert_within(out, want, bound, "out")
    return out


@pytest.mark.parametrize("sinks", [1, 4, 31, 32, 33, 127, 128, 129, 300, 5000])
@pytest.mark.parametrize("window", [1, 40, 128, 129, 1000])
def test_decode(ops, sinks, window):
    """One new token each; contexts below the sinks, between sinks and window, and far beyond both."""
    keys = [1, 2, 5, 33, 128, 129, 0, 300, 431, 1500]
    check(ops, Sinks(sinks, [1] * len(keys), keys, 4, 2, 64, 16, window=window, sinks=sinks))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("heads,kv_heads", [(4, 4), (7, 1), (24, 1), (32, 1)])
def test_decode_heads(ops, dim, fp8, heads, kv_heads):
    keys = [700, 3, 260, 1200]
    check(ops, Sinks(dim, [1, 1, 2, 1], keys, heads, kv_heads, dim, 16, fp8=fp8, window=130, sinks=6))


@pytest.mark.parametrize("page", [1, 5, 16, 64])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("sinks", [4, 700])
def test_one_long_request(ops, page, fp8, sinks):
    """A request's keys over many workgroups, joined; the first parts are the sinks'."""
    check(ops, Sinks(page, [1], [9001], 8, 2, 128, page, fp8=fp8, index64=True, window=3001, sinks=sinks))


@pytest.mark.parametrize("sinks", [1, 4, 63, 64, 65, 100, 128, 5000])
@pytest.mark.parametrize("window", [1, 50, 64, 200])
def test_prefill(ops, sinks, window):
    """Prompts and chunks; tiles whose window begins before, in and behind the sinks' tiles."""
    new = [130, 0, 64, 1, 33]
    before = [0, 5, 64, 1000, 90]
    check(ops, Sinks(sinks + window, new, [a + b for a, b in zip(new, before)], 4, 2, 64, 16, window=window, sinks=sinks))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("page", [16, 24, 5, 128])
def test_prefill_layouts(ops, dim, fp8, page):
    check(ops, Sinks(page, [200, 40], [900, 300], 9, 3, dim, page, fp8=fp8, window=100, sinks=20, index64=fp8, before=2, after=3))


@pytest.mark.parametrize("new", [5, 100])
@pytest.mark.parametrize("sinks", [3, 400])
def test_few_tiles_over_many_keys(ops, new, sinks):
    """Few rows over a long window: the walk over sinks and window split and joined."""
    check(ops, Sinks(new, [new], [new + 4000], 8, 1, 128, 16, window=2500, sinks=sinks))


@pytest.mark.parametrize("cap", [0.5, 20.0])
@pytest.mark.parametrize("new", [[1, 1], [90, 20]])
def test_cap(ops, cap, new):
    check(ops, Sinks(3, new, [400, 150], 8, 2, 128, 16, cap=cap, spread=20.0, window=60, sinks=5))


@pytest.mark.parametrize("hint", [0, 1, 3, 1000])
def test_holds_for_any_hint(ops, hint):
    check(ops, Sinks(11, [40, 1, 3], [240, 500, 90], 4, 2, 64, 16, window=70, sinks=9), max_query_len=hint)


@pytest.mark.parametrize("new", [[1, 3, 1], [100, 3, 40]])
def test_sinks_that_add_nothing(ops, new):
    """No sinks, no window, or a window that reaches back to the start: bit by bit the call without."""
    keys = [n + 200 for n in new]
    case = Sinks(12, new, keys, 4, 2, 128, 16)
    plain = case.kwargs(DEV)
    del plain["sink_tokens"]
    q = case.q.to(DEV)
    want = ops.paged_attention(q, **plain)
    assert torch.equal(ops.paged_attention(q, **{**plain, "sink_tokens": 7}), want)
    want = ops.paged_attention(q, **{**plain, "window": 50})
    assert torch.equal(ops.paged_attention(q, **{**plain, "window": 50, "sink_tokens": 0}), want)
    out = check(ops, case, window=100000, sink_tokens=8)
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("hint", [1, 100])
@pytest.mark.parametrize("page", [16, 5, 64])
@pytest.mark.parametrize("how", ["outside", "nan"])
def test_pages_between_sinks_and_window_are_free(ops, hint, page, how):
    """What lies between the sinks' page and the window's may be anybody's: its entries point outside the pool, or to a page of NaN."""
    case = Sinks(13, [1, 2, 1], [1200, 700, 300], 4, 2, 64, page, window=100, sinks=7)
    want, bound = case.exact()
    for n, length in enumerate(case.keys):
        first, last = -(-case.sinks // page), (length - case.new[n] - case.window) // page
        if last > first:
            case.page_table[n, first:last] = 1 << 20 if how == "outside" else case.unused[0]
    case.k_cache[case.unused[0]] = NAN
    case.v_cache[case.unused[0]] = NAN
    out = ops.paged_attention(case.q.to(DEV), **case.kwargs(DEV, max_query_len=hint))
    C.assert_within(out, want, bound, "out")


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("new,hint", [([1, 3], 3), ([60, 20], 60), ([1], 100)])
def test_hidden_keys_cannot_reach_a_row(ops, fp8, new, hint):
    """Infinite and NaN keys and values that a row does not see, some of them in the tiles it reads; those it sees do."""
    keys = [n + 500 for n in new]
    for sinks, window in ((5, 90), (70, 33), (130, 200)):
        case = Sinks(sinks, new, keys, 4, 2, 64, 16, fp8=fp8, window=window, sinks=sinks)
        n = 0
        first, last = case.keys[n] - case.new[n], case.keys[n] - 1
        hidden = torch.ones(case.keys[n], dtype=torch.bool)
        hidden[case.seen(n).any(0)] = False  # by every row
        some = case.seen(n).any(0) & ~case.seen(n).all(0)
        page, off = case.slots_of(n)
        bad = torch.tensor(NAN).to(case.k_cache.dtype)
        for j in hidden.nonzero()[:, 0].tolist():
            case.k_cache.view(torch.uint8 if fp8 else torch.int16)[page[j], off[j]] = bad.view(torch.uint8 if fp8 else torch.int16)
            case.v_cache.view(torch.uint8 if fp8 else torch.int16)[page[j], off[j]] = bad.view(torch.uint8 if fp8 else torch.int16)
        check(ops, case, max_query_len=hint)
        if some.any():  # a value that some rows see and others do not
            j = int(some.nonzero()[0])
            case.v_cache.view(torch.uint8 if fp8 else torch.int16)[page[j], off[j], 0, 3] = bad.view(torch.uint8 if fp8 else torch.int16)
            check(ops, case, max_query_len=hint)
        case.v_cache.view(torch.uint8 if fp8 else torch.int16)[page[0], off[0], 1, 7] = bad.view(torch.uint8 if fp8 else torch.int16)
        out = check(ops, case, max_query_len=hint)  # the first sink: every row sees it
        start = int(case.cu_seqlens[n])
        assert torch.isnan(out[0, start:start + case.new[n], 2:, 7]).all()
        assert torch.isfinite(out[0, start:start + case.new[n], 2:, 8]).all()
        assert first <= last


@pytest.mark.parametrize("seed", range(40))
def test_random(ops, seed):
    rng = random.Random(1000 + seed)
    kv_heads, group = rng.choice([(1, 1), (2, 4), (3, 3), (2, 8), (1, 16), (1, 33), (1, 5)])
    n = rng.randint(1, 5)
    new = C.lengths(rng, n, rng.choice([1, 3, 9, 70]))
    keys = [max(0, m + rng.choice([0, 1, 17, rng.randint(0, 900), -rng.randint(0, 2)])) for m in new]
    check(ops, Sinks(seed, new, keys, kv_heads * group, kv_heads, rng.choice([64, 128]), rng.choice([1, 3, 16, 48, 64]),
                     fp8=rng.random() < 0.4, index64=rng.random() < 0.4, window=rng.choice([1, 5, 64, 130, 400]),
                     sinks=rng.choice([1, 4, 16, 64, 65, 200]), cap=rng.choice([0.0, 0.0, 5.0]),
                     before=rng.choice([0, 2]), after=rng.choice([0, 3]), spread=rng.choice([1.0, 4.0])))


@pytest.mark.parametrize("new", [[1, 1, 1], [70, 1, 33]])
def test_graph_replay(ops, new):
    """A replayed graph follows lengths, pages and queries as they change."""
    cases = [Sinks(s, new, [n + 300 + 50 * s for n in new], 4, 2, 128, 16, window=100, sinks=4, extra_pages=40 - 9 * s) for s in range(3)]
    pages = max(c.k_cache.shape[0] for c in cases)
    width = max(c.page_table.shape[1] for c in cases)

    def inputs(c):
        q, kw = c.q.to(DEV), c.kwargs(DEV)
        for name in ("k_cache", "v_cache"):
            whole = torch.zeros(pages, *kw[name].shape[1:], dtype=kw[name].dtype, device=DEV)
            whole[:kw[name].shape[0]] = kw[name]
            kw[name] = whole
        table = torch.zeros(len(new), width, dtype=torch.int32, device=DEV)
        table[:, :kw["page_table"].shape[1]] = kw["page_table"]
        kw["page_table"] = table
        return q, kw

    q, kw = inputs(cases[0])
    ops.paged_attention(q, **kw)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.paged_attention(q, **kw)
    for c in cases + cases[:1]:
        q2, kw2 = inputs(c)
        q.copy_(q2)
        for name in ("k_cache", "v_cache", "page_table", "kv_lens"):
            kw[name].copy_(kw2[name])
        graph.replay()
        want = ops.paged_attention(q2, **kw2)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        exact, bound = c.exact()
        C.assert_within(out, exact, bound, "out")
