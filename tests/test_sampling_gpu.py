"""Sampling against its definition in 64 bits, row by row.

Tokens have to be equal. The kernel rounds weights to multiples of 2^-44 of the largest or finer, and
the definition here sums in 64-bit floats, so a border could only be read differently where a sum falls within
about 1e-11 of it: none of these seeded cases does (``test_borders`` puts sums on borders exactly, with weights
that are whole). Log probabilities are rounded once to fp32, from logarithms of 64 bits whose mass is
within 1e-9: |p| 2^-24 + 1e-8.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")


@pytest.fixture(scope="module")
def ops(gpu_ops):
    from sgl_glm53_ascend_ops import ops

    return ops


def plain(x, u, t=1.0, k=0, p=1.0, floor=0.0):
    """(token, log probability) of one row of logits (a float tensor on the CPU)."""
    x = x.double()
    x = torch.where(torch.isnan(x), -INF, x)
    top = x.max()
    if top == -INF:
        return -1, -INF
    if not t > 0:
        return int((x == top).nonzero()[0]), 0.0
    if top == INF:
        x = torch.where(x == INF, 0.0, -INF).double()  # of two numbers it would be fp32
        top = x.max()
    w = torch.exp((x - top) / t)
    w[x == -INF] = 0.0
    order = torch.sort(x, descending=True, stable=True).indices
    if k > 0:
        order = order[:k]
    if p < 1:
        total = w[order].cumsum(0)
        before = total - w[order]
        most = max(1, int((before < p * total[-1]).sum()))
        order = order[:most]
    order = order[w[order] >= min(floor, 1.0)]
    order = order.sort().values
    mass = w[order].cumsum(0)
    at = min(int((mass <= max(u, 0.0) * mass[-1]).sum()), len(order) - 1)
    while w[order[at]] == 0:
        at -= 1
    return int(order[at]), math.log(float(w[order[at]] / mass[-1]))


def check(ops, logits, u, t=None, k=None, p=None, floor=None, index=torch.int32, view=None):
    dev = lambda x, dtype=torch.float32: None if x is None else torch.tensor(x, dtype=dtype).cuda()  # noqa: E731
    x = logits.cuda() if view is None else view(logits.cuda())
    tokens, logprobs = ops.sample_tokens(x, dev(u), temperature=dev(t), top_k=dev(k, index), top_p=dev(p), min_p=dev(floor))
    assert tokens.dtype == torch.int64 and logprobs.dtype == torch.float32
    f = lambda x, n, default: default if x is None else float(torch.tensor(x[n], dtype=torch.float32))  # noqa: E731
    for n in range(logits.shape[0]):
        token, logprob = plain(logits[n].float(), f(u, n, 0.0), f(t, n, 1.0), 0 if k is None else k[n], f(p, n, 1.0), f(floor, n, 0.0))
        assert int(tokens[n]) == token, (n, int(tokens[n]), token)
        if token >= 0:
            assert abs(float(logprobs[n]) - logprob) <= abs(logprob) * 2.0 ** -24 + 1e-8, (n, float(logprobs[n]), logprob)
        else:
            assert float(logprobs[n]) == -INF


def draw(seed, rows, vocab, dtype, spread=2.5):
    gen = torch.Generator().manual_seed(seed)
    logits = torch.randn(rows, vocab, generator=gen) * spread
    return logits.to(dtype), torch.rand(rows, generator=gen).tolist(), gen


VOCABS = [1, 2, 7, 64, 100, 511, 1000, 1024, 1025, 2048, 4097, 32001, 50000]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", VOCABS)
def test_temperatures(ops, vocab, dtype):
    logits, u, gen = draw(vocab, 6, vocab, dtype)
    check(ops, logits, u)
    check(ops, logits, u, t=[0.0, 0.3, 1.0, 3.0, 1e-3, 50.0])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [5, 1024, 1500, 8192, 32001])
def test_filters(ops, vocab, dtype):
    """Each filter alone and all together, from one element to all."""
    logits, u, gen = draw(vocab + 1, 8, vocab, dtype)
    k = [1, 2, 50, 512, 513, vocab // 2 + 1, vocab, 0]
    p = [0.0, 0.1, 0.5, 0.9, 0.99, 0.9999, 1.0, 0.7]
    floor = [0.0, 1e-6, 0.001, 0.05, 0.5, 1.0, 2.0, 0.01]
    t = [0.7, 1.0, 1.3, 0.5, 2.0, 1.0, 1.0, 5.0]
    check(ops, logits, u, k=k)
    check(ops, logits, u, k=k[::-1], index=torch.int64, t=t)
    check(ops, logits, u, p=p, t=t)
    check(ops, logits, u, p=p[::-1])
    check(ops, logits, u, floor=floor, t=t)
    check(ops, logits, u, t=t, k=k, p=p[::-1], floor=floor[::-1])
    check(ops, logits, u, t=t, k=k[::-1], p=p, floor=floor)
    check(ops, logits, u, p=[0.95] * 8, floor=[0.02] * 8)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [4000, 32001, 131072])
def test_top_k_where_lists_fill(ops, vocab, dtype):
    """Around the lengths at which candidates are sorted otherwise, or are not gathered at all."""
    logits, u, gen = draw(vocab + 2, 8, vocab, dtype)
    k = [190, 255, 256, 257, 319, 320, 321, 400]
    check(ops, logits, u, k=k)
    check(ops, logits, u, k=k[::-1], p=[0.9, 0.5, 0.99, 1.0, 0.7, 0.95, 0.2, 0.8], t=[0.5, 1.0, 2.0, 1.0, 3.0, 0.7, 1.0, 1.5])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_flat_rows_and_ties(ops, dtype):
    """Equal logits by the thousand: more than one list holds, cut by index; two values; steps."""
    V = 20000
    rows = torch.zeros(6, V)
    rows[1, ::3] = -1.0
    rows[2] = torch.arange(V) // 5000 * -0.5
    rows[3, 100:] = -2.0
    rows[4] = 7.25
    rows[5] = torch.arange(V).flip(0) // 100 * 0.0078125
    u = [0.1, 0.9, 0.5, 0.7, 0.999, 0.3]
    logits = rows.to(dtype)
    check(ops, logits, u)
    check(ops, logits, u, k=[9000, 5000, 12000, 150, 19999, 5000])
    check(ops, logits, u, p=[0.5, 0.8, 0.33, 0.9, 0.25, 0.6])
    check(ops, logits, u, k=[17000, 13334, 6001, 4500, 8192, 600], p=[0.77, 0.9, 0.5, 0.99, 0.1, 0.3], t=[1.0, 2.0, 0.5, 4.0, 1.0, 1.0])


def test_borders(ops):
    """Sums that meet a border exactly: equal weights are whole, and so are their sums."""
    for V in (16, 4096, 8192):
        logits = torch.full((5, V), 1.5)
        u = [0.0, 0.25, 0.5, 0.75, 1 - 2.0 ** -24]
        check(ops, logits, u)
        check(ops, logits, u, p=[0.5, 0.25, 0.125, 0.75, 0.0625])
        check(ops, logits.bfloat16(), u, k=[V // 2, V // 4, 8, 16, V], p=[0.5, 0.5, 0.5, 0.25, 0.25])


def test_masked_and_infinite_logits(ops):
    for V in (40, 5000):
        gen = torch.Generator().manual_seed(V)
        rows = torch.randn(10, V, generator=gen) * 3
        rows[0] = -INF
        rows[1] = NAN
        rows[2, 1:] = -INF
        rows[3, :-1] = -INF
        rows[4, 7] = NAN
        rows[5, 3] = INF
        rows[6, ::5] = INF
        rows[7] = torch.finfo(torch.float32).min
        rows[8, ::2] = torch.finfo(torch.float32).min
        rows[9, V // 2:] = -INF
        u = torch.rand(10, generator=gen).tolist()
        few = [3] * 10
        for dtype in (torch.float32, torch.bfloat16):
            logits = rows.to(dtype)
            check(ops, logits, u)
            check(ops, logits, u, t=[0.0] * 10)
            check(ops, logits, u, k=few)
            check(ops, logits, u, p=[0.6] * 10)
            check(ops, logits, u, k=[V - 1] * 10, p=[0.6] * 10, floor=[0.1] * 10)


def test_extreme_parameters(ops):
    """Values outside the documented ranges count as their ends."""
    logits, _, gen = draw(3, 8, 3000, torch.float32)
    u = [-1.0, 0.0, 1.0, 7.0, NAN, 0.5, 1 - 2.0 ** -24, 1e-30]
    tokens, _ = ops.sample_tokens(logits.cuda(), torch.tensor(u).cuda())
    same, _ = ops.sample_tokens(logits.cuda(), torch.tensor([0.0, 0.0, 1 - 2.0 ** -24, 1 - 2.0 ** -24, 0.0, 0.5, 1 - 2.0 ** -24, 1e-30]).cuda())
    assert torch.equal(tokens[[0, 1, 4, 5, 6, 7]], same[[0, 1, 4, 5, 6, 7]])
    assert (tokens[2:4] >= same[2:4]).all() and (tokens < 3000).all()
    u = torch.rand(8, generator=gen).tolist()
    check(ops, logits, u, t=[-1.0, NAN, 1e-30, 1e30, 1e-5, 1.0, 0.01, 100.0])
    check(ops, logits, u, k=[-5, -(1 << 40), 1 << 40, 3000, 2999, (1 << 32) + 1, 1, 0], index=torch.int64)
    none = torch.tensor([NAN, 1.0, 2.0, INF, NAN, NAN, 1.0, 1.5]).cuda()
    got = ops.sample_tokens(logits.cuda(), torch.tensor(u).cuda(), top_p=none, min_p=torch.full((8,), NAN).cuda())
    want = ops.sample_tokens(logits.cuda(), torch.tensor(u).cuda())
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    first = ops.sample_tokens(logits.cuda(), torch.tensor(u).cuda(), top_p=torch.full((8,), -1.0).cuda())[0]
    assert torch.equal(first, logits.argmax(1).cuda())


def test_strides_and_alignment(ops):
    """Rows of a wider buffer, at odd offsets; rows that repeat one."""
    for dtype in (torch.bfloat16, torch.float32):
        logits, u, _ = draw(5, 5, 2777, dtype)

        def view(x):
            wide = torch.full((5, 3001), 100.0, dtype=dtype, device="cuda")
            wide[:, 3:2780] = x
            return wide[:, 3:2780]

        check(ops, logits, u, view=view, p=[0.9] * 5)
        check(ops, logits, u, view=view, k=[700] * 5)
        check(ops, logits[:1].expand(5, -1), u, view=lambda x: x[:1].expand(5, -1), t=[0.5] * 5)


def test_rows_do_not_depend_on_the_batch(ops):
    logits, u, _ = draw(6, 300, 9000, torch.bfloat16, spread=4.0)
    x, u = logits.cuda(), torch.tensor(u).cuda()
    p = torch.full((300,), 0.92, device="cuda")
    tokens, logprobs = ops.sample_tokens(x, u, top_p=p)
    again, _ = ops.sample_tokens(x, u, top_p=p)
    assert torch.equal(tokens, again)
    for n in (0, 17, 299):
        one, lp = ops.sample_tokens(x[n:n + 1], u[n:n + 1], top_p=p[:1])
        assert int(one) == int(tokens[n]) and float(lp) == float(logprobs[n])


def test_frequencies(ops):
    """Tokens come as often as their probabilities say: 65536 evenly spread numbers hit each share to within two."""
    logits = torch.tensor([0.3, -1.0, 2.0, -INF, 1.1, 0.0, -4.0]).expand(65536, 7)
    u = (torch.arange(65536) + 0.5) / 65536
    tokens, _ = ops.sample_tokens(logits.cuda(), u.cuda())
    share = torch.softmax(logits[0].double(), 0) * 65536
    assert (torch.bincount(tokens.cpu(), minlength=7) - share).abs().max() <= 2


def test_captured(ops):
    logits, u, gen = draw(8, 4, 6000, torch.float32)
    x, u = logits.cuda(), torch.tensor(u).cuda()
    more = dict(temperature=torch.tensor([0.0, 0.8, 1.0, 1.2]).cuda(), top_k=torch.tensor([0, 40, 3000, 0]).cuda(),
                top_p=torch.tensor([1.0, 0.9, 0.95, 0.8]).cuda(), min_p=torch.tensor([0.0, 0.1, 0.0, 0.0]).cuda())
    ops.sample_tokens(x, u, **more)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tokens, logprobs = ops.sample_tokens(x, u, **more)
    for _ in range(4):
        x.copy_(torch.randn(4, 6000, generator=gen) * 3)
        u.copy_(torch.rand(4, generator=gen))
        graph.replay()
        want, want_lp = ops.sample_tokens(x, u, **more)
        torch.cuda.synchronize()
        assert torch.equal(tokens, want) and torch.equal(logprobs, want_lp)


def test_another_stream_and_no_rows(ops):
    logits, u, _ = draw(9, 3, 5000, torch.bfloat16)
    x, u = logits.cuda(), torch.tensor(u).cuda()
    want, _ = ops.sample_tokens(x, u)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got, _ = ops.sample_tokens(x, u)
    side.synchronize()
    assert torch.equal(got, want)
    tokens, logprobs = ops.sample_tokens(x[:0], u[:0])
    assert tokens.shape == (0,) and logprobs.shape == (0,)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kind", ["small", "large", "zeros", "mostly_zeros", "positive", "negative", "far", "masked"])
def test_ranges_of_logits(ops, kind, dtype):
    """Magnitudes around those that bf16 rows are counted in, zeros by the thousand at a border, rows of one sign, far from 0."""
    V = 6000
    logits, u, gen = draw(17, 6, V, torch.float32)
    if kind == "small":
        logits = logits * torch.tensor([1e-1, 1e-2, 1e-3, 1e-5, 1e-20, 1e-38])[:, None]
    elif kind == "large":
        logits = logits * torch.tensor([10.0, 30.0, 60.0, 1e3, 1e10, 1e37])[:, None]
    elif kind == "zeros":
        logits = torch.where(torch.rand(6, V, generator=gen) < 0.3, torch.tensor([0.0, -0.0])[torch.randint(2, (6, V), generator=gen)], logits)
    elif kind == "mostly_zeros":
        logits = torch.where(torch.rand(6, V, generator=gen) < 0.97, 0.0, logits)
    elif kind == "positive":
        logits = logits.abs() + torch.tensor([0.0, 0.01, 1.0, 8.0, 100.0, 1000.0])[:, None]
    elif kind == "negative":
        logits = -logits.abs() - torch.tensor([0.0, 0.01, 1.0, 8.0, 100.0, 1000.0])[:, None]
    elif kind == "far":
        logits = logits + torch.tensor([120.0, 128.0, -120.0, -128.0, 1e4, -1e4])[:, None]
    else:  # all but a few masked, by -infinity or the lowest number
        hidden = torch.rand(6, V, generator=gen) < torch.tensor([0.5, 0.9, 0.99, 0.999, 0.5, 0.99])[:, None]
        logits = torch.where(hidden, torch.tensor([-INF, -INF, -INF, -INF, torch.finfo(dtype).min, -1e4])[:, None], logits)
    logits = logits.to(dtype)
    check(ops, logits, u)
    check(ops, logits, u, t=[0.5, 1.0, 2.0, 0.1, 10.0, 200.0])
    check(ops, logits, u, p=[0.3, 0.6, 0.9, 0.99, 0.5, 0.8])
    check(ops, logits, u, p=[0.9, 0.5, 0.3, 0.7, 0.999, 0.95], t=[3.0, 0.7, 1.5, 20.0, 0.01, 5.0])
    check(ops, logits, u, k=[600, 3000, 4000, 5999, 513, 2500], p=[0.9, 0.8, 0.7, 0.6, 0.99, 0.5])
    check(ops, logits, u, k=[600, 3000, 4000, 5999, 20, 2500], floor=[0.1, 0.01, 0.3, 0.001, 0.5, 0.9])
    check(ops, logits, u, p=[0.9] * 6, floor=[0.1, 0.01, 0.3, 0.001, 0.5, 0.9], t=[2.0] * 6)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_vocabulary_of_millions(ops, dtype):
    """More elements than a block of one group a wave holds."""
    logits, u, _ = draw(18, 3, (1 << 22) + 4097, dtype, spread=1.5)
    check(ops, logits, u, k=[0, 100, 2000000], p=[0.9, 0.8, 0.5], t=[1.0, 0.7, 2.0])
    check(ops, logits, u, floor=[0.0, 0.01, 0.3])
