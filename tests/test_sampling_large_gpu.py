"""Sampling from vocabularies above 65536, whose bf16 rows are counted in a table of their own size."""

import pytest
import torch

from tests.test_sampling_gpu import INF, NAN, check, draw

pytestmark = pytest.mark.gpu

V = 70001


@pytest.fixture(scope="module")
def ops(gpu_ops):
    from sgl_glm53_ascend_ops import ops

    return ops


def filtered(ops, logits, u):
    """Each filter alone and together, for six rows."""
    check(ops, logits, u)
    check(ops, logits, u, t=[0.5, 1.0, 2.0, 0.1, 10.0, 200.0])
    check(ops, logits, u, p=[0.3, 0.6, 0.9, 0.99, 0.5, 0.8])
    check(ops, logits, u, p=[0.9, 0.5, 0.3, 0.7, 0.999, 0.95], t=[3.0, 0.7, 1.5, 20.0, 0.01, 5.0])
    check(ops, logits, u, floor=[0.1, 0.01, 0.3, 0.001, 0.5, 1.0])
    check(ops, logits, u, k=[600, 3000, 40000, V - 1, 513, 25000], p=[0.9, 0.8, 0.7, 0.6, 0.99, 0.5])
    check(ops, logits, u, k=[600, 3000, 40000, V, 20, 25000], floor=[0.1, 0.01, 0.3, 0.001, 0.5, 0.9])
    check(ops, logits, u, p=[0.9] * 6, floor=[0.1, 0.01, 0.3, 0.001, 0.5, 0.9], t=[2.0] * 6)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("spread", [0.3, 2.5, 8.0])
def test_filters(ops, spread, dtype):
    logits, u, _ = draw(41, 6, V, dtype, spread=spread)
    filtered(ops, logits, u)


@pytest.mark.parametrize("kind", ["small", "large", "zeros", "mostly_zeros", "positive", "negative", "far", "masked"])
def test_ranges_of_logits(ops, kind):
    """Magnitudes around those that rows are counted in, more zeros than are kept aside, rows of one sign, far from 0."""
    logits, u, gen = draw(42, 6, V, torch.float32)
    if kind == "small":
        logits = logits * torch.tensor([1e-3, 1e-6, 1e-7, 1e-8, 1e-20, 1e-38])[:, None]
    elif kind == "large":
        logits = logits * torch.tensor([10.0, 30.0, 60.0, 1e3, 1e10, 1e37])[:, None]
    elif kind == "zeros":
        some = torch.rand(6, V, generator=gen) < torch.tensor([0.02, 0.0285, 0.0295, 0.04, 0.3, 0.5])[:, None]  # 2048: 0.02926
        logits = torch.where(some, torch.tensor([0.0, -0.0])[torch.randint(2, (6, V), generator=gen)], logits)
    elif kind == "mostly_zeros":
        logits = torch.where(torch.rand(6, V, generator=gen) < 0.97, 0.0, logits)
    elif kind == "positive":
        logits = logits.abs() + torch.tensor([0.0, 0.01, 1.0, 8.0, 100.0, 1000.0])[:, None]
    elif kind == "negative":
        logits = -logits.abs() - torch.tensor([0.0, 0.01, 1.0, 8.0, 100.0, 1000.0])[:, None]
    elif kind == "far":
        logits = logits + torch.tensor([120.0, 128.0, -120.0, -128.0, 1e4, -1e4])[:, None]
    else:  # all but a few masked, by -infinity or the lowest number
        hidden = torch.rand(6, V, generator=gen) < torch.tensor([0.5, 0.9, 0.99, 0.9999, 0.5, 0.99])[:, None]
        lowest = torch.finfo(torch.bfloat16).min
        logits = torch.where(hidden, torch.tensor([-INF, -INF, -INF, -INF, lowest, -1e4])[:, None], logits)
    filtered(ops, logits.bfloat16(), u)


def test_flat_rows_and_ties(ops):
    """Equal logits by the thousand, cut by index: within a block, at its ends, in the last one."""
    rows = torch.zeros(6, V)
    rows[1, ::3] = -1.0
    rows[2] = torch.arange(V) // 5000 * -0.5
    rows[3, 100:] = -2.0
    rows[4] = 7.25
    rows[5] = torch.arange(V).flip(0) // 100 * 0.0078125
    u = [0.1, 0.9, 0.5, 0.7, 0.999, 0.3]
    logits = rows.bfloat16()
    check(ops, logits, u)
    check(ops, logits, u, k=[9000, 5000, 12000, 400, V - 1, 5000])
    check(ops, logits, u, k=[2048, 2049, 4096, 2047, 65536, 6144])
    check(ops, logits, u, p=[0.5, 0.8, 0.33, 0.9, 0.25, 0.6])
    check(ops, logits, u, p=[1e-6, 0.99999, 0.7, 0.01, 0.5, 0.001], floor=[0.1] * 6)
    check(ops, logits, u, k=[17000, 13334, 6001, 4500, 8192, 600], p=[0.77, 0.9, 0.5, 0.99, 0.1, 0.3], t=[1.0, 2.0, 0.5, 4.0, 1.0, 1.0])


def test_masked_and_infinite_logits(ops):
    gen = torch.Generator().manual_seed(43)
    rows = torch.randn(10, V, generator=gen) * 3
    rows[0] = -INF
    rows[1] = NAN
    rows[2, 1:] = -INF
    rows[3, :-1] = -INF
    rows[4, 7] = NAN
    rows[4, 8] = -NAN
    rows[5, 3] = INF
    rows[6, ::5] = INF
    rows[7] = torch.finfo(torch.bfloat16).min
    rows[8, ::2] = torch.finfo(torch.bfloat16).min
    rows[9, V // 2:] = -INF
    u = torch.rand(10, generator=gen).tolist()
    logits = rows.bfloat16()
    check(ops, logits, u)
    check(ops, logits, u, t=[0.0] * 10)
    check(ops, logits, u, k=[3] * 10)
    check(ops, logits, u, k=[400] * 10)
    check(ops, logits, u, p=[0.6] * 10)
    check(ops, logits, u, floor=[0.05] * 10)
    check(ops, logits, u, k=[V - 1] * 10, p=[0.6] * 10, floor=[0.1] * 10)


def test_rows_repeat_beside_others(ops):
    logits, u, _ = draw(44, 300, V, torch.bfloat16, spread=4.0)
    x, u = logits.cuda(), torch.tensor(u).cuda()
    p, floor = torch.full((300,), 0.92, device="cuda"), torch.full((300,), 0.01, device="cuda")
    tokens, logprobs = ops.sample_tokens(x, u, top_p=p, min_p=floor)
    again, _ = ops.sample_tokens(x, u, top_p=p, min_p=floor)
    assert torch.equal(tokens, again)
    for n in (0, 17, 299):
        one, lp = ops.sample_tokens(x[n:n + 1], u[n:n + 1], top_p=p[:1], min_p=floor[:1])
        assert int(one) == int(tokens[n]) and float(lp) == float(logprobs[n])
