"""Linear attention with a decay for each head against the recurrence in 64 bits."""

import pytest
import torch

from tests.decoder_cases import assert_within
from tests.linear_cases import Linear, bounds

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")


@pytest.fixture(scope="module")
def ops(gpu_ops):
    from sgl_glm53_ascend_ops import ops

    return ops


def run(ops, case, chunk, checkpoints=False):
    """(out, pool, middle or None) of one call."""
    inputs, args = case.on("cuda")
    middle = None
    if checkpoints:
        N, longest, H, D = len(case.lens), max(case.lens), case.heads, case.dim
        middle = torch.full((N, longest, H, D, D), 7.0, device="cuda").transpose(3, 4)
        args["intermediate_state"] = middle
    out = (ops.linear_varlen_chunk if chunk else ops.linear_varlen_recurrent)(*inputs, **args)
    return out, args["initial_state_source"], middle


def check(ops, case, chunk, checkpoints=False):
    out, pool, middle = run(ops, case, chunk, checkpoints)
    want_out, want_pool, want_middle = case.exact(device="cuda")
    off_out, off_pool, off_middle = bounds(case, chunk, device="cuda")
    assert out.dtype == case.q.dtype and out.is_contiguous()
    assert_within(out[0], want_out, off_out, "out")
    if not checkpoints:
        assert_within(pool, want_pool, off_pool, "pool")
        return
    assert torch.equal(pool.cpu(), case.pool)  # left as it was
    for n, m in enumerate(case.lens):
        if int(case.indices[n]) > 0:
            assert_within(middle[n, :m], want_middle[n, :m], off_middle[n, :m], "middle")
            assert (middle[n, m:] == 7.0).all()
        else:
            assert (middle[n] == 7.0).all()


RECURRENT = [
    dict(lens=[1], heads=1, dim=128),
    dict(lens=[1], heads=16, dim=64, gated=False),
    dict(lens=[1] * 37, heads=16, dim=128, zero_slots=(3, 36), index64=True),
    dict(lens=[1] * 40, heads=32, dim=64, fused=True),
    dict(lens=[4, 1, 0, 3, 2], heads=5, dim=128, fp32=True, before=2, after=3),
    dict(lens=[0, 0, 7], heads=3, dim=64, fp32=True, fused=True, track=[0, 1, 7]),
    dict(lens=[9, 5, 1, 3], heads=2, dim=128, track=[4, 0, 1, 9], index64=True, zero_slots=(0,)),
    dict(lens=[33], heads=7, dim=64, gated=False, after=1),
    dict(lens=[1] * 300, heads=8, dim=128, gated=False, index64=True),
    dict(lens=[1] * 9, heads=8, dim=128, fp32=True),
    dict(lens=[2, 1, 0, 5] * 3, heads=8, dim=128, fp32=True, track=[1, 0, 0, 5] * 3),
    dict(lens=[2, 1, 0, 5] * 3, heads=8, dim=128, zero_slots=(1,), track=[2, 0, 0, 3] * 3, after=1),
    dict(lens=[3, 1] * 5, heads=8, dim=64, fp32=True, after=2),
    dict(lens=[1] * 4, heads=16, dim=128),                                  # 63 and 64 states
    dict(lens=[1] * 9, heads=7, dim=128),
]


@pytest.mark.parametrize("spec", RECURRENT, ids=range(len(RECURRENT)))
def test_recurrent(ops, spec):
    check(ops, Linear(1, **spec), chunk=False)


@pytest.mark.parametrize("spec", [
    dict(lens=[4, 4, 4], heads=16, dim=128, zero_slots=(1,)),
    dict(lens=[3, 1, 0, 2], heads=3, dim=64, fp32=True),
    dict(lens=[2] * 70, heads=8, dim=128, gated=False, index64=True),
])
def test_recurrent_checkpoints(ops, spec):
    check(ops, Linear(2, **spec), chunk=False, checkpoints=True)


CHUNK = [
    dict(lens=[1], heads=1, dim=128),
    dict(lens=[1], heads=3, dim=64, gated=False),
    dict(lens=[63, 64, 65, 1, 0, 128], heads=2, dim=128, before=5, after=70),
    dict(lens=[63, 64, 65, 1, 0, 128], heads=5, dim=64, gated=False, fused=True, zero_slots=(1, 3)),
    dict(lens=[700], heads=2, dim=128),                                     # several segments
    dict(lens=[129, 1, 640, 255, 0, 257], heads=2, dim=64, index64=True, after=1),
    dict(lens=[129, 384, 3, 256], heads=1, dim=128, fused=True, gated=False, zero_slots=(1,)),
    dict(lens=[700, 200], heads=2, dim=128, track=[333, 128]),
    dict(lens=[400, 64, 100, 0, 77, 10], heads=2, dim=64, track=[384, 64, 0, 0, 78, 3], index64=True),
    dict(lens=[520], heads=1, dim=128, track=[520], zero_slots=(0,)),
    dict(lens=[1] * 300, heads=2, dim=64),
    dict(lens=[5] * 64 + [700], heads=3, dim=128),
    dict(lens=[1030], heads=9, dim=128, gated=False),                       # a head count that is no power of two
]


@pytest.mark.parametrize("spec", CHUNK, ids=range(len(CHUNK)))
def test_chunk(ops, spec):
    check(ops, Linear(3, **spec), chunk=True)


@pytest.mark.parametrize("g", ["steep", "resets", "none", "mixed"])
@pytest.mark.parametrize("chunk", [True, False])
def test_decays_of_any_steepness(ops, g, chunk):
    """No decay, hundreds of nats a token, and tokens that forget everything before them."""
    case = Linear(4, lens=[300, 70], heads=2, dim=64)
    gen = torch.Generator().manual_seed(5)
    x = torch.rand(case.g.shape, generator=gen)
    if g == "steep":
        case.g = -300.0 * x
    elif g == "resets":
        case.g = torch.where(x < 0.05, -INF, case.g)
    elif g == "none":
        case.g = torch.zeros_like(case.g)
    else:
        case.g = torch.where(x < 0.1, -5000.0, -1e-4 * x)
    check(ops, case, chunk)


@pytest.mark.parametrize("chunk", [True, False])
@pytest.mark.parametrize("which,value", [("v", INF), ("v", NAN), ("k", NAN), ("q", NAN), ("k", -INF)])
def test_what_is_not_finite_stays_behind_its_token(ops, chunk, which, value):
    """Earlier tokens, other requests and other heads keep their results; of v, other columns too."""
    case = Linear(6, lens=[200, 300], heads=2, dim=64)
    out0, pool0, _ = run(ops, case, chunk)
    t, head = 200 + 150, 1  # inside a chunk, and inside a segment
    getattr(case, which)[0, t, head, 5] = value
    out, pool, _ = run(ops, case, chunk)
    same = torch.ones_like(out[0], dtype=torch.bool)
    if which == "q":
        same[t, head] = False
    elif which == "v":
        same[t:500, head, 5] = False
    else:
        same[t:500, head] = False
    # a chunk with such a value is formed token by token: other roundings, within the bounds
    want, _, _ = Linear(6, lens=[200, 300], heads=2, dim=64).exact()
    off = bounds(Linear(6, lens=[200, 300], heads=2, dim=64), chunk)[0]
    assert_within(out[0].cpu()[same.cpu()], want[same.cpu()], off[same.cpu()], "elsewhere")
    assert not torch.isfinite(out[0][t, head][~same[t, head]]).any()
    held = int(case.indices[1])
    fine = torch.ones_like(pool, dtype=torch.bool)
    if which != "q":
        fine[held, head] = False
    assert torch.isfinite(pool[fine]).all()
    if which == "v":
        assert torch.isfinite(pool[held, head][:, torch.arange(64) != 5]).all()
        assert not torch.isfinite(pool[held, head][:, 5]).any()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("value", [INF, -INF, NAN])
def test_a_value_that_is_not_finite_is_found_anywhere(ops, dim, value):
    """In every eighth of a row and row of a chunk: earlier tokens and other columns keep finite results."""
    for token, column in [(0, 0), (1, 1), (2, 2), (17, 3), (31, dim // 2 + 4), (32, dim // 2 + 5), (62, dim - 2), (63, dim - 1)]:
        case = Linear(9, lens=[64], heads=1, dim=dim)
        case.v[0, token, 0, column] = value
        out, pool, _ = run(ops, case, True)
        fine = torch.ones(64, dim, dtype=torch.bool)
        fine[token:, column] = False
        assert torch.isfinite(out[0, :, 0].cpu()[fine]).all(), (token, column)
        assert not torch.isfinite(out[0, token, 0, column]), (token, column)
        state = pool[int(case.indices[0]), 0].cpu()
        assert torch.isfinite(state[:, torch.arange(dim) != column]).all()
        assert not torch.isfinite(state[:, column]).any()


def test_forms_agree_and_calls_repeat(ops):
    """The chunk form is the same from call to call, and split calls continue each other's states."""
    case = Linear(7, lens=[600], heads=4, dim=128)
    out, pool, _ = run(ops, case, True)
    again, pool2, _ = run(ops, case, True)
    assert torch.equal(out, again) and torch.equal(pool, pool2)
    inputs, args = case.on("cuda")
    parts = []
    for a, b in ((0, 100), (100, 101), (101, 600)):
        part = [x[:, a:b] for x in inputs]
        args["cu_seqlens"] = torch.tensor([0, b - a], dtype=torch.int32, device="cuda")
        parts.append((ops.linear_varlen_recurrent if b - a == 1 else ops.linear_varlen_chunk)(*part, **args))
    want, want_pool, _ = case.exact()
    off, off_pool, _ = bounds(case, False)
    assert_within(torch.cat(parts, 1)[0], want, off + bounds(case, True)[0], "out")
    assert_within(args["initial_state_source"], want_pool, off_pool + bounds(case, True)[1], "pool")


def test_slots_and_offsets_outside(ops):
    """Slots outside the pool count as the padding row, offsets past the tokens are cut; int64 entries count whole."""
    for chunk in (True, False):
        for index in (torch.int32, torch.int64):
            case = Linear(8, lens=[70, 20], heads=2, dim=64)
            inputs, args = case.on("cuda")
            far = [case.slots, -1] if index == torch.int32 else [(1 << 32) + 1, -(1 << 32) + 1]
            args["initial_state_indices"] = torch.tensor(far, dtype=index, device="cuda")
            args["cu_seqlens"] = torch.tensor([0, 70, 2000000000 if index == torch.int32 else (1 << 32) + 71], dtype=index, device="cuda")
            op = ops.linear_varlen_chunk if chunk else ops.linear_varlen_recurrent
            out = op(*inputs, **args)
            assert torch.equal(args["initial_state_source"].cpu(), case.pool)
            case.indices.zero_()
            want = case.exact()[0]
            assert_within(out[0], want, bounds(case, chunk)[0], "out")


def test_far_states_and_tokens(ops):
    """Offsets beyond 2^31 elements in the pool and in q, k, v."""
    case = Linear(9, lens=[90], heads=1, dim=64)
    inputs, args = case.on("cuda")
    stride = 1 << 30
    pool = torch.empty(4 * stride, device="cuda").as_strided((4, 1, 64, 64), (stride, 4096, 1, 64))
    pool[3] = args["initial_state_source"][int(case.indices[0])]
    far = torch.empty(90 * (1 << 25) + 64, dtype=torch.bfloat16, device="cuda")
    spread = []
    for i, x in enumerate(inputs[:3]):
        spread.append(far.as_strided((1, 90, 1, 64), (0, 1 << 25, 64, 1), i * 1024))
        spread[-1].copy_(x)
    args["initial_state_source"] = pool
    args["initial_state_indices"] = torch.tensor([3], dtype=torch.int32, device="cuda")
    begin = pool[3].clone()
    want, want_pool, _ = case.exact()
    for chunk in (True, False):
        pool[3] = begin
        out = (ops.linear_varlen_chunk if chunk else ops.linear_varlen_recurrent)(*spread, inputs[3], **args)
        off, off_pool, _ = bounds(case, chunk)
        assert_within(out[0], want, off, "out")
        assert_within(pool[3], want_pool[int(case.indices[0])], off_pool[int(case.indices[0])], "state")


@pytest.mark.parametrize("chunk", [True, False])
def test_captured(ops, chunk):
    """A replayed graph follows the contents of its inputs and gives what eager calls give, at every replay."""
    cases = [Linear(s, lens=[200, 5, 150] if chunk else [2, 1, 3], heads=2, dim=128) for s in (10, 11, 12)]
    op = ops.linear_varlen_chunk if chunk else ops.linear_varlen_recurrent
    inputs, args = cases[0].on("cuda")
    op(*inputs, **args)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = op(*inputs, **args)
    for case in cases + cases[::-1]:
        fresh, fresh_args = case.on("cuda")
        for to, x in zip(inputs, fresh):
            to.copy_(x)
        for name in ("initial_state_source", "initial_state_indices"):
            args[name].copy_(fresh_args[name])
        graph.replay()
        want = op(*fresh, **fresh_args)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert torch.equal(args["initial_state_source"], fresh_args["initial_state_source"])


def test_on_another_stream(ops):
    case = Linear(13, lens=[500], heads=2, dim=128)
    want, want_pool, _ = run(ops, case, True)
    inputs, args = case.on("cuda")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        out = ops.linear_varlen_chunk(*inputs, **args)
    side.synchronize()
    assert torch.equal(out, want) and torch.equal(args["initial_state_source"], want_pool)


def test_no_requests_and_no_tokens(ops):
    for op in (ops.linear_varlen_chunk, ops.linear_varlen_recurrent):
        case = Linear(14, lens=[3], heads=2, dim=64)
        inputs, args = case.on("cuda")
        args["initial_state_indices"] = args["initial_state_indices"][:0]
        args["cu_seqlens"] = args["cu_seqlens"][:1]
        assert (op(*inputs, **args) == 0).all()
        case = Linear(15, lens=[0, 0], heads=2, dim=64, track=[0, 1])
        inputs, args = case.on("cuda")
        assert op(*inputs, **args).shape == (1, 0, 2, 64)
        want = case.pool.clone()
        want[int(case.track[0][0])] = case.pool[int(case.indices[0])]
        assert torch.equal(args["initial_state_source"].cpu(), want)
