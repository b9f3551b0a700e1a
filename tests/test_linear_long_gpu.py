"""Linear attention in chunks: many segments, decays that grow, and how near states are to fp32."""

import pytest
import torch

from tests.decoder_cases import assert_within
from tests.linear_cases import Linear, bounds

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(gpu_ops):
    from sgl_glm53_ascend_ops import ops

    return ops


class Long(Linear):
    """Without the states after every token."""

    def exact(self, absolute=False, device="cpu"):
        f = (lambda t: t.to(device).double().abs()) if absolute else (lambda t: t.to(device).double())
        q, k, v, pool = f(self.q[0]), f(self.k[0]), f(self.v[0]), f(self.pool)
        decay = self.g.to(device).double().expand(1, self.q.shape[1], self.heads)[0].exp()
        out, begin, t = torch.zeros_like(q), pool.clone(), self.before
        for n, m in enumerate(self.lens):
            slot = int(self.indices[n])
            S = begin[slot].clone() if slot > 0 else torch.zeros_like(begin[0])
            for i in range(m + 1):
                if self.track is not None and int(self.track[1][n]) == i:
                    pool[int(self.track[0][n])] = S
                if i < m:
                    S = S * decay[t][:, None, None] + k[t][:, :, None] * v[t][:, None, :]
                    out[t] = (q[t][:, :, None] * S).sum(1) * self.scale
                    t += 1
            if slot > 0:
                pool[slot] = S
        return out, pool, torch.zeros((), dtype=torch.float64, device=device)


def check(ops, case, chunk=True):
    inputs, args = case.on("cuda")
    out = (ops.linear_varlen_chunk if chunk else ops.linear_varlen_recurrent)(*inputs, **args)
    want_out, want_pool, _ = case.exact(device="cuda")
    off_out, off_pool, _ = bounds(case, chunk, device="cuda")
    assert_within(out[0], want_out, off_out, "out")
    assert_within(args["initial_state_source"], want_pool, off_pool, "pool")


# Weak decays: what the first segments hold still matters in the last. Segments have 128 tokens here but where it says.
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("spec", [
    dict(lens=[2047], heads=1),
    dict(lens=[2048], heads=2),                                  # 16 segments
    dict(lens=[2049], heads=1, zero_slots=(0,)),                 # 17
    dict(lens=[2177, 3, 2500], heads=1, track=[2176, 0, 2300]),  # prefixes at the 17th segment's end and inside the 18th
    dict(lens=[4097], heads=1, gated=False),                     # 33
    dict(lens=[4300, 130], heads=2, before=3, after=2),
    dict(lens=[700, 1, 0, 1, 340], heads=64),                    # 320 tokens
    dict(lens=[1100] + [1] * 299, heads=2, track=[1000] + [2] * 299),  # 512
], ids=range(8))
def test_many_segments(ops, spec, dim):
    check(ops, Long(21, dim=dim, g_mean=-9.0, **spec))


@pytest.mark.parametrize("chunk", [True, False])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("begin", [0.0, 1e-12])
def test_positive_decays_are_limited_by_64_tokens(ops, begin, dim, chunk):
    """exp(sum) is past fp32 over a segment of 512 tokens, not over 64, and no state is near fp32's ends."""
    case = Long(22, lens=[1200] + [1] * 255, heads=2, dim=dim)
    case.g = torch.full_like(case.g, -0.2)
    case.g[:, :512] = 0.2
    case.v[:, :450] = 0
    case.pool.mul_(begin)
    check(ops, case, chunk)


@pytest.mark.parametrize("dim", [64, 128])
def test_states_are_those_of_fp32(ops, dim):
    """Token j alone has key element j: element j of the state is its value times its decay, no sum. Decays of up to a
    factor of two: an exponent is off by 2^-24 of at most 1 (2^-24 in the exponential), the exponential by 2^-23, its product by
    2^-24, the three parts of that by 2^-26, and they are added up in fp32, 2^-23 each: less than 2^-20 together. Two
    parts would be off by up to 2^-17."""
    case = Linear(23, lens=[64], heads=2, dim=dim)
    case.k = torch.eye(64, dim)[None, :, None].expand(1, 64, 2, dim).contiguous().bfloat16()
    case.g = -torch.rand(case.g.shape, generator=torch.Generator().manual_seed(24)) * (0.69 / 64)
    case.pool.zero_()
    inputs, args = case.on("cuda")
    ops.linear_varlen_chunk(*inputs, **args)
    slot = int(case.indices[0])
    want = case.exact()[1][slot]
    assert_within(args["initial_state_source"][slot], want, want.abs() * 2.0 ** -20, "state")
    rest = want - want.bfloat16().double()
    rest = rest - rest.bfloat16().double()
    assert (rest.abs() > want.abs() * 2.0 ** -20).any()  # the bound tells two parts from three
