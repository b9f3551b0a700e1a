"""Linear attention token by token on rows that start at 16 bytes and no more."""

import pytest
import torch

from tests.decoder_cases import assert_within
from tests.linear_cases import Linear, bounds

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fp32", [True, False])
@pytest.mark.parametrize("lens", [[1] * 40, [3, 1, 0, 4] * 10, [2, 1]], ids=["one", "several", "few"])
@pytest.mark.parametrize("dim", [64, 128])
def test_rows_aligned_to_16_bytes(gpu_ops, dim, lens, fp32):
    """q, k, v and the pool at odd multiples of 16 bytes, by their first element and by their strides."""
    from sgl_glm53_ascend_ops import ops

    case = Linear(31, lens=lens, heads=2, dim=dim, fp32=fp32)
    inputs, args = case.on("cuda")
    unit = 4 if fp32 else 8

    def moved(t):
        row = dim + unit
        flat = torch.zeros(t.shape[1] * 2 * row + unit, dtype=t.dtype, device="cuda")
        view = flat[unit:].view(1, t.shape[1], 2, row)[..., :dim]
        view.copy_(t)
        return view

    pool = args["initial_state_source"]
    slot = 2 * dim * dim + 4
    away = torch.zeros(case.slots * slot + 4, device="cuda").as_strided(pool.shape, (slot, dim * dim, 1, dim), 4)
    away.copy_(pool)
    args["initial_state_source"] = away
    out = ops.linear_varlen_recurrent(*[moved(t) for t in inputs[:3]], inputs[3], **args)
    want_out, want_pool, _ = case.exact(device="cuda")
    off_out, off_pool, _ = bounds(case, False, device="cuda")
    assert_within(out[0], want_out, off_out, "out")
    assert_within(away, want_pool, off_pool, "pool")
