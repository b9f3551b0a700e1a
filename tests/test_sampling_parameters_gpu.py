"""Sampling with parameters at the ends of their ranges, against its definition in 64 bits."""

import pytest
import torch

from tests.test_sampling_gpu import INF, check, draw

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(gpu_ops):
    from sgl_glm53_ascend_ops import ops

    return ops


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [5, 6000, 70001])
def test_an_infinite_temperature(ops, vocab, dtype):
    """All weights are 1, and reach any min_p: the draw is uniform over what top_k and top_p leave, -infinity left out."""
    logits, u, _ = draw(vocab, 4, vocab, dtype)
    logits[3, ::2] = -INF
    t, floor = [INF] * 4, [0.0, 0.5, 1.0, 2.0]
    k, p = [1, 2, max(vocab // 2, 1), vocab - 1], [0.2, 1.0, 0.9, 0.5]
    check(ops, logits, u, t=t)
    for floor in (floor, floor[::-1], [1.0] * 4):
        check(ops, logits, u, t=t, floor=floor)
        check(ops, logits, u, t=t, floor=floor, k=k)
        check(ops, logits, u, t=t, floor=floor, p=p)
        check(ops, logits, u, t=t, floor=floor, k=k, p=p)
