"""The hybrid decoder example: its operators together, over prefill, chunks, decode steps and a captured graph."""

import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example(gpu_ops):
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    try:
        import hybrid_decoder
    finally:
        sys.path.pop(0)
    return hybrid_decoder


def _split(lens, parts):
    """Every request's tokens in `parts` calls, the remainder in the last."""
    calls = [[n // parts for n in lens] for _ in range(parts - 1)]
    return calls + [[n - sum(c[i] for c in calls) for i, n in enumerate(lens)]]


@pytest.mark.parametrize("fp8,window", [(False, 0), (False, 50), (True, 0)])
def test_split_calls_agree_with_one_prefill(example, fp8, window):
    """The last tokens' hidden states do not depend on how the tokens were cut into calls.

    Both runs round the same quantities to bf16 at about 10 places a layer, at an rms of 2^-9 relative
    each: sqrt(2 * 4 * 10) * 2^-9 = 0.018 where all of it is independent, and twice that is allowed. 8 bits
    (steps of 2^-4, rms 0.02) come in at 4 places of the one attention layer: sqrt(2 * 4) * 0.02 = 0.05 more.
    """
    cfg = example.Config(fp8=fp8, window=window)
    lens = [130, 3, 77, 200]
    gen = torch.Generator().manual_seed(1)
    prompts = [torch.randint(cfg.vocab, (n,), generator=gen) for n in lens]
    results = []
    for calls in ([lens], _split(lens, 3), [[n - 2 for n in lens], [1] * 4, [1] * 4]):
        torch.manual_seed(0)
        pages = example.Pages(cfg, len(lens), max(lens), "cuda")
        model = example.HybridDecoder(cfg, len(lens), pages.pages)
        at = [0] * len(lens)
        for new in calls:
            tokens = torch.cat([p[a:a + m] for p, a, m in zip(prompts, at, new)]).cuda()
            at = [a + m for a, m in zip(at, new)]
            step = pages.step(new)
            hidden = model.hidden(tokens, step)
        assert at == lens
        results.append(hidden[step.cu_seqlens[1:].long() - 1].float())
    for other in results[1:]:
        error = (other - results[0]).norm(dim=-1) / results[0].norm(dim=-1)
        assert error.max() < (0.086 if fp8 else 0.036), error


@pytest.mark.parametrize("fp8", [False, True])
def test_captured_decode_agrees_with_eager(example, fp8):
    cfg = example.Config(fp8=fp8)
    gen = torch.Generator().manual_seed(2)
    prompts = [torch.randint(cfg.vocab, (n,), generator=gen).tolist() for n in (64, 1, 190)]
    torch.manual_seed(0)
    got, _ = example.generate(cfg, prompts, 6)

    torch.manual_seed(0)
    pages = example.Pages(cfg, 3, 190 + 6, "cuda")
    model = example.HybridDecoder(cfg, 3, pages.pages)
    tokens = torch.tensor([t for p in prompts for t in p], device="cuda")
    want = [model.next_tokens(tokens, pages.step([len(p) for p in prompts]))]
    for _ in range(5):
        want.append(model.next_tokens(want[-1], pages.step([1, 1, 1])))
    assert torch.equal(got, torch.stack(want, 1))
