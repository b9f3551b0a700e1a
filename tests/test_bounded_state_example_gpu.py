"""The hybrid decoder example with layers of bounded state: linear attention, windows with sinks and sampling together."""

import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SAMPLED = dict(temperature=0.9, top_k=200, top_p=0.95, min_p=0.01)


@pytest.fixture(scope="module")
def example(gpu_ops):
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    try:
        import hybrid_decoder
    finally:
        sys.path.pop(0)
    return hybrid_decoder


@pytest.mark.parametrize("layers,window,sinks", [("llal", 50, 4), ("la", 0, 0), ("kla", 33, 70)])
def test_split_calls_agree_with_one_prefill(example, layers, window, sinks):
    """The last tokens' hidden states do not depend on how the tokens were cut into calls.

    Both runs round the same quantities to bf16 at about 10 places a layer, at an rms of 2^-9 relative each:
    sqrt(2 * 4 * 10) * 2^-9 = 0.018 for four layers where all of it is independent, and twice that is allowed.
    """
    cfg = example.Config(layers=layers, window=window, sinks=sinks)
    lens = [130, 3, 77, 200]
    gen = torch.Generator().manual_seed(1)
    prompts = [torch.randint(cfg.vocab, (n,), generator=gen) for n in lens]
    parts = [[n // 3 for n in lens], [n // 3 for n in lens], [n - 2 * (n // 3) for n in lens]]
    results = []
    for calls in ([lens], parts, [[n - 2 for n in lens], [1] * 4, [1] * 4]):
        torch.manual_seed(0)
        pages = example.Pages(cfg, len(lens), max(lens), "cuda")
        model = example.HybridDecoder(cfg, len(lens), pages.pages)
        at = [0] * len(lens)
        for new in calls:
            tokens = torch.cat([p[a:a + m] for p, a, m in zip(prompts, at, new)]).cuda()
            at = [a + m for a, m in zip(at, new)]
            step = pages.step(new)
            hidden = model.hidden(tokens, step)
        results.append(hidden[step.cu_seqlens[1:].long() - 1].float())
    for other in results[1:]:
        error = (other - results[0]).norm(dim=-1) / results[0].norm(dim=-1)
        assert error.max() < 0.036, error


@pytest.mark.parametrize("sampling", [{}, SAMPLED])
def test_captured_decode_agrees_with_eager(example, sampling):
    """Prompts, then six drawn tokens of each request: the graph's are those of eager calls with the same numbers."""
    cfg = example.Config(layers="llal", window=40, sinks=4, **sampling)
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


def test_drawn_tokens_follow_the_logits(example):
    """The step's token is the one that its own logits and number give (one row in 64 bits; ties and borders are elsewhere)."""
    from tests.test_sampling_gpu import plain

    cfg = example.Config(layers="l", **SAMPLED)
    torch.manual_seed(3)
    pages = example.Pages(cfg, 2, 20, "cuda")
    model = example.HybridDecoder(cfg, 2, pages.pages)
    tokens = torch.randint(cfg.vocab, (20,)).cuda()
    step = pages.step([12, 8])
    got = model.next_tokens(tokens, step)
    model.layers[0]["state"].zero_()
    last = model.hidden(tokens, step)[step.cu_seqlens[1:].long() - 1] @ model.head
    f32 = lambda x: float(torch.tensor(x, dtype=torch.float32))  # noqa: E731
    for n in range(2):
        token, _ = plain(last[n].float().cpu(), float(step.uniforms[n]), f32(0.9), 200, f32(0.95), f32(0.01))
        assert int(got[n]) == token
