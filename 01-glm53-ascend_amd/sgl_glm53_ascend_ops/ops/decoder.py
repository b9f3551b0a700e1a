"""Keyword wrappers over the norms and the paged attention of a hybrid decoder.

A model that interleaves KDA layers with full attention needs these beside
``ops.kda``: the residual RMS norm in front of every projection (with an 8-bit
output where the projection is an 8-bit product), for the full-attention
layers a paged key/value cache, its writer and the attention that reads it, and at its
end the choice of a token. The reference package has no counterpart. Like the KDA operators they enqueue on the
current stream, never synchronize the host and can be captured in a HIP graph.
"""

from typing import Optional, Tuple

import torch

from .. import load_library

load_library()
_OPS = torch.ops.sgl_glm53_ascend


def add_rms_norm(
    x: torch.Tensor,
    weight: torch.Tensor,
    eps: float,
    *,
    residual: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """``h = x + residual``, normed: ``h * weight / sqrt(mean(h^2) + eps)`` in x's dtype.

    ``x`` is ``[..., width]`` in bf16 or fp32 with rows at one stride, or at two (the
    heads of a fused projection, ``qkv[:, :, :heads]``); ``weight`` and ``residual``
    (rows at one stride) may each be bf16 or fp32. ``residual`` (None: ``h = x``) is
    updated in place to ``h``; the norm reads ``h`` in fp32, before that rounding.
    """
    return _OPS.add_rms_norm(x, weight, eps, residual=residual)


def add_rms_norm_fp8(
    x: torch.Tensor,
    weight: torch.Tensor,
    eps: float,
    *,
    residual: Optional[torch.Tensor] = None,
    group_size: int = 0,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """:func:`add_rms_norm` in 8 bits: ``(out, scale)`` with ``y = out.float() * scale``.

    ``out`` is ``float8_e4m3fn``; ``scale`` is fp32, ``[..., 1]`` (``group_size``
    0: one a row) or ``[..., ceil(width / 128)]`` (``group_size`` 128):
    ``max(max|y| / 448, 1e-12)`` of the group. ``y`` is not rounded in between; a value
    within a few fp32 roundings of a tie may take either 8-bit neighbour.
    """
    return _OPS.add_rms_norm_fp8(x, weight, eps, residual=residual, group_size=group_size)


def paged_kv_store(
    k: torch.Tensor,
    v: torch.Tensor,
    *,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    slot_indices: torch.Tensor,
    k_scale: Optional[torch.Tensor] = None,
    v_scale: Optional[torch.Tensor] = None,
) -> None:
    """Write the new tokens' keys and values into the pages of a cache, in place.

    ``k, v`` are bf16 ``[1, T, kv_heads, D]`` (slices of a fused projection work),
    the caches ``[pages, page_size, kv_heads, D]`` in bf16 or ``float8_e4m3fn``,
    D 64 or 128. Token ``t`` goes to slot ``slot_indices[t] = page * page_size +
    offset``; slots outside the pool (negative: padding) are skipped, and of two
    tokens with one slot either's values may remain. An 8-bit cache keeps
    ``x / scale[head]`` (fp32 ``[kv_heads]``, None: 1), held within +-448.
    """
    _OPS.paged_kv_store(k, v, k_cache=k_cache, v_cache=v_cache, slot_indices=slot_indices,
                        k_scale=k_scale, v_scale=v_scale)


def paged_attention(
    q: torch.Tensor,
    *,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    page_table: torch.Tensor,
    kv_lens: torch.Tensor,
    cu_seqlens: torch.Tensor,
    scale: float,
    max_query_len: int,
    window: int = 0,
    sink_tokens: int = 0,
    logit_cap: float = 0.0,
    k_scale: Optional[torch.Tensor] = None,
    v_scale: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Causal attention of new tokens over a paged cache that holds their keys already.

    ``q`` is bf16 ``[1, T, heads, D]``, ``heads`` a multiple of ``kv_heads`` (query
    head ``h`` reads key head ``h // (heads // kv_heads)``). Request ``n`` has the
    tokens ``cu_seqlens[n]`` to ``cu_seqlens[n + 1]`` and ``kv_lens[n]`` cached
    ones, the new ones last, on the pages ``page_table[n]`` (``[N, max_pages]``).
    One call serves decode steps, verify steps and prefill chunks alike, mixed too.

    ``window`` > 0 shows a token only the last ``window`` keys, its own among
    them, and beside those the request's first ``sink_tokens`` keys (the sinks), so a token at position
    ``p`` sees the keys ``j <= p`` with ``j > p - window or j < sink_tokens``; the pages in between are
    not read. ``logit_cap`` > 0 turns a score ``s`` into ``logit_cap * tanh(s /
    logit_cap)``. ``k_scale, v_scale`` as in :func:`paged_kv_store`. A token that
    sees no key, or that no request covers, gets zeros; pages outside the pool
    read as zero keys and values. Scores, softmax and sums are fp32; the softmax
    weights are rounded to bf16 for the product with the values. ``max_query_len``,
    the most new tokens of a request, chooses the kernel (results hold for any
    value). Returns ``[1, T, heads, D]`` in bf16.
    """
    return _OPS.paged_attention(
        q, k_cache=k_cache, v_cache=v_cache, page_table=page_table, kv_lens=kv_lens,
        cu_seqlens=cu_seqlens, scale=scale, max_query_len=max_query_len, window=window,
        logit_cap=logit_cap, k_scale=k_scale, v_scale=v_scale, sink_tokens=sink_tokens,
    )


def sample_tokens(
    logits: torch.Tensor,
    uniforms: torch.Tensor,
    *,
    temperature: Optional[torch.Tensor] = None,
    top_k: Optional[torch.Tensor] = None,
    top_p: Optional[torch.Tensor] = None,
    min_p: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """A token drawn from every row of logits, and the log of its probability.

    ``logits`` is bf16 or fp32 ``[rows, vocab]``, ``uniforms`` the fp32 random numbers in
    [0, 1), one a row; so are the fp32 ``temperature``, ``top_p``, ``min_p`` and the int32 or int64 ``top_k``
    (None: 1, 1, 0 and all). With the weights ``exp((l - max l) / temperature)``, kept are the
    ``top_k`` largest (of equal ones the lowest indices; not above 0: all), of those in falling order each before
    which less than ``top_p`` of their mass lies, of those the ones of at least ``min_p``
    (the largest always is). The token is the first in the vocabulary's order at which the kept mass so far
    exceeds ``uniform`` of the whole: the same for the same inputs, whatever else is in the batch.

    A temperature that is not above 0 takes the first largest logit. -infinity and NaN are never
    drawn; a row with nothing to draw gets -1 (and -infinity). Returns int64 tokens and fp32
    log probabilities, ``[rows]`` each.
    """
    return _OPS.sample_tokens(logits, uniforms, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
