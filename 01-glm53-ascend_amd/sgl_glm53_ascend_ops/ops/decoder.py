"""Keyword wrappers over the norms and the paged attention of a hybrid decoder.

A model that interleaves KDA layers with full attention needs these beside
``ops.kda``: the residual RMS norm in front of every projection (with an 8-bit
output where the projection is an 8-bit product), and for the full-attention
layers a paged key/value cache, its writer and the attention that reads it. The
reference package has no counterpart. Like the KDA operators they enqueue on the
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
    them; ``logit_cap`` > 0 turns a score ``s`` into ``logit_cap * tanh(s /
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
        logit_cap=logit_cap, k_scale=k_scale, v_scale=v_scale,
    )
