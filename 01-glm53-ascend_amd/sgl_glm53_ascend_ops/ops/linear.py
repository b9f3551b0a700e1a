"""Keyword wrappers over linear attention with a decay for each head.

The plain member of the KDA operators' family, for decoders whose linear layers have no delta
rule: per request and head, with the state ``S`` ``[K, V]`` and a log decay ``g_t``,

    S <- exp(g_t) S + k_t v_t^T;    o_t = scale * S^T q_t

on the same slot-indexed fp32 state pool (slot 0: the padding row, a zero state that is never
written), packed sequences, tracked prefixes and checkpoints as ``ops.kda``. The reference package has no
counterpart. Both forms enqueue on the current stream, never synchronize the host and can be
captured in a HIP graph.
"""

from typing import Optional

import torch

from .. import load_library

load_library()
_OPS = torch.ops.sgl_glm53_ascend


def linear_varlen_recurrent(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    g: torch.Tensor,
    *,
    initial_state_source: torch.Tensor,
    initial_state_indices: torch.Tensor,
    cu_seqlens: torch.Tensor,
    scale: float,
    intermediate_state: Optional[torch.Tensor] = None,
    track_state_indices: Optional[torch.Tensor] = None,
    track_state_lens: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Token by token: decode and verify steps, short prompts; states are updated in place.

    ``q, k, v`` are ``[1, T, H, D]`` in bf16 or fp32 (slices of a fused projection work), D 64 or
    128; ``g`` is the fp32 log decay, ``[H]`` or ``[1, T, H]``. Request ``n`` has the tokens
    ``cu_seqlens[n]`` to ``cu_seqlens[n + 1]`` and the state ``initial_state_source[initial_state_indices[n]]``
    (``[slots, H, K, V]``, K contiguous). In one call a slot other than 0 is named once, as a state or as a tracked
    prefix's.

    ``intermediate_state`` ``[requests, steps, H, K, V]`` receives the state after every token, and the
    pool is then left as it is. ``track_state_indices/lens``: the state after ``lens[n]`` tokens of request ``n``
    goes into slot ``indices[n]``. Returns ``o`` in q's dtype, zeros for tokens that no request covers.
    """
    return _OPS.linear_varlen_recurrent(
        q, k, v, g, initial_state_source=initial_state_source, initial_state_indices=initial_state_indices,
        cu_seqlens=cu_seqlens, scale=scale, intermediate_state=intermediate_state,
        track_state_indices=track_state_indices, track_state_lens=track_state_lens,
    )


def linear_varlen_chunk(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    g: torch.Tensor,
    *,
    initial_state_source: torch.Tensor,
    initial_state_indices: torch.Tensor,
    cu_seqlens: torch.Tensor,
    scale: float,
    track_state_indices: Optional[torch.Tensor] = None,
    track_state_lens: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """:func:`linear_varlen_recurrent` for prompts: 64 tokens at a time on the matrix cores, bf16 only.

    Any lengths; log decays from 0 down to -infinity, exact for any steepness (positive ones work while ``exp`` of
    their sum over 64 tokens stays finite). The states are those of a loop
    in fp32 to within its own roundings. An infinite or NaN value reaches its own token and
    later ones of its request only; an infinite one may end as NaN where the recurrent form keeps it.
    """
    return _OPS.linear_varlen_chunk(
        q, k, v, g, initial_state_source=initial_state_source, initial_state_indices=initial_state_indices,
        cu_seqlens=cu_seqlens, scale=scale, track_state_indices=track_state_indices,
        track_state_lens=track_state_lens,
    )
