from .decoder import add_rms_norm, add_rms_norm_fp8, paged_attention, paged_kv_store, sample_tokens
from .kda import (
    kda_prepared_varlen_chunk,
    kda_prepared_varlen_recurrent,
    kda_varlen_chunk,
    kda_varlen_chunk_v2,
    kda_varlen_chunk_with_state,
    kda_varlen_recurrent,
    kda_varlen_recurrent_v2,
    prepared_recurrent,
)
from .linear import linear_varlen_chunk, linear_varlen_recurrent

__all__ = [
    "add_rms_norm",
    "add_rms_norm_fp8",
    "kda_prepared_varlen_chunk",
    "kda_prepared_varlen_recurrent",
    "kda_varlen_chunk",
    "kda_varlen_chunk_v2",
    "kda_varlen_chunk_with_state",
    "kda_varlen_recurrent",
    "kda_varlen_recurrent_v2",
    "linear_varlen_chunk",
    "linear_varlen_recurrent",
    "paged_attention",
    "paged_kv_store",
    "prepared_recurrent",
    "sample_tokens",
]
