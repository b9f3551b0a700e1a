"""Refusals of linear attention, of attention with sinks and of sampling, on the CPU.

As for the other operators: every rule holds for host tensors too, a valid host call then fails on the
device check, and the C launchers' own checks return before any device call.
"""

import ctypes

import pytest
import torch

from sgl_glm53_ascend_ops._load import abi_library_path
from sgl_glm53_ascend_ops.ops import linear_varlen_chunk, linear_varlen_recurrent, paged_attention, sample_tokens
from tests import decoder_cases as C
from tests.linear_cases import Linear
from tests.test_decoder_validation import AttentionArgs, _cache

BF16 = torch.bfloat16
I32 = torch.int32


def _refused(match, call, *args, **kwargs):
    with pytest.raises(RuntimeError, match=match):
        call(*args, **kwargs)


# ---------------------------------------------------------------------------
# linear attention
# ---------------------------------------------------------------------------

BOTH = [linear_varlen_recurrent, linear_varlen_chunk]


@pytest.mark.parametrize("call", BOTH)
@pytest.mark.parametrize("gated,fused", [(True, False), (False, True)])
def test_valid_host_calls_fail_on_the_device_check(call, gated, fused):
    (q, k, v, g), args = Linear(0, [3, 2], 2, 64, gated=gated, fused=fused, track=[1, 2]).on("cpu")
    _refused("must be a CUDA", call, q, k, v, g, **args)


@pytest.mark.parametrize("call", BOTH)
@pytest.mark.parametrize("match,over", [
    ("expects q, k, v as", dict(q=torch.zeros(5, 2, 64, dtype=BF16))),
    ("one packed token batch", dict(q=torch.zeros(2, 5, 2, 64, dtype=BF16))),
    ("q must be bf16 or fp32", dict(q=torch.zeros(1, 5, 2, 64, dtype=torch.float16))),
    ("k must have q's dtype", dict(k=torch.zeros(1, 5, 2, 64))),
    ("expects q, k, v all", dict(v=torch.zeros(1, 5, 2, 128, dtype=BF16))),
    ("expects q, k, v all", dict(k=torch.zeros(1, 5, 1, 64, dtype=BF16))),
    ("v must be contiguous in D", dict(v=torch.zeros(1, 5, 64, 2, dtype=BF16).transpose(2, 3))),
    ("rows of q must be 16-byte aligned", dict(q=torch.zeros(1, 5, 2, 68, dtype=BF16)[..., :64])),
    ("rows of k must be 16-byte aligned", dict(k=torch.zeros(5 * 2 * 64 + 1, dtype=BF16)[1:].view(1, 5, 2, 64))),
    ("g must be fp32", dict(g=torch.zeros(1, 5, 2, dtype=torch.float64))),
    ("expects g as", dict(g=torch.zeros(1, 5, 2, 64))),
    ("expects g as", dict(g=torch.zeros(3))),
    ("expects g as", dict(g=torch.zeros(5, 2))),
    ("state must be a 4-D fp32", dict(initial_state_source=torch.zeros(5, 2, 64, 64, dtype=BF16))),
    ("matching the head", dict(initial_state_source=torch.zeros(5, 3, 64, 64).transpose(2, 3))),
    ("K-contiguous", dict(initial_state_source=torch.zeros(5, 2, 64, 64))),
    ("rows of state must be 16-byte aligned", dict(initial_state_source=torch.zeros(5 * 8192 + 1)[1:].view(5, 2, 64, 64).transpose(2, 3))),
    ("initial_state_indices must be int32 or int64", dict(initial_state_indices=torch.zeros(2))),
    ("numReq\\+1 entries", dict(cu_seqlens=torch.zeros(2, dtype=I32))),
    ("requires track_state_lens", dict(track_state_indices=torch.zeros(2, dtype=I32))),
    ("one entry per request", dict(track_state_indices=torch.zeros(3, dtype=I32), track_state_lens=torch.zeros(2, dtype=I32))),
])
def test_linear_refusals(call, match, over):
    (q, k, v, g), args = Linear(0, [3, 2], 2, 64).on("cpu")
    args.update(q=q, k=k, v=v, g=g)
    args.update(over)
    _refused(match, call, *[args.pop(x) for x in ("q", "k", "v", "g")], **args)


def test_linear_heads_dims_and_types():
    (q, k, v, g), args = Linear(0, [3], 2, 64).on("cpu")
    wide = torch.zeros(1, 3, 2, 96, dtype=BF16)
    _refused("requires K == V in", linear_varlen_chunk, wide, wide, wide, g, **args)
    none = torch.zeros(1, 3, 0, 64, dtype=BF16)
    _refused("heads", linear_varlen_recurrent, none, none, none, torch.zeros(1, 3, 0), **args)
    (q, k, v, g), args = Linear(0, [3], 2, 64, fp32=True).on("cpu")
    _refused("takes bf16 q, k, v", linear_varlen_chunk, q, k, v, g, **args)
    _refused("must be a CUDA", linear_varlen_recurrent, q, k, v, g, **args)
    # tokens and heads of a single one may have any stride
    (q, k, v, g), args = Linear(0, [1], 1, 64).on("cpu")
    q = q.as_strided((1, 1, 1, 64), (3, 5, 7, 1))
    _refused("must be a CUDA", linear_varlen_chunk, q, k, v, g, **args)


@pytest.mark.parametrize("match,middle", [
    ("5-D fp32", torch.zeros(2, 3, 2, 64, 64, dtype=BF16)),
    ("matching the head", torch.zeros(2, 3, 1, 64, 64).transpose(3, 4)),
    ("K-contiguous", torch.zeros(2, 3, 2, 64, 64)),
    ("a row per request", torch.zeros(1, 5, 2, 64, 64).transpose(3, 4)),
    ("too few for 5 tokens", torch.zeros(2, 2, 2, 64, 64).transpose(3, 4)),
    ("16-byte aligned", torch.zeros(2 * 3 * 8192 + 1)[1:].view(2, 3, 2, 64, 64).transpose(3, 4)),
])
def test_checkpoint_refusals(match, middle):
    (q, k, v, g), args = Linear(0, [3, 2], 2, 64).on("cpu")
    _refused(match, linear_varlen_recurrent, q, k, v, g, intermediate_state=middle, **args)


# ---------------------------------------------------------------------------
# sinks, sampling
# ---------------------------------------------------------------------------

def test_sink_refusals():
    case = C.Attention(0, [1, 3], [5, 9], 4, 2, 64, 16, window=3)
    for sinks in (-1, 1 << 31):
        _refused("sink_tokens must be", paged_attention, case.q, **case.kwargs("cpu", sink_tokens=sinks))
    _refused("must be a CUDA", paged_attention, case.q, **case.kwargs("cpu", sink_tokens=4))


@pytest.mark.parametrize("match,over", [
    ("expects logits as", dict(logits=torch.zeros(8))),
    ("expects logits as", dict(logits=torch.zeros(3, 0))),
    ("logits must be bf16 or fp32", dict(logits=torch.zeros(3, 8, dtype=torch.float16))),
    ("contiguous in the vocabulary", dict(logits=torch.zeros(8, 3).t())),
    ("uniforms must be contiguous with an entry per row", dict(uniforms=torch.zeros(2))),
    ("uniforms must be contiguous with an entry per row", dict(uniforms=torch.zeros(6)[::2])),
    ("uniforms must be fp32", dict(uniforms=torch.zeros(3, dtype=torch.float64))),
    ("temperature must be fp32", dict(temperature=torch.zeros(3, dtype=BF16))),
    ("temperature must be contiguous with an entry", dict(temperature=torch.zeros(1))),
    ("top_k must be int32 or int64", dict(top_k=torch.zeros(3))),
    ("top_k must be contiguous with an entry", dict(top_k=torch.zeros(3, 1, dtype=I32))),
    ("top_p must be fp32", dict(top_p=torch.zeros(3, dtype=I32))),
    ("min_p must be contiguous with an entry", dict(min_p=torch.zeros(4))),
    ("must be a CUDA", dict()),
    ("must be a CUDA", dict(logits=torch.zeros(3, 1).expand(3, 8)[:, :1], top_k=torch.zeros(3, dtype=torch.int64))),
])
def test_sampling_refusals(match, over):
    args = dict(logits=torch.zeros(3, 8), uniforms=torch.zeros(3))
    args.update(over)
    _refused(match, sample_tokens, args.pop("logits"), args.pop("uniforms"), **args)


# ---------------------------------------------------------------------------
# C ABI
# ---------------------------------------------------------------------------

P, L, N, F = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32, ctypes.c_float
OK, INVALID, UNSUPPORTED, WORKSPACE, TOO_LARGE = 0, 1, 2, 4, 5
BASE = 1 << 20


class LinearArgs(ctypes.Structure):
    _fields_ = [("q", P), ("k", P), ("v", P), ("q_stride_token", L), ("q_stride_head", L), ("k_stride_token", L),
                ("k_stride_head", L), ("v_stride_token", L), ("v_stride_head", L), ("g", P), ("g_stride_token", L),
                ("g_stride_head", L), ("state", P), ("state_stride_slot", L), ("state_stride_head", L), ("num_slots", L),
                ("state_indices", P), ("cu_seqlens", P), ("out", P), ("intermediate", P), ("mid_stride_req", L),
                ("mid_stride_step", L), ("mid_stride_head", L), ("mid_rows", L), ("mid_steps", L), ("track_indices", P),
                ("track_lens", P), ("scale", F), ("num_seqs", N), ("num_tokens", N), ("num_heads", N), ("head_dim", N),
                ("dtype", N), ("wide", N)]


class SampleArgs(ctypes.Structure):
    _fields_ = [("logits", P), ("logits_stride", L), ("uniforms", P), ("temperature", P), ("top_k", P), ("top_p", P),
                ("min_p", P), ("tokens", P), ("logprobs", P), ("rows", L), ("vocab", N), ("dtype", N), ("top_k_int64", N)]


@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(str(abi_library_path()))
    lib.kda_linear_recurrent_launch.argtypes = [ctypes.POINTER(LinearArgs), P]
    lib.kda_linear_chunk_launch.argtypes = [ctypes.POINTER(LinearArgs), P, ctypes.c_size_t, P]
    lib.kda_linear_chunk_workspace_bytes.argtypes = [ctypes.POINTER(LinearArgs)]
    lib.kda_linear_chunk_workspace_bytes.restype = ctypes.c_size_t
    lib.kda_sample_launch.argtypes = [ctypes.POINTER(SampleArgs), P]
    lib.kda_paged_attention_launch_sinks.argtypes = [ctypes.POINTER(AttentionArgs), N, P, ctypes.c_size_t, P]
    return lib


def _linear(**over):
    a = dict(q=BASE, k=BASE, v=BASE, q_stride_token=128, q_stride_head=64, k_stride_token=128, k_stride_head=64,
             v_stride_token=128, v_stride_head=64, g=BASE, g_stride_token=2, g_stride_head=1, state=BASE,
             state_stride_slot=8192, state_stride_head=4096, num_slots=3, state_indices=BASE, cu_seqlens=BASE, out=BASE,
             scale=1.0, num_seqs=2, num_tokens=5, num_heads=2, head_dim=64, dtype=0)
    a.update(over)
    return ctypes.byref(LinearArgs(**a))


def test_linear_launch_refusals(lib):
    forms = [lambda **over: lib.kda_linear_recurrent_launch(_linear(**over), None),
             lambda **over: lib.kda_linear_chunk_launch(_linear(**over), BASE, 1 << 40, None)]
    assert lib.kda_linear_recurrent_launch(None, None) == INVALID
    assert lib.kda_linear_chunk_launch(None, None, 0, None) == INVALID
    assert lib.kda_linear_chunk_workspace_bytes(None) == 0
    for status in forms:
        assert status(num_seqs=0, num_tokens=0, q=None, state=None) == OK
        for over in (dict(q=None), dict(k=BASE + 8), dict(out=None), dict(g=None), dict(g=BASE + 2), dict(q_stride_token=4),
                     dict(v_stride_head=2), dict(cu_seqlens=None), dict(cu_seqlens=BASE + 4, wide=1), dict(state_indices=None),
                     dict(state_indices=BASE + 4, wide=2), dict(state=None), dict(state=BASE + 4), dict(state_stride_slot=2),
                     dict(state_stride_head=1), dict(num_slots=-1), dict(track_indices=BASE), dict(wide=16), dict(wide=-1),
                     dict(track_indices=BASE, track_lens=BASE + 2), dict(num_heads=0), dict(num_heads=(1 << 20) + 1),
                     dict(num_seqs=-1), dict(num_tokens=-1), dict(num_seqs=0)):
            assert status(**over) == INVALID, over
        for over in (dict(head_dim=96), dict(dtype=2)):
            assert status(**over) == UNSUPPORTED, over
        # a grid counts its threads in 32 bits
        assert status(num_seqs=1 << 24, num_heads=64) == TOO_LARGE
    assert forms[0](intermediate=BASE + 4) == INVALID and forms[0](intermediate=BASE, mid_stride_step=2) == INVALID
    assert forms[0](dtype=1, q_stride_token=2) == INVALID
    assert forms[1](dtype=1) == UNSUPPORTED and forms[1](intermediate=BASE) == UNSUPPORTED


def test_linear_chunk_workspace(lib):
    """It follows from the sizes alone, grows with no more than the segments, and is asked for."""
    size = lambda **over: lib.kda_linear_chunk_workspace_bytes(_linear(**over))  # noqa: E731
    assert size(num_tokens=320) == 0 and size(num_tokens=0) == 0 and size(num_tokens=4000, num_seqs=0) == 0
    need = size(num_tokens=4000)
    assert need > 0 and need == size(num_tokens=4000, q=None, g=None, wide=3, state=None)
    for D in (64, 128):  # at most about twice as many states as workgroups at once, whatever the length
        for T, H in ((1 << 20, 1), (8192, 32), (1 << 24, 64), (400, 4), (2000, 200)):
            assert size(num_tokens=T, num_heads=H, head_dim=D, num_seqs=1) <= (2 * 1536 + 3 * H) * (D * D + 1) * 4 + 256
    for ws, given in ((None, need), (BASE, need - 1), (BASE + 128, need)):
        assert lib.kda_linear_chunk_launch(_linear(num_tokens=4000), ws, given, None) == WORKSPACE
    assert size(head_dim=80, num_tokens=4000) == 0


def test_linear_chunk_most_tokens(lib):
    """Offsets a segment (2^26 tokens at most) behind the last token would pass 32 bits."""
    for tokens in ((1 << 31) - 1, (1 << 31) - (1 << 26)):
        assert lib.kda_linear_chunk_launch(_linear(num_tokens=tokens, num_heads=1), BASE, 1 << 60, None) == TOO_LARGE


def test_sample_launch_refusals(lib):
    def status(**over):
        a = dict(logits=BASE, logits_stride=100, uniforms=BASE, tokens=BASE, logprobs=BASE, rows=2, vocab=100)
        a.update(over)
        return lib.kda_sample_launch(ctypes.byref(SampleArgs(**a)), None)

    assert lib.kda_sample_launch(None, None) == INVALID
    assert status(rows=0, logits=None) == OK
    for over in (dict(rows=-1), dict(vocab=0), dict(vocab=-5), dict(logits=None), dict(logits=BASE + 1), dict(logits=BASE + 2, dtype=1),
                 dict(uniforms=None), dict(uniforms=BASE + 2), dict(temperature=BASE + 1), dict(top_p=BASE + 2), dict(min_p=BASE + 3),
                 dict(top_k=BASE + 2), dict(top_k=BASE + 4, top_k_int64=1), dict(tokens=None), dict(tokens=BASE + 4),
                 dict(logprobs=None), dict(logprobs=BASE + 2)):
        assert status(**over) == INVALID, over
    assert status(dtype=2) == UNSUPPORTED
    assert status(vocab=(1 << 31) - 1) == TOO_LARGE and status(rows=1 << 22) == TOO_LARGE


def test_sinks_launch_refusals(lib):
    args = ctypes.byref(AttentionArgs(q=BASE, out=BASE, page_table=BASE, kv_lens=BASE, cu_seqlens=BASE, num_seqs=1, num_tokens=1,
                                      num_heads=4, max_pages=64, max_query_len=1, window=5, cache=_cache()))
    assert lib.kda_paged_attention_launch_sinks(None, 0, None, 0, None) == INVALID
    assert lib.kda_paged_attention_launch_sinks(args, -1, BASE, 1 << 30, None) == INVALID
    assert lib.kda_paged_attention_launch_sinks(args, 4, None, 0, None) == WORKSPACE
