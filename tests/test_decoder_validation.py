"""Refusals of the norms, the paged store and the paged attention, on the CPU.

Like the KDA operators these are registered for host tensors too, so every rule
can be checked here; a valid host call then fails on the device check. The C
launchers' own checks return before any device call (their addresses are never
dereferenced).
"""

import ctypes
import re
from pathlib import Path

import pytest
import torch

from sgl_glm53_ascend_ops._load import abi_library_path
from sgl_glm53_ascend_ops.ops import add_rms_norm, add_rms_norm_fp8, paged_attention, paged_kv_store
from tests import decoder_cases as C

BF16, F32 = torch.bfloat16, torch.float32


def _refused(match, call, *args, **kwargs):
    with pytest.raises(RuntimeError, match=match):
        call(*args, **kwargs)


# ---------------------------------------------------------------------------
# torch operators
# ---------------------------------------------------------------------------

def test_valid_host_calls_fail_on_the_device_check():
    case = C.Attention(0, [1, 3], [5, 9], 4, 2, 64, 16)
    _refused("must be a CUDA", paged_attention, case.q, **case.kwargs("cpu"))
    k = torch.zeros(1, 2, 2, 64, dtype=BF16)
    _refused("must be a CUDA", paged_kv_store, k, k, k_cache=case.k_cache, v_cache=case.v_cache,
             slot_indices=torch.zeros(2, dtype=torch.int32))
    x = torch.zeros(2, 8)
    _refused("must be a CUDA", add_rms_norm, x, torch.ones(8), 1e-6, residual=x.clone())
    _refused("must be a CUDA", add_rms_norm_fp8, x, torch.ones(8), 1e-6, group_size=128)


def test_norm_refusals():
    x, w = torch.zeros(4, 16), torch.ones(16)
    for call in (add_rms_norm, add_rms_norm_fp8):
        _refused("x must be bf16 or fp32", call, x.half(), w, 1e-6)
        _refused("weight must be bf16 or fp32", call, x, w.half(), 1e-6)
        _refused("contiguous weight of the width", call, x, torch.ones(15), 1e-6)
        _refused("contiguous weight of the width", call, x, torch.ones(32)[::2], 1e-6)
        _refused("expects x as", call, torch.zeros(4, 0), torch.ones(0), 1e-6)
        _refused("contiguous in its last dimension", call, torch.zeros(16, 4).t(), w, 1e-6)
        _refused("rows at one stride", call, torch.zeros(2, 3, 3, 2, 16)[:, :2, :2, :1], w, 1e-6)
        _refused("rows at one stride", call, torch.zeros(2, 2, 16), w, 1e-6, residual=torch.zeros(2, 3, 16)[:, :2])
        _refused("rows at one stride", call, torch.zeros(2, 3, 16), w, 1e-6, residual=torch.zeros(2, 1, 16).expand(2, 3, 16))
        _refused("residual in x's shape", call, x, w, 1e-6, residual=torch.zeros(3, 16))
        _refused("residual must be bf16 or fp32", call, x, w, 1e-6, residual=x.half())
        _refused("must not overlap", call, x, w, 1e-6, residual=torch.zeros(1, 16).expand(4, 16))
    _refused("group_size 0", add_rms_norm_fp8, x, w, 1e-6, group_size=64)


@pytest.mark.parametrize("shape", [(2, 0, 64), (0, 3, 64), (0, 64), (3, 2, 0, 64)])
def test_norm_takes_an_empty_residual(shape):
    """No rows, whatever strides torch gives their dimensions: the call gets as far as the device check."""
    x, w = torch.zeros(shape), torch.ones(64)
    for call in (add_rms_norm, add_rms_norm_fp8):
        _refused("must be a CUDA", call, x, w, 1e-6)
        _refused("must be a CUDA", call, x, w, 1e-6, residual=x.clone())


def _store(**over):
    a = dict(k=torch.zeros(1, 3, 2, 64, dtype=BF16), v=torch.zeros(1, 3, 2, 64, dtype=BF16),
             k_cache=torch.zeros(4, 8, 2, 64, dtype=BF16), v_cache=torch.zeros(4, 8, 2, 64, dtype=BF16),
             slot_indices=torch.zeros(3, dtype=torch.int32))
    a.update(over)
    return a.pop("k"), a.pop("v"), a


def test_store_refusals():
    for match, over in [
        ("as one packed token batch", dict(k=torch.zeros(2, 3, 2, 64, dtype=BF16))),
        ("as one packed token batch", dict(k=torch.zeros(1, 3, 2, 128, dtype=BF16))),
        ("k must be bf16", dict(k=torch.zeros(1, 3, 2, 64))),
        ("v must be bf16", dict(v=torch.zeros(1, 3, 2, 64))),
        ("with the cache's kv_heads", dict(k=torch.zeros(1, 3, 4, 64, dtype=BF16), v=torch.zeros(1, 3, 4, 64, dtype=BF16))),
        ("with the cache's kv_heads", dict(v=torch.zeros(1, 2, 2, 64, dtype=BF16))),
        ("v must be contiguous in D", dict(v=torch.zeros(1, 3, 64, 2, dtype=BF16).transpose(2, 3))),
        ("an entry per token", dict(slot_indices=torch.zeros(2, dtype=torch.int32))),
        ("must be int32 or int64", dict(slot_indices=torch.zeros(3))),
        ("contiguous in its last dimension", dict(slot_indices=torch.zeros(6, dtype=torch.int32)[::2])),
    ]:
        k, v, kw = _store(**over)
        _refused(match, paged_kv_store, k, v, **kw)


CACHE_REFUSALS = [
    ("as \\[pages, page_size, kv_heads, D\\]", lambda c: dict(v_cache=c[:3])),
    ("as \\[pages, page_size, kv_heads, D\\]", lambda c: dict(k_cache=c[0], v_cache=c[0])),
    ("both be bf16 or both float8_e4m3fn", lambda c: dict(k_cache=c.float(), v_cache=c.float())),
    ("both be bf16 or both float8_e4m3fn", lambda c: dict(k_cache=c.to(C.FP8))),
    ("requires D in", lambda c: dict(k_cache=c[..., :32], v_cache=c[..., :32])),
    ("pages of at least one token", lambda c: dict(k_cache=c[:, :0], v_cache=c[:, :0])),
    ("k_cache must be contiguous in D", lambda c: dict(k_cache=torch.zeros(4, 16, 2, 128, dtype=BF16)[..., ::2])),
    ("rows of v_cache must be 16-byte aligned", lambda c: dict(v_cache=torch.zeros(4, 16, 2, 72, dtype=BF16)[..., 1:65])),
    ("rows of v_cache must be 16-byte aligned", lambda c: dict(v_cache=torch.zeros(4, 16, 2, 68, dtype=BF16)[..., :64])),
    ("belongs to a float8_e4m3fn cache", lambda c: dict(k_scale=torch.ones(2))),
    ("an entry per kv head", lambda c: dict(k_cache=c.to(C.FP8), v_cache=c.to(C.FP8), v_scale=torch.ones(3))),
    ("an entry per kv head", lambda c: dict(k_cache=c.to(C.FP8), v_cache=c.to(C.FP8), k_scale=torch.ones(2).double())),
]


@pytest.mark.parametrize("match,change", CACHE_REFUSALS)
def test_cache_refusals(match, change):
    cache = torch.zeros(4, 16, 2, 64, dtype=BF16)
    k, v, kw = _store(k_cache=cache, v_cache=cache, **{})
    kw.update(change(cache))
    _refused(match, paged_kv_store, k, v, **kw)
    case = C.Attention(0, [1, 3], [5, 9], 4, 2, 64, 16)
    kw = case.kwargs("cpu")
    kw.update(dict(k_cache=cache, v_cache=cache))
    kw.update(change(cache))
    _refused(match, paged_attention, case.q, **kw)


@pytest.mark.parametrize("pages,page_size,kv_heads", [(4, 16, 1), (4, 1, 2), (1, 16, 2), (1, 1, 1)])
def test_strides_of_single_pages_tokens_and_heads_do_not_matter(pages, page_size, kv_heads):
    """A stride that nothing is multiplied by is any number: torch calls such a cache contiguous."""
    sizes = (pages, page_size, kv_heads, 64)
    whole = torch.zeros(sizes, dtype=BF16)
    cache = whole.as_strided(sizes, [s if n > 1 else 3 for n, s in zip(sizes, whole.stride())])
    assert cache.is_contiguous() and 3 in cache.stride()
    k = torch.zeros(1, 2, kv_heads, 64, dtype=BF16)
    _refused("must be a CUDA", paged_kv_store, k, k, k_cache=cache, v_cache=cache, slot_indices=torch.zeros(2, dtype=torch.int32))
    case = C.Attention(0, [1, 1], [1, 1], 2, kv_heads, 64, page_size)
    _refused("must be a CUDA", paged_attention, case.q, **case.kwargs("cpu", k_cache=cache, v_cache=cache))


@pytest.mark.parametrize("match,over", [
    ("multiple of kv_heads", dict(q=torch.zeros(1, 4, 3, 64, dtype=BF16))),
    ("as one packed token batch", dict(q=torch.zeros(4, 4, 64, dtype=BF16))),
    ("q must be bf16", dict(q=torch.zeros(1, 4, 4, 64))),
    ("numReq\\+1 entries", dict(cu_seqlens=torch.zeros(2, dtype=torch.int32))),
    ("a row per request", dict(page_table=torch.zeros(3, 1, dtype=torch.int32))),
    ("page_table with 2 dimensions", dict(page_table=torch.zeros(2, dtype=torch.int32))),
    ("kv_lens must be int32 or int64", dict(kv_lens=torch.zeros(2))),
    ("page_table must be contiguous in its last", dict(page_table=torch.zeros(3, 2, dtype=torch.int32).t())),
    ("window must be", dict(window=-1)),
    ("logit_cap must be", dict(logit_cap=-1.0)),
    ("logit_cap must be", dict(logit_cap=float("nan"))),
    ("logit_cap must be", dict(logit_cap=float("inf"))),
    ("logit_cap must be", dict(logit_cap=1e-40)),
    ("at most 2\\^31-1", dict(max_query_len=-1)),
])
def test_attention_refusals(match, over):
    case = C.Attention(0, [1, 3], [5, 9], 4, 2, 64, 16)
    kw = case.kwargs("cpu")
    kw.update(over)
    q = kw.pop("q", case.q)
    _refused(match, paged_attention, q, **kw)


# ---------------------------------------------------------------------------
# C ABI
# ---------------------------------------------------------------------------

P, I64, I32, F = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32, ctypes.c_float


class NormArgs(ctypes.Structure):
    _fields_ = [("x", P), ("residual", P), ("weight", P), ("out", P), ("scale", P), ("x_stride", I64),
                ("residual_stride", I64), ("out_stride", I64), ("rows", I64), ("width", I32), ("eps", F),
                ("x_dtype", I32), ("residual_dtype", I32), ("weight_dtype", I32), ("out_dtype", I32), ("group", I32),
                ("x_inner", I32), ("x_outer_stride", I64)]


class Cache(ctypes.Structure):
    _fields_ = [("k", P), ("v", P), ("k_stride_page", I64), ("k_stride_token", I64), ("k_stride_head", I64),
                ("v_stride_page", I64), ("v_stride_token", I64), ("v_stride_head", I64), ("k_scale", P), ("v_scale", P),
                ("num_pages", I64), ("page_size", I32), ("kv_heads", I32), ("head_dim", I32), ("dtype", I32)]


class StoreArgs(ctypes.Structure):
    _fields_ = [("k", P), ("v", P), ("k_stride_token", I64), ("k_stride_head", I64), ("v_stride_token", I64),
                ("v_stride_head", I64), ("slots", P), ("slots_int64", I32), ("num_tokens", I32), ("cache", Cache)]


class AttentionArgs(ctypes.Structure):
    _fields_ = [("q", P), ("out", P), ("q_stride_token", I64), ("q_stride_head", I64), ("out_stride_token", I64),
                ("out_stride_head", I64), ("page_table", P), ("page_table_stride", I64), ("kv_lens", P), ("cu_seqlens", P),
                ("scale", F), ("logit_cap", F), ("window", I32), ("wide", I32), ("num_seqs", I32), ("num_tokens", I32),
                ("num_heads", I32), ("max_pages", I32), ("max_query_len", I32), ("cache", Cache)]


OK, INVALID, UNSUPPORTED, WORKSPACE, TOO_LARGE = 0, 1, 2, 4, 5
BASE = 1 << 20


@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(str(abi_library_path()))
    lib.kda_rms_norm_launch.argtypes = [ctypes.POINTER(NormArgs), P]
    lib.kda_paged_store_launch.argtypes = [ctypes.POINTER(StoreArgs), P]
    lib.kda_paged_attention_launch.argtypes = [ctypes.POINTER(AttentionArgs), P, ctypes.c_size_t, P]
    lib.kda_paged_attention_workspace_bytes.argtypes = [ctypes.POINTER(AttentionArgs)]
    lib.kda_paged_attention_workspace_bytes.restype = ctypes.c_size_t
    return lib


def test_norm_launch_refusals(lib):
    def status(**over):
        a = dict(x=BASE, weight=BASE, out=BASE, x_stride=64, out_stride=64, rows=4, width=64, eps=1e-6)
        a.update(over)
        return lib.kda_rms_norm_launch(ctypes.byref(NormArgs(**a)), None)

    assert lib.kda_rms_norm_launch(None, None) == INVALID
    assert status(rows=0, x=None) == OK
    for over in (dict(rows=-1), dict(width=0), dict(x=None), dict(weight=None), dict(out=None), dict(x=BASE + 1),
                 dict(out_stride=63), dict(residual=BASE, residual_stride=63), dict(out_dtype=2),
                 dict(out_dtype=2, scale=BASE + 2), dict(x_dtype=1, out_dtype=1, x=BASE + 2)):
        assert status(**over) == INVALID, over
    for over in (dict(x_dtype=2), dict(weight_dtype=3), dict(out_dtype=1), dict(group=128), dict(out_dtype=2, scale=BASE, group=64),
                 dict(residual=BASE, residual_dtype=2, residual_stride=64)):
        assert status(**over) == UNSUPPORTED, over


def _cache(**over):
    a = dict(k=BASE, v=BASE, k_stride_page=2048, k_stride_token=128, k_stride_head=64, v_stride_page=2048,
             v_stride_token=128, v_stride_head=64, num_pages=8, page_size=16, kv_heads=2, head_dim=64, dtype=0)
    a.update(over)
    return Cache(**a)


@pytest.mark.parametrize("over,expected", [
    (dict(head_dim=96), UNSUPPORTED), (dict(dtype=1), UNSUPPORTED), (dict(page_size=0), INVALID),
    (dict(kv_heads=0), INVALID), (dict(num_pages=-1), INVALID), (dict(num_pages=1 << 27), INVALID), (dict(k=None), INVALID),
    (dict(v=BASE + 8), INVALID), (dict(k_stride_token=4), INVALID), (dict(dtype=2, v_stride_head=72), INVALID),
    (dict(k_scale=BASE), INVALID), (dict(dtype=2, k_scale=BASE + 2), INVALID)])
def test_cache_launch_refusals(lib, over, expected):
    store = StoreArgs(k=BASE, v=BASE, slots=BASE, num_tokens=1, cache=_cache(**over))
    assert lib.kda_paged_store_launch(ctypes.byref(store), None) == expected
    attention = AttentionArgs(q=BASE, out=BASE, page_table=BASE, kv_lens=BASE, cu_seqlens=BASE, num_seqs=1, num_tokens=1,
                              num_heads=4, max_pages=1, max_query_len=1, cache=_cache(**over))
    assert lib.kda_paged_attention_launch(ctypes.byref(attention), BASE, 1 << 30, None) == expected


def test_store_launch_refusals(lib):
    def status(**over):
        a = dict(k=BASE, v=BASE, slots=BASE, num_tokens=1, cache=_cache())
        a.update(over)
        return lib.kda_paged_store_launch(ctypes.byref(StoreArgs(**a)), None)

    assert lib.kda_paged_store_launch(None, None) == INVALID
    assert status(num_tokens=0, k=None) == OK and status(cache=_cache(num_pages=0, k=None)) == OK
    for over in (dict(num_tokens=-1), dict(k=None), dict(v=None), dict(slots=None), dict(k=BASE + 1),
                 dict(slots=BASE + 2), dict(slots=BASE + 4, slots_int64=1)):
        assert status(**over) == INVALID, over


def test_attention_launch_refusals(lib):
    def args(**over):
        a = dict(q=BASE, out=BASE, page_table=BASE, kv_lens=BASE, cu_seqlens=BASE, num_seqs=1, num_tokens=1, num_heads=4,
                 max_pages=64, max_query_len=1, cache=_cache())
        a.update(over)
        return ctypes.byref(AttentionArgs(**a))

    def status(**over):
        return lib.kda_paged_attention_launch(args(**over), BASE, 1 << 30, None)

    assert lib.kda_paged_attention_launch(None, None, 0, None) == INVALID
    assert lib.kda_paged_attention_workspace_bytes(None) == 0
    assert status(num_tokens=0, q=None) == OK
    for over in (dict(q=None), dict(out=BASE + 1), dict(cu_seqlens=None), dict(kv_lens=None), dict(page_table=None),
                 dict(kv_lens=BASE + 2), dict(kv_lens=BASE + 4, wide=32), dict(wide=2), dict(num_heads=5), dict(num_heads=0),
                 dict(window=-1), dict(logit_cap=-1.0), dict(logit_cap=float("nan")), dict(max_pages=-1), dict(num_seqs=-1)):
        assert status(**over) == INVALID, over
    # row numbers, keys and the grid stay in 32 bits
    assert status(num_tokens=1 << 30) == TOO_LARGE and status(max_pages=(1 << 27) - 1) == TOO_LARGE
    assert status(num_tokens=1 << 29, num_seqs=1 << 23, max_query_len=1000) == TOO_LARGE
    need = lib.kda_paged_attention_workspace_bytes(args())
    assert need > 0
    for ws, size in ((None, need), (BASE, need - 1), (BASE + 128, need)):
        assert lib.kda_paged_attention_launch(args(), ws, size, None) == WORKSPACE


@pytest.mark.parametrize("max_query_len,num_tokens", [(1, 7), (300, 300)])
@pytest.mark.parametrize("dtype", [0, 2])
def test_attention_workspace_follows_from_the_sizes_alone(lib, max_query_len, num_tokens, dtype):
    """The query may come before there is anything to point at."""
    sizes = dict(num_seqs=7, num_tokens=num_tokens, num_heads=4, max_pages=640, max_query_len=max_query_len)
    pool = dict(num_pages=999, page_size=16, kv_heads=2, head_dim=64, dtype=dtype)
    bare = lib.kda_paged_attention_workspace_bytes(ctypes.byref(AttentionArgs(cache=Cache(**pool), **sizes)))
    full = AttentionArgs(q=BASE, out=BASE, page_table=BASE, kv_lens=BASE, cu_seqlens=BASE, window=5, logit_cap=2.0, wide=48,
                         cache=_cache(**pool), **sizes)
    assert bare == lib.kda_paged_attention_workspace_bytes(ctypes.byref(full)) > 0
    odd = AttentionArgs(q=BASE + 1, window=-1, logit_cap=-1.0, wide=1,
                        cache=_cache(k=BASE + 1, v=None, k_stride_token=3, v_stride_page=1, k_scale=1, **pool), **sizes)
    assert bare == lib.kda_paged_attention_workspace_bytes(ctypes.byref(odd))
    assert lib.kda_paged_attention_launch(ctypes.byref(odd), BASE, bare, None) == INVALID
    for wrong in (dict(num_heads=5), dict(num_tokens=0), dict(num_seqs=-1)):
        args = AttentionArgs(cache=Cache(**pool), **dict(sizes, **wrong))
        assert lib.kda_paged_attention_workspace_bytes(ctypes.byref(args)) == 0


def test_too_large_names_every_reason(lib):
    """The norms and the attention refuse sizes past their counts with the status that the static buffer has."""
    lib.kda_status_string.restype = ctypes.c_char_p
    text = lib.kda_status_string(TOO_LARGE)
    for reason in (b"sizes", b"rows", b"keys", b"workgroups", b"kda_chunk_launch_noalloc"):
        assert reason in text, text


# ---------------------------------------------------------------------------
# kernel sources
# ---------------------------------------------------------------------------

def test_asm_that_writes_m0_says_so():
    """A register that an asm statement writes and does not name is one the compiler may keep a value in across it."""
    csrc = Path(__file__).resolve().parent.parent / "01-glm53-ascend_amd" / "csrc"
    found = 0
    for source in sorted(csrc.glob("*.h*")):
        for statement in re.findall(r"\basm\b[^;]*?\((.*?)\);", source.read_text(), re.S):
            if re.search(r"\bs_mov_b32 m0\b", statement):
                found += 1
                clobbers = statement.rsplit(":", 1)[1]
                assert '"m0"' in clobbers and '"memory"' in clobbers, (source.name, statement)
    assert found > 0
