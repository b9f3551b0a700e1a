"""Norms, paged store and paged attention on the GPU against their definitions in 64 bits."""

import random

import pytest
import torch

from tests import decoder_cases as C

pytestmark = pytest.mark.gpu

DEV = "cuda"
EPS = 1e-6
ROUND = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


@pytest.fixture(scope="module")
def ops(gpu_ops):
    from sgl_glm53_ascend_ops import ops as package

    return package


# ---------------------------------------------------------------------------
# norms
# ---------------------------------------------------------------------------

def _norm_inputs(rows, width, dtype, residual, weight_dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, width, generator=gen).to(dtype)
    r = None if residual is None else (torch.randn(rows, width, generator=gen) * 3).to(residual)
    w = (1 + 0.3 * torch.randn(width, generator=gen)).to(weight_dtype)
    return x, r, w


def _check_norm(ops, x, r, w, group, x_dev=None, r_dev=None):
    """add_rms_norm (group None) or add_rms_norm_fp8 of the CPU inputs, on views of them if given."""
    x_dev = x.to(DEV) if x_dev is None else x_dev
    if r is not None:
        r_dev = r.to(DEV) if r_dev is None else r_dev
    h, y = C.norm_exact(x, w, EPS, r)
    if group is None:
        out = ops.add_rms_norm(x_dev, w.to(DEV), EPS, residual=r_dev)
        assert out.dtype == x.dtype and out.shape == x.shape
        C.assert_within(out, y, y.abs() * (ROUND[x.dtype] * 1.01 + 4e-6), "out")
    else:
        out, scale = ops.add_rms_norm_fp8(x_dev, w.to(DEV), EPS, residual=r_dev, group_size=group)
        scales, spread = C.norm_scales(y, group)
        assert out.dtype == C.FP8 and out.shape == x.shape and scale.shape == scales.shape
        C.assert_within(scale, scales, scales * 4e-6, "scale")
        exact = y / spread
        # half a step of 3 mantissa bits, or of the smallest ones; fp32 errors before it
        C.assert_within(out.float(), exact, torch.clamp(exact.abs() * 2.0 ** -4, min=2.0 ** -10) * 1.0001 + 448 * 1e-5, "out")
    if r is not None:
        C.assert_within(r_dev, h, h.abs() * ROUND[r.dtype] * 1.01, "residual")


@pytest.mark.parametrize("width", [1, 7, 8, 127, 128, 136, 512, 513, 1000, 2048, 2056, 4096, 5003, 8192, 8200, 32768, 32776, 70001])
@pytest.mark.parametrize("kind", ["bf16", "fp32", "fp8", "fp8_groups"])
def test_norm_widths(ops, width, kind):
    dtype = torch.float32 if kind == "fp32" or width % 2 else torch.bfloat16
    x, r, w = _norm_inputs(5, width, dtype, dtype, dtype, seed=width)
    _check_norm(ops, x, r, w, {"fp8": 0, "fp8_groups": 128}.get(kind))


@pytest.mark.parametrize("group", [None, 0, 128])
@pytest.mark.parametrize("x_type,r_type,w_type", [
    (torch.bfloat16, None, torch.bfloat16), (torch.bfloat16, torch.float32, torch.bfloat16),
    (torch.bfloat16, torch.bfloat16, torch.float32), (torch.float32, None, torch.float32),
    (torch.float32, torch.bfloat16, torch.bfloat16)])
def test_norm_types(ops, x_type, r_type, w_type, group):
    x, r, w = _norm_inputs(9, 1031, x_type, r_type, w_type)
    _check_norm(ops, x, r, w, group)


@pytest.mark.parametrize("group", [None, 128])
def test_norm_strided_rows_and_leading_dimensions(ops, group):
    """Columns 3 .. of a wider buffer (rows misaligned), in three dimensions; what lies between the rows stays."""
    width, pad = 777, 11
    x, r, w = _norm_inputs(6, width, torch.bfloat16, torch.bfloat16, torch.bfloat16)
    wide_x = torch.zeros(2, 3, width + pad, dtype=torch.bfloat16, device=DEV)
    wide_r = torch.full((2, 3, width + pad), 7.0, dtype=torch.bfloat16, device=DEV)
    x3, r3 = x.view(2, 3, width), r.view(2, 3, width)
    wide_x[..., 3:3 + width] = x3.to(DEV)
    wide_r[..., 3:3 + width] = r3.to(DEV)
    _check_norm(ops, x3, r3, w, group, wide_x[..., 3:3 + width], wide_r[..., 3:3 + width])
    assert (wide_r[..., :3] == 7).all() and (wide_r[..., 3 + width:] == 7).all()


def test_norm_broadcast_x_and_no_rows(ops):
    x, r, w = _norm_inputs(1, 640, torch.bfloat16, None, torch.bfloat16)
    r = torch.randn(4, 640).bfloat16()
    _check_norm(ops, x.expand(4, 640), r, w, None, x.to(DEV).expand(4, 640))
    out, scale = ops.add_rms_norm_fp8(torch.empty(0, 640, device=DEV), w.float().to(DEV), EPS, group_size=128)
    assert out.shape == (0, 640) and scale.shape == (0, 5)


@pytest.mark.parametrize("width", [256, 40000])
def test_norm_special_rows(ops, width):
    """Zeros (scale floor), NaN, infinity and tiny values; a NaN or infinite row is that in the definition too."""
    x = torch.randn(5, width, generator=torch.Generator().manual_seed(1))
    x[0] = 0
    x[1, 130] = float("nan")
    x[2, 5] = float("inf")
    x[3] *= 1e-30
    w = torch.ones(width)
    h, y = C.norm_exact(x, w, EPS)
    out = ops.add_rms_norm(x.to(DEV), w.to(DEV), EPS)
    C.assert_within(out, y, y.abs() * 5e-6, "out")
    for group in (0, 128):
        out, scale = ops.add_rms_norm_fp8(x.to(DEV), w.to(DEV), EPS, group_size=group)
        scale = scale.cpu()
        assert (out[0].float() == 0).all() and (scale[0] == scale[0, 0]).all() and abs(scale[0, 0] / 1e-12 - 1) < 1e-6
        assert out[1].float().isnan().all() and scale[1].isnan().all()
        first = out[2].float().cpu()
        assert first[:128].isnan().all() and scale[2, 0].isnan()  # inf * 0 in the infinite value's group
        if group == 128:
            assert (first[128:] == 0).all()
        assert (scale[3] > 0).all() and torch.isfinite(out[3].float()).all()


@pytest.mark.parametrize("width", [9, 60, 128, 129, 200, 255, 256, 257, 500, 1023, 1024, 1025, 2047])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("group", [None, 0, 128])
def test_norm_rows_that_share_a_workgroup(ops, width, dtype, group):
    x, r, w = _norm_inputs(37, width, dtype, torch.float32, torch.bfloat16, seed=width)
    _check_norm(ops, x, r, w, group)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("group", [None, 128])
@pytest.mark.parametrize("tokens,heads,width", [(1, 3, 128), (19, 5, 128), (33, 2, 200), (7, 3, 5), (3, 2, 40000)])
def test_norm_heads_of_a_fused_projection(ops, tokens, heads, width, dtype, group):
    x, r, w = _norm_inputs(tokens * heads, width, dtype, torch.float32, torch.float32, seed=heads)
    x, r = x.view(1, tokens, heads, width), r.view(1, tokens, heads, width)
    fused = torch.randn(1, tokens, heads + 3, width + 1, device=DEV).to(dtype)
    part = fused[:, :, 1:heads + 1, :width]
    part.copy_(x)
    _check_norm(ops, x, r, w, group, x_dev=part)


def test_norm_broadcast_groups(ops):
    x, _, w = _norm_inputs(4, 64, torch.bfloat16, None, torch.bfloat16)
    _check_norm(ops, x.view(4, 1, 64).expand(4, 3, 64), None, w, None, x_dev=x.to(DEV).view(4, 1, 64).expand(4, 3, 64))
    _check_norm(ops, x.view(1, 4, 64).expand(3, 4, 64), None, w, None, x_dev=x.to(DEV).view(1, 4, 64).expand(3, 4, 64))


def test_norm_groups_over_several_launches(ops):
    heads = 5
    tokens = ((1 << 22) + 40) // heads
    fused = torch.randn(tokens, heads + 1, 4, device=DEV).bfloat16()
    x, w = fused[:, :heads], torch.randn(4, device=DEV)
    _, y = C.norm_exact(x, w, EPS)
    C.assert_within(ops.add_rms_norm(x, w, EPS), y, y.abs() * (2.0 ** -8 * 1.01 + 4e-6), "out")


def test_norm_more_rows_than_a_launch_takes(ops):
    rows = (1 << 22) + 5
    gen = torch.Generator(device=DEV).manual_seed(0)
    x = torch.randn(rows, 4, device=DEV, generator=gen).bfloat16()
    r = torch.randn(rows, 4, device=DEV, generator=gen)
    w = torch.randn(4, device=DEV, generator=gen)
    want, h = r.clone(), None
    out = ops.add_rms_norm(x, w, EPS, residual=r)
    h, y = C.norm_exact(x, w, EPS, want)
    C.assert_within(out, y, y.abs() * (2.0 ** -8 * 1.01 + 4e-6), "out")
    C.assert_within(r, h, h.abs() * 2.0 ** -24 * 1.01, "residual")
    _, scale = ops.add_rms_norm_fp8(x, w, EPS)
    _, y = C.norm_exact(x, w, EPS)
    scales, _ = C.norm_scales(y, 0)
    C.assert_within(scale, scales, scales * 4e-6, "scale")


# ---------------------------------------------------------------------------
# store
# ---------------------------------------------------------------------------

def _store_exact(cache, rows, slots, page, scale):
    want = cache.clone()
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < cache.shape[0] * page:
            x = rows[t].float()
            if scale is not None:
                want[s // page, s % page] = (x.double() / scale.double()[:, None]).clamp(-448, 448).float().to(C.FP8)
            else:
                want[s // page, s % page] = rows[t]
    return want


@pytest.mark.parametrize("tokens,kv_heads,dim,page", [(1, 1, 64, 1), (3, 8, 128, 16), (70, 3, 64, 7), (5, 40, 128, 64),
                                                      (300, 2, 128, 100), (9, 1, 128, 1)])
@pytest.mark.parametrize("fp8", [False, True])
def test_store(ops, tokens, kv_heads, dim, page, fp8):
    """Fused-projection slices, interleaved caches, padded and out-of-pool slots; other slots keep their bytes."""
    gen = torch.Generator().manual_seed(tokens * 7 + kv_heads)
    pages = 2 * tokens // page + 2
    qkv = (torch.randn(1, tokens, 4 * kv_heads, dim, generator=gen) * 3).bfloat16()
    k, v = qkv[:, :, 2 * kv_heads:3 * kv_heads], qkv[:, :, 3 * kv_heads:]
    k_scale = v_scale = None
    both = torch.randn(pages, 2, page, kv_heads, dim, generator=gen).bfloat16()
    if fp8:  # some values pass 448 of their scale
        k_scale, v_scale = 0.01 + 0.01 * torch.rand(kv_heads, generator=gen), 0.01 + 0.01 * torch.rand(kv_heads, generator=gen)
        both = both.to(C.FP8)
    slots = torch.randperm(pages * page, generator=gen)[:tokens]
    if tokens > 2:
        slots[1], slots[2] = -1, pages * page
    index = torch.int64 if tokens % 2 else torch.int32
    on = both.to(DEV)
    qkv_on = qkv.to(DEV)
    move = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    ops.paged_kv_store(qkv_on[:, :, 2 * kv_heads:3 * kv_heads], qkv_on[:, :, 3 * kv_heads:], k_cache=on[:, 0], v_cache=on[:, 1],
                       slot_indices=slots.to(index).to(DEV), k_scale=move(k_scale), v_scale=move(v_scale))
    for at, rows, scale in ((0, k, k_scale), (1, v, v_scale)):
        want = _store_exact(both[:, at], rows[0], slots, page, scale)
        got = on[:, at].cpu()
        if not fp8:
            assert torch.equal(got, want)
        else:
            # x * (1 / scale) may fall on the other side of a tie: a neighbouring value, rarely
            differ = got.view(torch.uint8) != want.view(torch.uint8)
            assert differ.float().mean() < 1e-3
            step = torch.clamp(want.float().abs() * 2.0 ** -3, min=2.0 ** -9)
            assert ((got.float() - want.float()).abs() <= step).all()


def test_store_special_values_and_int64_slots(ops):
    """NaN stays, infinities become +-448; an int64 slot beyond 32 bits is outside the pool, not its low word."""
    k = torch.zeros(1, 3, 1, 64, dtype=torch.bfloat16, device=DEV)
    k[0, 0, 0, :4] = torch.tensor([float("nan"), float("inf"), -float("inf"), 1000.0])
    cache = torch.ones(2, 4, 1, 64, device=DEV).to(C.FP8)
    other = cache.clone()
    slots = torch.tensor([5, (1 << 32) + 2, -(1 << 40)], device=DEV)
    ops.paged_kv_store(k, k, k_cache=cache, v_cache=other, slot_indices=slots)
    row = cache[1, 1, 0].float().cpu()
    assert row[0].isnan() and row[1:4].tolist() == [448.0, -448.0, 448.0] and (row[4:] == 0).all()
    cache[1, 1] = 1.0
    assert (cache.float() == 1).all()


def test_store_more_tokens_than_a_launch_takes(ops):
    tokens = (1 << 24) + 5
    k = torch.randn(1, 1, 16, 128, device=DEV).bfloat16()
    slots = torch.full((tokens,), -1, dtype=torch.int32, device=DEV)
    slots[0], slots[-7], slots[-1] = 3, 1, 0
    cache = torch.zeros(2, 2, 16, 128, dtype=torch.bfloat16, device=DEV)
    other = torch.zeros_like(cache)
    ops.paged_kv_store(k.expand(1, tokens, 16, 128), (-k).expand(1, tokens, 16, 128), k_cache=cache, v_cache=other,
                       slot_indices=slots)
    for at, want in ((0, k[0, 0]), (1, k[0, 0]), (2, torch.zeros_like(k[0, 0])), (3, k[0, 0])):
        assert torch.equal(cache.view(4, 16, 128)[at], want) and torch.equal(other.view(4, 16, 128)[at], -want)


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

def _check_attention(ops, case, **over):
    out = ops.paged_attention(case.q.to(DEV), **case.kwargs(DEV, **over))
    assert out.shape == case.q.shape and out.dtype == torch.bfloat16
    want, bound = case.exact()
    C.assert_within(out, want, bound, "out")
    return out


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("heads,kv_heads", [(4, 4), (6, 2), (7, 1), (16, 1), (24, 1), (32, 1)])
def test_attention_decode(ops, dim, fp8, heads, kv_heads):
    """One new token each; contexts around the tile edges, and requests without a key."""
    keys = [1, 2, 31, 32, 33, 127, 128, 129, 0, 300, 640]
    _check_attention(ops, C.Attention(heads + dim, [1] * len(keys), keys, heads, kv_heads, dim, 16, fp8=fp8))


@pytest.mark.parametrize("page", [1, 5, 16, 64])
@pytest.mark.parametrize("fp8", [False, True])
def test_attention_one_long_request(ops, page, fp8):
    """A request's keys over many workgroups, joined."""
    _check_attention(ops, C.Attention(page, [1], [9001], 8, 2, 128, page, fp8=fp8, index64=True))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("page", [16, 24])
@pytest.mark.parametrize("heads,kv_heads", [(4, 4), (9, 3), (40, 1)])
def test_attention_prefill(ops, dim, fp8, page, heads, kv_heads):
    """Prompts and chunks of every size around the tiles, some without a new token."""
    new = [130, 0, 64, 1, 33, 200, 0]
    before = [0, 5, 64, 1000, 31, 77, 0]
    _check_attention(ops, C.Attention(heads * dim, new, [a + b for a, b in zip(new, before)], heads, kv_heads, dim, page, fp8=fp8))


@pytest.mark.parametrize("new", [5, 300])
def test_attention_few_tiles_over_many_keys(ops, new):
    """Few rows over a long context, its keys split and joined."""
    _check_attention(ops, C.Attention(new, [new], [new + 5000], 8, 1, 128, 16))


@pytest.mark.parametrize("window", [1, 2, 63, 64, 65, 129, 1000])
@pytest.mark.parametrize("new", [[1, 1, 1], [4, 2, 7], [150, 3, 64]])
def test_attention_window(ops, window, new):
    keys = [new[0], new[1] + 500, new[2] + 77]
    _check_attention(ops, C.Attention(window, new, keys, 6, 2, 64, 16, window=window))


@pytest.mark.parametrize("group", [7, 10, 11, 15])
def test_attention_window_of_heads_that_straddle_tiles(ops, group):
    """Tiles of 16 rows that begin and end inside tokens see one token's keys more."""
    for window in (1, 3, 128, 130):
        _check_attention(ops, C.Attention(group, [3, 2], [259, 517], group, 1, 64, 1, window=window),
                         max_query_len=1)


@pytest.mark.parametrize("cap", [0.5, 20.0])
@pytest.mark.parametrize("new", [[1, 1], [90, 20]])
def test_attention_cap(ops, cap, new):
    _check_attention(ops, C.Attention(3, new, [400, 150], 8, 2, 128, 16, cap=cap, spread=20.0))


@pytest.mark.parametrize("cap", [1e4, 1e6, 1e30])
@pytest.mark.parametrize("new", [[1, 1], [90, 20]])
def test_attention_cap_far_above_the_scores(ops, cap, new):
    """There the capped scores are the scores (off by s^3 / 3 cap^2 < 1e-6 here) and no accuracy is lost."""
    case = C.Attention(3, new, [n + 100 for n in new], 4, 2, 64, 16, cap=cap)
    out = ops.paged_attention(case.q.to(DEV), **case.kwargs(DEV))
    case.cap = 0.0
    want, bound = case.exact()
    C.assert_within(out, want, bound, "out")


@pytest.mark.parametrize("cap", [4.0, 200.0])
@pytest.mark.parametrize("hint", [1, 100])
def test_attention_cap_on_both_sides_of_the_series(ops, cap, hint):
    """Scores of up to four times the cap: the series, its end at a tenth, and saturation, in one request."""
    case = C.Attention(5, [2, 40], [70, 90], 4, 2, 64, 16, cap=cap, spread=cap)
    _check_attention(ops, case, max_query_len=hint)


@pytest.mark.parametrize("cap", [0.0, 1e-30, 30.0])
@pytest.mark.parametrize("hint", [1, 100])
def test_attention_nan_scales_stay(ops, cap, hint):
    """A NaN scale of one head's keys or values is that head's result, capped or not; other heads keep their bits."""
    case = C.Attention(23, [1, 40], [50, 90], 4, 2, 64, 16, fp8=True, cap=cap)
    kw = case.kwargs(DEV, max_query_len=hint)
    clean = ops.paged_attention(case.q.to(DEV), **kw)
    for name in ("k_scale", "v_scale"):
        scale = kw[name].clone()
        scale[1] = float("nan")
        out = ops.paged_attention(case.q.to(DEV), **dict(kw, **{name: scale}))
        assert torch.equal(out[:, :, :2], clean[:, :, :2]) and out[:, :, 2:].isnan().all(), name
    assert ops.paged_attention(case.q.to(DEV), **dict(kw, scale=float("nan"))).isnan().all()


@pytest.mark.parametrize("cap", [1e-30, 1e-3])
@pytest.mark.parametrize("hint", [1, 100])
def test_attention_cap_far_below_the_scores(ops, cap, hint):
    case = C.Attention(4, [1, 40], [50, 90], 4, 2, 64, 16, cap=cap)
    case.q[0, 0] = 0  # scores of 0
    _check_attention(ops, case, max_query_len=hint)


@pytest.mark.parametrize("hint", [1, 100])
@pytest.mark.parametrize("page", [16, 5])
def test_attention_wide_tables_of_few_keys(ops, hint, page):
    """Entries past a request's pages are any numbers; the table's width cuts the keys in many parts."""
    case = C.Attention(16, [1, 60, 3], [70, 2000, 3], 8, 2, 64, page)
    wide = torch.full((3, 9000), -7, dtype=torch.int32)
    wide[:, ::3] = 1 << 30
    wide[:, 1::3] = torch.tensor(case.unused[0], dtype=torch.int32)
    for n, k in enumerate(case.keys):
        used = -(-k // page)
        wide[n, :used] = case.page_table[n, :used]
    case.page_table = wide
    _check_attention(ops, case, max_query_len=hint)


@pytest.mark.parametrize("scale", [-0.125, 0.0, 3.0])
@pytest.mark.parametrize("new", [[1, 2], [90, 20]])
def test_attention_scales(ops, scale, new):
    """A negative, a zero and a large factor (large: one key takes nearly all the weight)."""
    case = C.Attention(5, new, [300, 150], 8, 2, 64, 16)
    case.scale = scale
    _check_attention(ops, case)


@pytest.mark.parametrize("hint", [0, 1, 3, 1000])
def test_attention_holds_for_any_hint(ops, hint):
    """max_query_len chooses a kernel, not a result: mixed decode, verify and prefill under each."""
    _check_attention(ops, C.Attention(9, [1, 0, 4, 130, 1, 17], [700, 9, 300, 130, 1, 1200], 12, 4, 128, 16),
                     max_query_len=hint)


@pytest.mark.parametrize("hint", [1, 100])
def test_attention_rows_without_keys_and_uncovered_tokens(ops, hint):
    """More new tokens than keys (the first see none), empty requests, tokens before and after the requests."""
    case = C.Attention(2, [5, 3, 70, 4], [2, 0, 50, 4], 4, 2, 64, 16, before=3, after=6)
    out = _check_attention(ops, case, max_query_len=hint)
    assert (out[0, :6] == 0).all() and (out[0, -6:] == 0).all() and (out[0, 8:11] == 0).all()


@pytest.mark.parametrize("new,keys,hint", [
    ([1, 3, 2, 1, 2], [5, 300, 1, 0, 600], 1), ([1], [9001], 1),             # decode, whole and over many workgroups
    ([1, 40, 50, 3], [5, 70, 44, 0], 50), ([70], [2570], 70)])               # prefill, whole and over split keys
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_rows_whose_scores_are_all_minus_infinity(ops, dim, new, keys, hint):
    """The softmax of such a row is 0 / 0, unlike that of a row that sees no key; one finite score is enough to make it
    that key's value."""
    case = C.Attention(22, new, keys, 4, 2, dim, 16)
    case.q[..., 0] = 1
    sees, last = [], []  # of each token: sees a key; the request's last key
    for m, L in zip(new, keys):
        sees += [L - m + i >= 0 for i in range(m)]
        last += [L - m + i == L - 1 and L > 0 for i in range(m)]
    sees, last = torch.tensor(sees), torch.tensor(last)
    clean = ops.paged_attention(case.q.to(DEV), **case.kwargs(DEV, max_query_len=hint)).cpu()
    held = case.k_cache.clone()
    case.k_cache[:, :, 1, 0] = -float("inf")
    out = ops.paged_attention(case.q.to(DEV), **case.kwargs(DEV, max_query_len=hint)).cpu()
    assert torch.equal(out[:, :, :2], clean[:, :, :2])
    assert out[0, sees, 2:].isnan().all() and (out[0, ~sees, 2:] == 0).all()
    for n, L in enumerate(keys):
        if L:
            page, off = (x[L - 1] for x in case.slots_of(n))
            case.k_cache[page, off] = held[page, off]
            value = case.v_cache[page, off, 1]
            out = ops.paged_attention(case.q.to(DEV), **case.kwargs(DEV, max_query_len=hint)).cpu()
            row = int(case.cu_seqlens[n + 1]) - 1
            assert torch.equal(out[0, row, 2:], value.expand(2, dim))
            last[row] = False
            assert out[0, last & sees, 2:].isnan().all()


@pytest.mark.parametrize("hint", [1, 100])
@pytest.mark.parametrize("page", [16, 5])
def test_attention_unwritten_slots_hold_nan(ops, hint, page):
    """NaN in every slot that holds no key of a request: beyond its length on its last page, on unused pages,
    and before the window of a single token."""
    case = C.Attention(4, [1, 1, 66, 30], [40, 9, 77, 30], 4, 2, 64, page)
    keep_k, keep_v = case.k_cache.clone(), case.v_cache.clone()
    case.k_cache.fill_(float("nan"))
    case.v_cache.fill_(float("nan"))
    for n in range(4):
        p, o = case.slots_of(n)
        case.k_cache[p, o], case.v_cache[p, o] = keep_k[p, o], keep_v[p, o]
    _check_attention(ops, case, max_query_len=hint)
    one = C.Attention(5, [1], [400], 4, 2, 128, page, window=37)
    p, o = one.slots_of(0)
    one.k_cache[p[:363], o[:363]] = float("nan")
    one.v_cache[p[:363], o[:363]] = float("nan")
    clean = C.Attention(5, [1], [400], 4, 2, 128, page, window=37)
    out = ops.paged_attention(one.q.to(DEV), **one.kwargs(DEV, max_query_len=hint * 40))
    want, bound = clean.exact()
    C.assert_within(out, want, bound, "out")


@pytest.mark.parametrize("hint", [1, 100])
@pytest.mark.parametrize("page", [16, 5])
def test_attention_pages_outside_the_pool_read_as_zeros(ops, hint, page):
    case = C.Attention(6, [2, 40], [90, 100], 4, 2, 64, page)
    case.page_table[0, 1] = -1
    case.page_table[0, 3] = case.k_cache.shape[0]
    case.page_table[1, 2] = 1 << 30
    case.page_table[1, 0] = -(1 << 31)
    _check_attention(ops, case, max_query_len=hint)


def test_attention_metadata_is_cut_to_the_tensors(ops):
    """Lengths beyond the table, and offsets beyond the tokens, address nothing outside."""
    for hint in (1, 100):
        case = C.Attention(7, [1, 30], [64, 100], 4, 2, 64, 16)
        kw = case.kwargs(DEV, max_query_len=hint)
        kw["kv_lens"] = torch.tensor([64, 1 << 30], dtype=torch.int32, device=DEV)
        kw["page_table"] = kw["page_table"][:, :5].contiguous()
        out = ops.paged_attention(case.q.to(DEV), **kw)
        case.keys = [64, 80]
        want, bound = case.exact()
        C.assert_within(out, want, bound, "out")
        kw["cu_seqlens"] = torch.tensor([0, 1, 1 << 30], dtype=torch.int32, device=DEV)
        assert torch.equal(ops.paged_attention(case.q.to(DEV), **kw), out)


@pytest.mark.parametrize("hint", [1, 100])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("page", [16, 5])
def test_attention_int64_entries_beyond_32_bits(ops, hint, fp8, page):
    """They are outside the pool, the table or the batch, as they are for the store: not their low words."""
    case = C.Attention(19, [2, 40], [90, 100], 4, 2, 64, page, fp8=fp8, index64=True)
    case.page_table[0, 1] += 1 << 32
    case.page_table[0, 3] -= 1 << 32
    case.page_table[1, 0] = (1 << 63) - 1
    case.page_table[1, 2] += 1 << 62
    kw = case.kwargs(DEV, max_query_len=hint)
    exact = C.Attention(19, [2, 40], [90, 100], 4, 2, 64, page, fp8=fp8, index64=True)
    for n, at in ((0, 1), (0, 3), (1, 0), (1, 2)):
        exact.page_table[n, at] = -1
    want, bound = exact.exact()
    C.assert_within(ops.paged_attention(case.q.to(DEV), **kw), want, bound, "pages")

    case = C.Attention(20, [1, 30], [64, 100], 4, 2, 64, page, fp8=fp8, index64=True)
    kw = case.kwargs(DEV, max_query_len=hint)
    kw["page_table"] = kw["page_table"][:, :80 // page].contiguous()
    kw["kv_lens"] = torch.tensor([-(1 << 32) + 9, (1 << 32) + 9], device=DEV)
    kw["cu_seqlens"] = torch.tensor([-(1 << 40) + 1, 1, (1 << 33) + 2], device=DEV)
    case.keys = [0, 80]
    want, bound = case.exact()
    C.assert_within(ops.paged_attention(case.q.to(DEV), **kw), want, bound, "lengths and offsets")


@pytest.mark.parametrize("hint", [1, 100])
@pytest.mark.parametrize("fp8", [False, True])
def test_attention_strides(ops, hint, fp8):
    """q a misaligned slice of a fused projection; keys and values interleaved in one allocation, heads outermost."""
    case = C.Attention(8, [1, 40], [77, 90], 6, 2, 64, 16, fp8=fp8)
    q = torch.zeros(1, 41, 9, 67, dtype=torch.bfloat16, device=DEV)[:, :, 2:8, 1:65]
    q.copy_(case.q)
    kw = case.kwargs(DEV, max_query_len=hint)
    pages = kw["k_cache"].shape[0]
    both = torch.zeros(2, pages, 2, 16, 64, dtype=torch.uint8 if fp8 else torch.bfloat16, device=DEV)
    if fp8:
        both = both.view(C.FP8)
    both[0].copy_(kw["k_cache"].permute(0, 2, 1, 3))
    both[1].copy_(kw["v_cache"].permute(0, 2, 1, 3))
    kw["k_cache"], kw["v_cache"] = both[0].permute(0, 2, 1, 3), both[1].permute(0, 2, 1, 3)
    table = torch.full((2, 40), -1, dtype=torch.int32, device=DEV)[:, 5:5 + kw["page_table"].shape[1]]
    table.copy_(kw["page_table"])
    kw["page_table"] = table
    out = ops.paged_attention(q, **kw)
    want, bound = case.exact()
    C.assert_within(out, want, bound, "out")


@pytest.mark.parametrize("hint", [1, 100])
def test_attention_single_head_at_any_stride(ops, hint):
    case = C.Attention(21, [1, 40], [40, 64], 4, 1, 64, 16)
    kw = case.kwargs(DEV, max_query_len=hint)
    for name in ("k_cache", "v_cache"):
        t = kw[name]
        kw[name] = t.as_strided(t.shape, (t.stride(0), t.stride(1), 3, 1))
        assert torch.equal(kw[name], t)
    want, bound = case.exact()
    C.assert_within(ops.paged_attention(case.q.to(DEV), **kw), want, bound, "out")


@pytest.mark.parametrize("hint", [1, 100])
def test_attention_offsets_past_32_bits(ops, hint):
    """Pages more than 2^32 elements apart, written by the store and read back."""
    case = C.Attention(9, [1, 40], [40, 64], 4, 2, 64, 16)
    kw = case.kwargs(DEV, max_query_len=hint)
    pages = kw["k_cache"].shape[0]
    step = (1 << 32) // (pages - 2) // 8 * 8
    room = torch.empty(2, pages * step, dtype=torch.bfloat16, device=DEV)
    caches = [room[i].as_strided((pages, 16, 2, 64), (step, 128, 64, 1)) for i in range(2)]
    assert (pages - 1) * step > 1 << 32
    slots = torch.arange(pages * 16, device=DEV)
    ops.paged_kv_store(kw["k_cache"].view(1, -1, 2, 64), kw["v_cache"].view(1, -1, 2, 64), k_cache=caches[0], v_cache=caches[1],
                       slot_indices=slots)
    assert torch.equal(caches[0], kw["k_cache"]) and torch.equal(caches[1], kw["v_cache"])
    kw["k_cache"], kw["v_cache"] = caches
    out = ops.paged_attention(case.q.to(DEV), **kw)
    want, bound = case.exact()
    C.assert_within(out, want, bound, "out")


def test_attention_many_requests(ops):
    """More requests than a workgroup has threads, most of them short, in both kernels."""
    rng = random.Random(3)
    new = [rng.choice([0, 1, 1, 1, 2]) for _ in range(600)]
    keys = [m + rng.choice([0, 3, 40, 200]) for m in new]
    case = C.Attention(10, new, keys, 4, 2, 64, 16)
    _check_attention(ops, case)
    _check_attention(ops, case, max_query_len=1000)


@pytest.mark.parametrize("n", [16, 17, 128, 129])
def test_attention_chunks_of_many_requests(ops, n):
    rng = random.Random(n)
    new = [rng.choice([0, 1, 20, 33, 64, 129]) for _ in range(n)]
    case = C.Attention(15, new, [m and m + rng.choice([0, 0, 100, 300]) for m in new], 8, 2, 64, 16, before=1, after=2)
    _check_attention(ops, case, max_query_len=129)


def test_attention_batches_padded_with_empty_requests(ops):
    new = [0] * 70 + [1] + [0] * 3000 + [2, 1] + [0] * 129 + [1] + [0] * 900
    keys = [m and 150 + 40 * m for m in new]
    case = C.Attention(12, new, keys, 4, 2, 64, 16)
    _check_attention(ops, case)
    _check_attention(ops, case, max_query_len=1000)


def test_attention_decreasing_offsets_address_nothing_outside(ops):
    """Such metadata has no meaning, and its requests' units may pass 32 bits; a good call after it is right."""
    case = C.Attention(13, [10, 20, 1], [40, 64, 30], 4, 2, 64, 16)
    for hint in (1, 100):
        kw = case.kwargs(DEV, max_query_len=hint)
        kw["cu_seqlens"] = torch.tensor([0, 30, 10, 31], dtype=torch.int32, device=DEV)
        assert ops.paged_attention(case.q.to(DEV), **kw).shape == case.q.shape
        _check_attention(ops, case, max_query_len=hint)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("window", [0, 70])
@pytest.mark.parametrize("new,heads,hint", [([1, 3], 2, 3), ([8, 1], 4, 8), ([2, 150], 4, 150), ([400], 2, 400)])
def test_attention_what_a_row_does_not_see_cannot_reach_it(ops, fp8, dim, window, new, heads, hint):
    _check_isolation(ops, fp8, dim, window, new, heads, hint, 333)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("window", [0, 700])
def test_attention_what_a_row_does_not_see_cannot_reach_it_over_splits(ops, fp8, window):
    _check_isolation(ops, fp8, 128, window, [70], 4, 70, 2500)


def _check_isolation(ops, fp8, dim, window, new, heads, hint, earlier):
    """Infinite and NaN keys and values of one token: rows that do not see it keep their bits, and of
    those that do only its columns change."""
    keys = [m + earlier for m in new]
    case = C.Attention(14, new, keys, heads, 2, dim, 16, fp8=fp8, window=window)
    clean = _check_attention(ops, case, max_query_len=hint).cpu()
    G, n = heads // 2, max(range(len(new)), key=lambda i: new[i])
    page, off = case.slots_of(n)
    nan, inf = float("nan"), float("inf")
    for back in {0, 1, new[n] // 2, new[n] - 1}:
        j = keys[n] - 1 - back
        sees = torch.zeros(case.q.shape[1], dtype=torch.bool)
        start = int(case.cu_seqlens[n])
        sees[start + new[n] - 1 - back:start + new[n]] = True
        if window:
            sees[start + new[n] - 1 - back + window:] = False
        for which in ("v", "k"):
            cache = case.v_cache if which == "v" else case.k_cache
            held = cache[page[j], off[j], 1].clone()
            bad = held.float()
            if which == "v":
                bad[3], bad[dim - 2] = nan, nan if fp8 else -inf
            else:
                bad[5] = nan
            cache[page[j], off[j], 1] = bad.to(cache.dtype)
            out = ops.paged_attention(case.q.to(DEV), **case.kwargs(DEV, max_query_len=hint)).cpu()
            cache[page[j], off[j], 1] = held
            hit = torch.zeros(out.shape, dtype=torch.bool)
            if which == "v":
                hit[:, sees, G:, 3] = hit[:, sees, G:, dim - 2] = True
            else:
                hit[:, sees, G:] = True
            assert torch.equal(out[~hit], clean[~hit]), (which, back)
            assert not torch.isfinite(out[hit]).any(), (which, back)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new,heads,requests,earlier,hint", [
    (4, 4, 300, 300, 4),     # decode, 16-row tiles: more units than workgroups, so that a wave has several blocks
    (4, 16, 300, 300, 4),    # 32-row tiles
    (40, 4, 2, 333, 40),     # prefill
    (70, 4, 1, 2500, 70)])   # prefill over split keys
def test_attention_rows_keep_their_bits_beside_large_hidden_scores(ops, fp8, dim, new, heads, requests, earlier, hint):
    """The last key, which only the last token sees, gets a score far above the running maximum there: the other
    rows of the tile keep theirs, and so their weights' roundings."""
    L = new + earlier
    case = C.Attention(18, [new] * requests, [L] * requests, heads, 2, dim, 16, fp8=fp8)
    q, kw = case.q.to(DEV), case.kwargs(DEV, max_query_len=hint)
    clean = ops.paged_attention(q, **kw)
    ends = case.cu_seqlens[1:].long() - 1
    page = torch.tensor([int(case.page_table[n, (L - 1) // 16]) for n in range(requests)], device=DEV)
    loud = q[0, ends.to(DEV)][:, [0, heads // 2]].float() * 4  # each key head's first query head, times 4
    if fp8:
        loud = (loud / kw["k_scale"][:, None]).clamp(-448, 448)
    kw["k_cache"].view(torch.uint8 if fp8 else torch.int16)[page, (L - 1) % 16] = \
        loud.to(kw["k_cache"].dtype).view(torch.uint8 if fp8 else torch.int16)
    out = ops.paged_attention(q, **kw)
    sees = torch.zeros(q.shape[1], dtype=torch.bool, device=DEV)
    sees[ends.to(DEV)] = True
    assert torch.equal(out[0, ~sees], clean[0, ~sees])
    assert (out[0, sees][:, [0, heads // 2]] != clean[0, sees][:, [0, heads // 2]]).any(-1).all()


def test_attention_nothing_to_do(ops):
    case = C.Attention(1, [0, 0], [5, 0], 4, 2, 64, 16)
    assert ops.paged_attention(case.q.to(DEV), **case.kwargs(DEV)).shape == (1, 0, 4, 64)
    case = C.Attention(1, [], [], 4, 2, 64, 16, before=3)  # no request: every token uncovered
    for hint in (0, 100):
        assert (ops.paged_attention(case.q.to(DEV), **case.kwargs(DEV, max_query_len=hint)) == 0).all()
    case = C.Attention(1, [1, 20], [5, 20], 4, 2, 64, 16)  # no page at all
    for hint in (1, 100):
        kw = case.kwargs(DEV, max_query_len=hint)
        kw["page_table"] = kw["page_table"][:, :0]
        assert (ops.paged_attention(case.q.to(DEV), **kw) == 0).all()


@pytest.mark.parametrize("seed", range(60))
def test_attention_random(ops, seed):
    case = C.random_attention(seed)
    print(case.new, case.keys, case.heads, case.kv_heads, case.dim, case.page, case.window, case.cap, flush=True)
    if case.q.shape[1] == 0:
        return
    _check_attention(ops, case, max_query_len=[case.max_query_len, 1, 1000][seed % 3])


def test_streams_and_graph_replay(ops):
    """The layer's calls on a stream of their own, captured once and replayed on changed inputs, bit for bit
    like eager calls; repeated calls agree bit for bit."""
    gen = torch.Generator(device=DEV).manual_seed(0)
    case = C.Attention(11, [1] * 5, [300, 2, 40, 1000, 77], 8, 2, 128, 16)
    kw = case.kwargs(DEV)
    x = torch.randn(5, 512, device=DEV, generator=gen).bfloat16()
    r = torch.randn(5, 512, device=DEV, generator=gen).bfloat16()
    w = torch.ones(512, device=DEV).bfloat16()
    q = case.q.to(DEV)
    k = torch.randn(1, 5, 2, 128, device=DEV, generator=gen).bfloat16()
    slots = torch.tensor([3, 17, 40, -1, 60], device=DEV)

    def step():
        y, s = ops.add_rms_norm_fp8(x, w, EPS, residual=r, group_size=128)
        ops.paged_kv_store(k, k, k_cache=kw["k_cache"], v_cache=kw["v_cache"], slot_indices=slots)
        return y.view(torch.uint8), s, ops.paged_attention(q, **kw)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for i in range(4):
        x.copy_(torch.randn(5, 512, device=DEV, generator=gen))
        q.copy_(torch.randn(q.shape, device=DEV, generator=gen))
        kw["kv_lens"].copy_(torch.tensor([1 + i, 2, 40 - i, 1000, 70], dtype=torch.int32))
        before = r.clone()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured] + [r.clone()]
        r.copy_(before)
        want = list(step()) + [r]
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b), i


@pytest.mark.parametrize("new,keys", [([70], [2570]), ([60, 1, 33], [60, 400, 200])])
def test_prefill_graph_replay(ops, new, keys):
    """Chunks, with their keys in parts and whole, captured and replayed on changed inputs and lengths."""
    gen = torch.Generator(device=DEV).manual_seed(1)
    case = C.Attention(17, new, keys, 8, 2, 128, 16)
    kw = case.kwargs(DEV)
    q = case.q.to(DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.paged_attention(q, **kw)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = ops.paged_attention(q, **kw)
    for i in range(4):
        q.copy_(torch.randn(q.shape, device=DEV, generator=gen))
        kw["kv_lens"].sub_(3)
        graph.replay()
        assert torch.equal(captured, ops.paged_attention(q, **kw)), i
        torch.cuda.synchronize()
