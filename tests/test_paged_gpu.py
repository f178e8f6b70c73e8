"""Paged caches on the GPU: appends (fa_paged_append) and attention (fa_paged_attn) against 64-bit
references, with the bounds that the kernels' roundings allow (paged_reference), and runs of both."""
import math
import random

import pytest
import torch

import pallas_flexattn as pf
from pallas_flexattn import _lib as L
from pallas_flexattn.flash_attn import check_device_status
from paged_reference import U_E4M3, assert_within, attend64, e4m3_step, rotate64, scale_for, to_e4m3_64, unit

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0) if torch.cuda.is_available() else None
BF16, F32, F8 = torch.bfloat16, torch.float32, torch.float8_e4m3fn


def make_cache(pages, hkv, ps, D, dtype, g, layout="hnd", spread=3):
    """A pool of random pages, each 8-bit page and head with a power-of-two scale of its own."""
    shape = (pages, hkv, ps, D) if layout == "hnd" else (pages, ps, hkv, D)
    pools, scales = [], []
    for _ in range(2):
        x = torch.randn(shape, generator=g).to(DEV)
        if dtype == F8:
            x = (x * 90).clamp(-448, 448)
            scales.append(torch.exp2(torch.randint(-8 - spread, -8 + spread, (pages, hkv), generator=g).float()).to(DEV))
        x = x.to(dtype)
        pools.append(x if layout == "hnd" else x.transpose(1, 2))
    return pf.PagedKVCache(*pools, *scales)


def make_table(B, cols, pages, g):
    return torch.randperm(pages, generator=g)[: B * cols].view(B, cols).to(DEV, torch.int32)


# ------------------------------------------------------------------------------- attention
# B, H, Hkv, Tq, D, dtype, ps, lens, q_lens, mask, window, score
ATTEND = {
    "one_token_one_key": (1, 1, 1, 1, 128, F8, 16, [1], None, "causal", 0, None),
    "gqa4_t1_f8": (3, 8, 2, 1, 128, F8, 64, [700, 1, 129], None, "causal", 0, None),
    "gqa8_t1_f8": (2, 8, 1, 1, 128, F8, 128, [1000, 127], None, None, 0, None),
    "gqa3_t3_f8_r16": (2, 6, 2, 3, 128, F8, 32, [300, 3], None, "causal", 0, "alibi"),
    "r32_f8_d64": (2, 24, 1, 1, 64, F8, 16, [513, 40], None, "causal", 0, "softcap"),
    "r64_f8_d128": (2, 16, 1, 4, 128, F8, 64, [260, 1024], None, "causal", 0, None),
    "r64_f8_d256": (1, 16, 2, 7, 256, F8, 32, [777], None, "causal", 0, "softcap"),
    "r8_f8_d64": (4, 4, 4, 1, 64, F8, 128, [128, 127, 129, 5], None, "causal", 0, None),
    "r8_f8_d256": (2, 14, 2, 1, 256, F8, 16, [400, 333], None, "causal", 0, "both"),
    "groups_f8": (2, 8, 1, 40, 128, F8, 64, [300, 77], [40, 23], "causal", 0, None),
    "groups_bf16_d256": (1, 4, 1, 30, 256, BF16, 64, [400], None, "causal", 0, None),
    "bf16_r16_d64": (3, 4, 4, 1, 64, BF16, 16, [257, 16, 15], None, "causal", 0, "alibi"),
    "bf16_r16_d128": (2, 32, 8, 1, 128, BF16, 64, [1500, 64], None, "causal", 0, None),
    "bf16_r32_d128": (1, 7, 1, 4, 128, BF16, 32, [555], None, "causal", 0, "softcap"),
    "bf16_r64_d128": (1, 64, 1, 1, 128, BF16, 128, [500], None, None, 0, None),
    "bf16_r64_d64": (2, 12, 2, 9, 64, BF16, 64, [90, 500], [9, 4], "causal", 0, None),
    "bf16_d256": (2, 8, 2, 1, 256, BF16, 64, [130, 700], None, "causal", 0, None),
    "window_f8": (3, 8, 2, 2, 128, F8, 64, [1000, 130, 40], None, "window", 100, None),
    "window_bf16_small": (2, 2, 1, 1, 64, BF16, 16, [900, 33], None, "window", 1, "alibi"),
    "window_groups": (1, 4, 1, 70, 128, F8, 16, [600], None, "window", 33, None),
    "zero_lens": (4, 4, 1, 1, 128, F8, 64, [0, 200, 0, 64], None, "causal", 0, None),
    "rows_before_the_start": (2, 4, 1, 5, 128, F8, 64, [3, 200], None, "causal", 0, None),
    "ragged_q": (4, 4, 2, 6, 64, F8, 32, [100, 50, 7, 9], [6, 1, 0, 3], "causal", 0, None),
    "no_mask_t4": (2, 4, 2, 4, 128, BF16, 64, [100, 250], [4, 2], None, 0, None),
    "many_short": (40, 4, 4, 1, 128, F8, 16, None, None, "causal", 0, None),
    "many_units_bf16": (70, 8, 8, 1, 64, BF16, 16, None, None, "causal", 0, None),
    "one_long": (1, 4, 2, 1, 128, F8, 64, [20000], None, "causal", 0, None),
    "one_long_bf16": (1, 2, 1, 1, 64, BF16, 128, [30011], None, "causal", 0, "softcap"),
    "long_and_short": (5, 8, 2, 1, 128, F8, 128, [9000, 1, 128, 3000, 0], None, "causal", 0, None),
}


def attend_case(name, layout="hnd"):
    B, H, Hkv, Tq, D, dtype, ps, lens, qlens, mask, window, score = ATTEND[name]
    seed = sum(map(ord, name))
    g = torch.Generator().manual_seed(seed)
    if lens is None:
        r = random.Random(seed)
        lens = [r.randint(0, 300) for _ in range(B)]
    cols = max(1, -(-max(lens) // ps)) + 1
    cache = make_cache(B * cols + 2, Hkv, ps, D, dtype, g, layout)
    table = make_table(B, cols, B * cols + 2, g)
    q = torch.randn(B, H, Tq, D, generator=g).to(DEV, BF16)
    mods = {None: None, "alibi": pf.alibi_score_mod(H), "softcap": pf.softcap_score_mod(15.0),
            "both": pf.compose_score_mods(pf.alibi_score_mod(H), pf.softcap_score_mod(15.0))}
    kw = dict(q_lens=qlens, score_mod=mods[score])
    mod = {None: None, "causal": pf.causal_mask, "window": pf.sliding_window_mask(window, 0)}[mask]
    slopes = pf.alibi_slopes(H).to(DEV) if score in ("alibi", "both") else None
    cap = 15.0 if score in ("softcap", "both") else 0.0
    ref = lambda: attend64(q, cache, table, lens, qlens or [Tq] * B, mask, window, slopes, cap, 1 / math.sqrt(D))  # noqa: E731
    return q, cache, table, lens, mod, kw, ref


def check_attend(q, cache, table, lens, mod, kw, ref):
    o, lse = pf.flash_attention_paged(q, cache, table, lens, mod, **kw)
    check_device_status(DEV)
    ro, rl, to, tl = ref()
    assert_within("lse", lse, rl, tl)
    assert_within("o", o, ro, to)
    return o, lse


@pytest.mark.parametrize("name", list(ATTEND))
def test_attention_matches_the_formula(name):
    check_attend(*attend_case(name))


@pytest.mark.parametrize("name", ["r64_f8_d128", "r64_f8_d256", "groups_f8", "bf16_r64_d128", "bf16_r64_d64",
                                  "window_groups", "groups_bf16_d256", "ragged_q", "long_and_short"])
def test_wide_tables(name):
    """Room for far longer sequences than there are: more query rows share a tile then, and nothing of the
    columns behind the lengths is read."""
    q, cache, table, lens, mod, kw, ref = attend_case(name)
    wide = torch.full((table.shape[0], 5000), -3, dtype=torch.int32, device=DEV)
    for b, n in enumerate(lens):
        used = -(-n // cache.page_size)
        wide[b, :used] = table[b, :used]
    check_attend(q, cache, wide[:, :4999], lens, mod, kw, ref)


@pytest.mark.parametrize("name", ["gqa4_t1_f8", "bf16_r16_d128", "r64_f8_d256"])
def test_pages_stored_token_major(name):
    check_attend(*attend_case(name, layout="nhd"))


@pytest.mark.parametrize("name", ["gqa3_t3_f8_r16", "bf16_r64_d64", "groups_f8"])
def test_strided_and_misaligned_queries(name):
    q, *rest = attend_case(name)
    B, H, Tq, D = q.shape
    flat = torch.empty(q.numel() + 5, dtype=BF16, device=DEV)
    odd = flat[5:].view(B, Tq, H, D).transpose(1, 2)
    odd.copy_(q)
    want = pf.flash_attention_paged(q, *rest[:4], **rest[4])
    got = pf.flash_attention_paged(odd, *rest[:4], **rest[4])
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])


@pytest.mark.parametrize("dtype", [F8, BF16])
def test_what_lies_outside_is_never_used(dtype):
    """Positions behind each sequence, pages left of a window, table entries outside and other pages hold
    NaN or nonsense: nothing of it shows."""
    g = torch.Generator().manual_seed(5)
    B, Hkv, ps, D, lens, window = 3, 2, 32, 128, [70, 333, 161], 50
    cache = make_cache(64, Hkv, ps, D, dtype, g)
    table = make_table(B, 12, 64, g)
    q = torch.randn(B, 8, 2, D, generator=g).to(DEV, BF16)
    want = pf.flash_attention_paged(q, cache, table, lens, pf.sliding_window_mask(window, 0))
    used = set()
    for b, n in enumerate(lens):
        lo = max(0, n - 2 - window)
        used |= {int(table[b, c]) for c in range(lo // ps, -(-n // ps))}
        for c in range(12):
            page = int(table[b, c])
            for pool in (cache.k, cache.v):
                if (c + 1) * ps > n:  # behind the last position
                    pool[page, :, max(0, n - c * ps):] = torch.full((1,), math.nan, device=DEV).to(dtype)
                if c * ps < lo:
                    pool[page, :, : min(ps, lo - c * ps)] = torch.full((1,), math.nan, device=DEV).to(dtype)
        table[b, : lo // ps] = -7
        table[b, -(-n // ps):] = 1 << 30
    if dtype == F8:
        rest = torch.tensor([p not in used for p in range(64)], device=DEV)
        cache.k_scale[rest], cache.v_scale[rest] = math.nan, math.inf
    got = pf.flash_attention_paged(q, cache, table, lens, pf.sliding_window_mask(window, 0))
    check_device_status(DEV)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])


def test_scales_far_apart():
    """Pages whose values differ by 2^30 in size, and weight that sits on the pages of small ones."""
    g = torch.Generator().manual_seed(8)
    cache = make_cache(12, 1, 16, 128, F8, g)
    table = torch.arange(12, device=DEV, dtype=torch.int32).view(1, 12)
    cache.v_scale.copy_(torch.exp2(torch.tensor([-20.0, 10, -8, 0, -30, -3, -100, -12, 4, -9, 2, -1]))[:, None])
    cache.k_scale.copy_(torch.exp2(torch.full((12, 1), -9.0)))
    cache.k_scale[4] = 2.0 ** -5  # large logits on the page of scale 2^-30
    q = torch.randn(1, 4, 1, 128, generator=g).to(DEV, BF16)
    for n in (192, 80, 112):
        check_attend(q, cache, table, [n], pf.causal_mask, {},
                     lambda: attend64(q, cache, table, [n], [1], "causal", 0, None, 0, 1 / math.sqrt(128)))
    cache.v_scale.zero_()
    o, lse = pf.flash_attention_paged(q, cache, table, [192], pf.causal_mask)
    assert torch.all(o == 0) and torch.isfinite(lse).all()


def test_large_and_growing_logits():
    """Logits that grow along the sequence, so that the running references move again and again, and
    queries far from 1 in size."""
    g = torch.Generator().manual_seed(9)
    for dtype in (F8, BF16):
        cache = make_cache(40, 1, 64, 64, dtype, g, spread=1)
        table = torch.arange(40, device=DEV, dtype=torch.int32).view(1, 40)
        u = torch.sign(torch.randn(64, generator=g)).to(DEV)
        grow = (torch.arange(40, device=DEV) + 1)[:, None, None, None].float()
        cache.k.copy_((u * grow * 4 + cache.k.float() * 0.01).to(dtype))
        for size in (1.0, 2.0 ** -20, 0.03):
            q = (u * size + torch.randn(1, 2, 1, 64, generator=g).to(DEV) * size * 0.1).to(BF16)
            scale = 0.5 / size / (float(cache.k_scale.max()) * 64 if dtype == F8 else 64)
            check_attend(q, cache, table, [2500], pf.causal_mask, dict(scale=scale),
                         lambda: attend64(q, cache, table, [2500], [1], "causal", 0, None, 0, scale))


def test_bad_pages_are_hidden_and_reported():
    q, cache, table, lens, mod, kw, _ = attend_case("gqa4_t1_f8")
    n = cache.k.shape[0]
    for bad in (-1, n, 1 << 30, -(1 << 31)):
        t = table.clone()
        t[0, 3] = bad
        o, lse = pf.flash_attention_paged(q, cache, t, lens, mod, **kw)
        with pytest.raises(L.FlexAttnError, match="out of range"):
            check_device_status(DEV)
        ro, rl, to, tl = attend64(q, cache, t, lens, [1] * 3, "causal", 0, None, 0, 1 / math.sqrt(128))
        assert_within("lse", lse, rl, tl)
        assert_within("o", o, ro, to)
    for bad in ([700, -1, 129], [700, 1, 64 * table.shape[1] + 1]):
        pf.flash_attention_paged(q, cache, table, bad, mod, **kw)
        with pytest.raises(L.FlexAttnError, match="out of range"):
            check_device_status(DEV)


def test_nan_in_one_query_stays_in_its_row():
    q, cache, table, lens, mod, kw, _ = attend_case("gqa3_t3_f8_r16")
    want = pf.flash_attention_paged(q, cache, table, lens, mod, **kw)
    for v in (math.nan, math.inf):
        x = q.clone()
        x[0, 1, 1, 5] = v
        o, lse = pf.flash_attention_paged(x, cache, table, lens, mod, **kw)
        hit = torch.zeros(2, 6, 3, dtype=torch.bool, device=DEV)
        hit[0, 1, 1] = True
        assert torch.isnan(o[hit]).all() and torch.equal(o[~hit], want[0][~hit]) and torch.equal(lse[~hit], want[1][~hit])


@pytest.mark.parametrize("left,right", [(20, 3), (0, 0), (-1, 2), (1 << 30, 1 << 30), ((1 << 31) - 1, (1 << 31) - 1)])
def test_windows_to_both_sides(left, right):
    q, cache, table, lens, _, kw, _ = attend_case("ragged_q")
    wl, wr = (1 << 40 if left < 0 else left), right
    check_attend(q, cache, table, lens, pf.sliding_window_mask(left, right), kw,
                 lambda: attend64(q, cache, table, lens, kw["q_lens"], "band", (wl, wr), None, 0, 1 / math.sqrt(64)))


def test_thousands_of_sequences_most_of_them_empty():
    """More sequences than threads, and more empty ones than a CTA's list of them holds."""
    g = torch.Generator().manual_seed(2)
    B, H, hkv, ps = 4000, 4, 4, 16
    cache = make_cache(50, hkv, ps, 64, F8, g)
    table = torch.randint(0, 50, (B, 2), generator=g).to(DEV, torch.int32)  # pages shared by sequences
    lens = [0] * B
    for i in range(0, B, 97):
        lens[i] = 1 + i % 32
    q = torch.randn(B, H, 1, 64, generator=g).to(DEV, BF16)
    o, lse = pf.flash_attention_paged(q, cache, table, torch.tensor(lens, dtype=torch.int32, device=DEV), pf.causal_mask)
    check_device_status(DEV)
    some = [i for i in range(B) if lens[i]]
    idx = torch.tensor(some, device=DEV)
    ro, rl, to, tl = attend64(q[idx], cache, table[idx], [lens[i] for i in some], [1] * len(some), "causal", 0, None, 0,
                              1 / math.sqrt(64))
    assert_within("o", o[idx], ro, to)
    assert_within("lse", lse[idx], rl, tl)
    empty = torch.ones(B, dtype=torch.bool, device=DEV)
    empty[idx] = False
    assert torch.all(o[empty] == 0) and torch.all(lse[empty] == -math.inf)


def test_many_heads_share_one_key_head():
    g = torch.Generator().manual_seed(12)
    for dtype in (F8, BF16):
        cache = make_cache(12, 1, 64, 128, dtype, g)
        table = make_table(2, 5, 12, g)
        q = torch.randn(2, 128, 1, 128, generator=g).to(DEV, BF16)  # two row groups of 64, or four of 32
        check_attend(q, cache, table, [300, 129], pf.causal_mask, {},
                     lambda: attend64(q, cache, table, [300, 129], [1, 1], "causal", 0, None, 0, 1 / math.sqrt(128)))


@pytest.mark.parametrize("dtype", [F8, BF16])
def test_nan_that_a_row_sees_reaches_it(dtype):
    """A NaN key makes every row that sees it NaN, a NaN value only its element of D."""
    g = torch.Generator().manual_seed(6)
    cache = make_cache(10, 2, 32, 64, dtype, g)
    table = make_table(1, 8, 10, g)
    q = torch.randn(1, 4, 1, 64, generator=g).to(DEV, BF16)
    want = pf.flash_attention_paged(q, cache, table, [250], pf.causal_mask)
    nan = torch.full((1,), math.nan, device=DEV).to(dtype)
    page = int(table[0, 3])
    cache.v[page, 1, 5, 7:8] = nan
    o, lse = pf.flash_attention_paged(q, cache, table, [250], pf.causal_mask)
    hit = torch.zeros_like(o, dtype=torch.bool)
    hit[0, 2:, 0, 7] = True
    assert torch.isnan(o[hit]).all() and torch.equal(o[~hit], want[0][~hit]) and torch.equal(lse, want[1])
    cache.k[page, 0, 9, 0:1] = nan
    o, lse = pf.flash_attention_paged(q, cache, table, [250], pf.causal_mask)
    assert torch.isnan(o[0, :2]).all() and torch.isnan(lse[0, :2]).all() and torch.equal(lse[0, 2:], want[1][0, 2:])


def test_other_device_is_not_needed_to_be_current_and_python_lists_work():
    q, cache, table, lens, mod, kw, _ = attend_case("gqa4_t1_f8")
    a = pf.flash_attention_paged(q, cache, table.long(), lens, mod, **kw)
    b = pf.flash_attention_paged(q, cache, table.cpu(), torch.tensor(lens), mod, **kw)
    c = pf.flash_attention_paged(q, cache, table, torch.tensor(lens, device=DEV, dtype=torch.int32), mod, **kw)
    assert all(torch.equal(x, y) for x, y in zip(a, b)) and all(torch.equal(x, y) for x, y in zip(a, c))


def test_runs_are_bitwise_repeatable_and_streams_independent():
    q, cache, table, lens, mod, kw, _ = attend_case("long_and_short")
    want = pf.flash_attention_paged(q, cache, table, lens, mod, **kw)
    q2, c2, t2, l2, m2, kw2, _ = attend_case("one_long")
    want2 = pf.flash_attention_paged(q2, c2, t2, l2, m2, **kw2)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        with torch.cuda.stream(streams[0]):
            got.append((pf.flash_attention_paged(q, cache, table, lens, mod, **kw), want))
        with torch.cuda.stream(streams[1]):
            got.append((pf.flash_attention_paged(q2, c2, t2, l2, m2, **kw2), want2))
    torch.cuda.synchronize()
    for g, w in got:
        assert torch.equal(g[0], w[0]) and torch.equal(g[1], w[1])


# ------------------------------------------------------------------------------- appends
# B, H, Hkv, T, D, in dtype, cache dtype, ps, rotary_dim, interleaved, starts, new_lens
APPEND = {
    "token_f8": (5, 4, 2, 1, 128, BF16, F8, 64, 128, False, [0, 63, 64, 100, 130], None),
    "token_bf16": (3, 2, 1, 1, 64, BF16, BF16, 16, 64, True, [0, 15, 33], None),
    "drafts_f8": (3, 4, 4, 5, 64, BF16, F8, 16, 32, True, [14, 0, 31], [5, 3, 0]),
    "warp_edge_f8": (2, 0, 1, 16, 128, BF16, F8, 32, 128, False, [5, 20], None),
    "block_edge_f8": (2, 0, 1, 17, 128, BF16, F8, 32, 128, False, [5, 31], None),
    "prompt_f8": (3, 8, 2, 300, 128, BF16, F8, 64, 128, False, [0, 77, 64], [300, 123, 299]),
    "prompt_bf16_part": (2, 3, 3, 131, 64, BF16, BF16, 16, 32, True, [9, 0], [131, 64]),
    "prompt_fp32_d256": (2, 2, 1, 150, 256, F32, F8, 128, 64, False, [100, 3], None),
    "prompt_d256": (2, 2, 1, 150, 256, BF16, F8, 128, 256, True, [100, 3], None),
    "prompt_large_pages": (2, 2, 2, 200, 128, BF16, F8, 128, 128, False, [60, 0], [200, 129]),
    "far_f8": (1, 2, 1, 70, 128, BF16, F8, 128, 128, False, [200001], None),
    "fp32_into_bf16": (1, 2, 2, 40, 128, F32, BF16, 32, 128, True, [30], None),
    "no_rotary": (2, 2, 1, 50, 128, BF16, F8, 16, 0, False, [7, 0], None),
    "small_pages_d64": (2, 1, 1, 100, 64, BF16, F8, 16, 64, False, [3, 16], [100, 1]),
}


def append_case(name, layout="hnd"):
    B, H, Hkv, T, D, dt, cdt, ps, rd, inter, starts, new = APPEND[name]
    g = torch.Generator().manual_seed(sum(map(ord, name)))
    new_l = new or [T] * B
    lens = [s + n for s, n in zip(starts, new_l)]
    cols = max(1, -(-max(lens) // ps)) + 1
    cache = make_cache(B * cols + 1, Hkv, ps, D, cdt, g, layout)
    table = make_table(B, cols, B * cols + 1, g)
    amp = torch.exp(torch.randn(D, generator=g))
    q, k, v = ((torch.randn(B, T, h, D, generator=g) * amp).to(DEV, dt).transpose(1, 2) for h in (H, Hkv, Hkv))
    spec = pf.rotary_spec(D, rotary_dim=rd, interleaved=inter) if rd else None
    return cache, table, lens, new_l, new, q, k, v, spec


def copy_of(cache):
    return [None if t is None else t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]


def check_append(cache, before, table, lens, new, q, out, k, v, spec):
    ps, f8 = cache.page_size, cache.k_scale is not None
    for which, (pool, old, x) in enumerate(((cache.k, before[0], k), (cache.v, before[1], v))):
        scale, old_s = ((cache.k_scale, before[2]), (cache.v_scale, before[3]))[which] if f8 else (None, None)
        want_same = torch.ones(pool.shape[:3], dtype=torch.bool, device=DEV)  # rows that must not change
        scale_same = torch.ones(pool.shape[:2], dtype=torch.bool, device=DEV)
        for b, (n, t) in enumerate(zip(lens, new)):
            pos = torch.arange(n - t, n, device=DEV)
            if which == 0 and spec is not None:
                ref, err = rotate64(x[b, :, :t], spec, pos)
            else:
                ref, err = x[b, :, :t].double(), torch.zeros_like(x[b, :, :t].double())
            for c in range((n - t) // ps, -(-n // ps) if t else 0):
                page, lo, hi = int(table[b, c]), max(c * ps, n - t), min(n, c * ps + ps)
                r, e = ref[:, lo - (n - t): hi - (n - t)], err[:, lo - (n - t): hi - (n - t)]
                got = pool[page, :, lo - c * ps: hi - c * ps].double()
                want_same[page, :, lo - c * ps: hi - c * ps] = False
                if not f8:
                    assert_within("rows", got, r, e + unit(torch.bfloat16) * r.abs())
                    continue
                top = r.abs().amax((1, 2))
                s = scale_for(top)
                held = lo > c * ps
                if held:
                    s = torch.maximum(s, old_s[page].double())
                # the inputs keep clear of the border at which a scale doubles
                assert bool(((top / (448 * scale_for(top))) < 1 - 1e-5).all()) or which == 1
                assert torch.equal(scale[page].double(), s)
                scale_same[page] = False
                code = r / s[:, None, None]
                assert_within("codes", got, code, 0.5 * e4m3_step(code.abs() * (1 + 1e-6)) + e / s[:, None, None])
                if not bool(e.any()):
                    assert torch.equal(got, to_e4m3_64(code))
                if held:  # requantised when the scale grew, else untouched
                    ratio = (old_s[page].double() / s)[:, None, None]
                    want = to_e4m3_64(old[page, :, : lo - c * ps].double() * ratio)
                    assert torch.equal(pool[page, :, : lo - c * ps].double(), want)
                    want_same[page, :, : lo - c * ps] = False
        assert torch.equal(pool.float()[want_same], old.float()[want_same])
        if f8:
            assert torch.equal(scale[scale_same], old_s[scale_same])
    for b, (n, t) in enumerate(zip(lens, new)):
        if out is None:
            break
        pos = torch.arange(n - t, n, device=DEV)
        ref, err = rotate64(q[b, :, :t], spec, pos) if spec is not None else (q[b, :, :t].double(), 0.0)
        assert_within("q", out[b, :, :t], ref, err + unit(q.dtype) * ref.abs() + 1e-37)
        assert torch.all(out[b, :, t:] == 0)


@pytest.mark.parametrize("name", list(APPEND))
def test_append_matches_the_definition(name):
    cache, table, lens, new, new_arg, q, k, v, spec = append_case(name)
    before = copy_of(cache)
    out = pf.paged_kv_append(cache, table, lens, k, v, new_lens=new_arg, rotary=spec, q=q if q.shape[1] else None)
    check_device_status(DEV)
    check_append(cache, before, table, lens, new, q, out, k, v, spec)


@pytest.mark.parametrize("name", ["prompt_f8", "drafts_f8", "prompt_bf16_part"])
def test_append_token_major_pages_and_misaligned_inputs(name):
    cache, table, lens, new, new_arg, q, k, v, spec = append_case(name, layout="nhd")

    def odd(x):
        y = torch.empty(x.numel() + 1, dtype=x.dtype, device=DEV)[1:].view(x.shape)
        return y.copy_(x)

    before = copy_of(cache)
    q, k, v = odd(q), odd(k), odd(v)
    out = pf.paged_kv_append(cache, table, lens, k, v, new_lens=new_arg, rotary=spec, q=q)
    check_append(cache, before, table, lens, new, q, out, k, v, spec)


def test_append_special_values():
    cache = pf.PagedKVCache.empty(4, 1, 16, 64, F8, DEV)
    table = torch.tensor([[2, 1]], device=DEV, dtype=torch.int32)
    k = torch.zeros(1, 1, 6, 64, device=DEV, dtype=F32)
    v = k.clone()
    v[0, 0, 0, 0], v[0, 0, 1, 1], v[0, 0, 2, 2], v[0, 0, 3, 3] = math.inf, math.nan, -math.inf, 3.0
    pf.paged_kv_append(cache, table, [6], k, v)
    assert float(cache.k_scale[2, 0]) == 2.0 ** -100 and torch.all(cache.k[2].float() == 0)
    s = float(cache.v_scale[2, 0])
    got = cache.v[2, 0].float() * s
    assert s == 2.0 ** -7 and got[0, 0] == 448 * s and got[2, 2] == -448 * s and got[3, 3] == 3.0
    assert torch.isnan(got[1, 1]) and int(torch.isnan(got).sum()) == 1
    # all-zero rows held: the scale grows from 2^-100 to whatever comes
    k[..., 0] = 1e30
    pf.paged_kv_append(cache, table, [8], k[:, :, :2], v[:, :, 4:6])
    assert float(cache.k_scale[2, 0]) == float(scale_for(k[0, 0, 0, 0].cpu()))
    # a page whose row 0 is written anew starts over
    pf.paged_kv_append(cache, table, [1], k[:, :, :1] * 0 + 1, v[:, :, 3:4])
    assert float(cache.k_scale[2, 0]) == 2.0 ** -8 and float(cache.k[2, 0, 0, 0]) * 2.0 ** -8 == 1.0
    # 448 * 2^e fits exactly, the next fp32 does not
    for top, s in ((448.0, 1.0), (math.nextafter(448.0, 1e9) + 1e-4, 2.0), (224.0, 0.5), (2.0 ** -118, 2.0 ** -100)):
        x = torch.full((1, 1, 1, 64), top, device=DEV)
        pf.paged_kv_append(cache, table, [1], x, x)
        assert float(cache.k_scale[2, 0]) == s, (top, s)


def test_append_bad_lengths_and_pages_write_nothing():
    cache, table, lens, new, _, q, k, v, spec = append_case("drafts_f8")
    for tb, ln, nl in ((None, [19, -1, 31], [5, 3, 0]), (None, [19, 2, 31], [5, 3, 0]), (None, [19, 3, 31], [6, 3, 0]),
                       (None, [10 ** 6, 3, 31], [5, 3, 0]), (-1, lens, new), (cache.k.shape[0], lens, new)):
        before = copy_of(cache)
        t = table.clone()
        if tb is not None:
            t[0, 0] = tb
        pf.paged_kv_append(cache, t, ln, k, v, new_lens=nl, rotary=spec)
        with pytest.raises(L.FlexAttnError, match="out of range"):
            check_device_status(DEV)
        bad = 0 if tb is not None or ln[1] == 3 else 1
        pages = [int(p) for p in (table[bad] if tb is None else table[0, :1])]
        for a, b in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), before):
            assert torch.equal(a.float()[pages], b.float()[pages])


# ------------------------------------------------------------------------------- as they are used
def _serve(dtype, steps=9, D=128, ps=16):
    """A small server: prompts, then tokens one by one, each step an append and an attention."""
    g = torch.Generator().manual_seed(21)
    B, H, Hkv, T = 3, 8, 2, 41
    cache = pf.PagedKVCache.empty(B * 6 + 1, Hkv, ps, D, dtype, DEV)
    table = make_table(B, 6, B * 6 + 1, g)
    spec = pf.rotary_spec(D, interleaved=True, scaling=pf.by_parts_scaling(4.0, 32))
    new = torch.tensor([41, 7, 20], dtype=torch.int32, device=DEV)
    lens = new.clone()
    history = [[] for _ in range(B)]
    steps_in = [(new, *(torch.randn(B, h, T, D, generator=g).to(DEV, BF16) for h in (H, Hkv, Hkv)))]
    for _ in range(steps):
        steps_in.append((torch.ones_like(new), *(torch.randn(B, h, 1, D, generator=g).to(DEV, BF16) for h in (H, Hkv, Hkv))))
    return B, H, Hkv, D, cache, table, spec, lens, history, steps_in


@pytest.mark.parametrize("dtype", [BF16, F8])
def test_prompt_and_decode_steps_together(dtype):
    """The run of both operators against plain attention over everything that was appended.

    bf16 pages: each cached value is off by 2^-8 relative at most; 8-bit ones by 2^-4 per value when
    written and once more when a page's scale grew (the ratio of scales is a power of two, so a second
    rounding only meets values that fall below the smallest step)."""
    B, H, Hkv, D, cache, table, spec, lens, history, steps = _serve(dtype)
    for i, (new, q, k, v) in enumerate(steps):
        if i:
            lens += 1
        rq = pf.paged_kv_append(cache, table, lens, k, v, new_lens=new, rotary=spec, q=q)
        o, lse = pf.flash_attention_paged(rq, cache, table, lens, pf.causal_mask, q_lens=new)
        check_device_status(DEV)
        n, t = lens.tolist(), new.tolist()
        # the attention against what the cache holds
        ro, rl, to, tl = attend64(rq, cache, table, n, t, "causal", 0, None, 0, 1 / math.sqrt(D))
        assert_within("lse", lse, rl, tl)
        assert_within("o", o, ro, to)
        # and what the cache holds against what was given
        for b in range(B):
            pos = torch.arange(n[b] - t[b], n[b], device=DEV)
            history[b].append((rotate64(k[b, :, : t[b]], spec, pos)[0], v[b, :, : t[b]].double()))
            kk, vv = cache.gather(table[b])
            u = 2.0 ** -8 if dtype == BF16 else U_E4M3
            for got, want in ((kk, torch.cat([h[0] for h in history[b]], 1)), (vv, torch.cat([h[1] for h in history[b]], 1))):
                got = got[:, : n[b]].double()
                top = want.abs().amax((1, 2), keepdim=True)
                low = 0 if dtype == BF16 else 2 * top * 2.0 ** -17  # two smallest steps of 2^-9 / 2 with 448 s < 2 top
                assert_within("held", got, want, want.abs() * (u * (1 + 1e-3) + 1e-6) + low + 1e-6 * top)


@pytest.mark.parametrize("dtype", [BF16, F8])
def test_captured_step_replays_at_every_length(dtype):
    """One captured graph of a decode step serves the growing lengths; two graphs are alive at once."""
    B, H, Hkv, D, cache, table, spec, lens, _, steps = _serve(dtype, steps=12)
    new, q, k, v = steps[0]
    pf.paged_kv_append(cache, table, lens, k, v, new_lens=new, rotary=spec, q=q)
    eager = pf.PagedKVCache(*[t.clone() for t in (cache.k, cache.v)],
                            *([] if dtype == BF16 else [t.clone() for t in (cache.k_scale, cache.v_scale)]))
    xq, xk, xv = (t.clone() for t in steps[1][1:])
    glens = lens + 1

    def step(c, ln, q, k, v):
        rq = pf.paged_kv_append(c, table, ln, k, v, rotary=spec, q=q)
        return pf.flash_attention_paged(rq, c, table, ln, pf.causal_mask)

    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(cache, glens, xq, xk, xv)
        graphs.append((graph, out))
    glens.copy_(lens)
    for i, (_, q, k, v) in enumerate(steps[1:]):
        glens += 1
        for x, y in ((xq, q), (xk, k), (xv, v)):
            x.copy_(y)
        graph, out = graphs[i & 1]
        graph.replay()
        want = step(eager, glens.clone(), q, k, v)
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
        assert torch.equal(cache.k.float(), eager.k.float()) and torch.equal(cache.v.float(), eager.v.float())
    check_device_status(DEV)


def test_agrees_with_the_contiguous_decode():
    """bf16 pages that hold a contiguous cache: flash_attention_decode's answer, within both kernels' bounds."""
    g = torch.Generator().manual_seed(4)
    B, H, Hkv, Tq, D, ps, T = 3, 16, 4, 2, 128, 64, 640
    k, v = (torch.randn(B, Hkv, T, D, generator=g).to(DEV, BF16) for _ in range(2))
    q = torch.randn(B, H, Tq, D, generator=g).to(DEV, BF16)
    pages = [x.view(B, Hkv, T // ps, ps, D).transpose(1, 2).reshape(-1, Hkv, ps, D).contiguous() for x in (k, v)]
    cache = pf.PagedKVCache(*pages)
    table = torch.arange(B * T // ps, device=DEV, dtype=torch.int32).view(B, -1)
    lens = [640, 333, 65]
    o, lse = pf.flash_attention_paged(q, cache, table, lens, pf.causal_mask)
    o2, lse2 = pf.flash_attention_decode(q, k, v, lens, pf.causal_mask)
    _, _, to, tl = attend64(q, cache, table, lens, [Tq] * B, "causal", 0, None, 0, 1 / math.sqrt(D))
    assert_within("o", o, o2.double(), 2 * to)
    assert_within("lse", lse, lse2.double(), 2 * tl)


# ------------------------------------------------------------------------------- refusals
def test_refusals():
    g = torch.Generator().manual_seed(1)
    cache = make_cache(8, 2, 16, 64, F8, g)
    table = make_table(2, 3, 8, g)
    q = torch.randn(2, 4, 1, 64, device=DEV).to(BF16)
    k = torch.randn(2, 2, 1, 64, device=DEV).to(BF16)
    lens = [5, 6]
    attend, append = pf.flash_attention_paged, pf.paged_kv_append
    for bad in (lambda: attend(q.float(), cache, table, lens), lambda: attend(q[0], cache, table, lens),
                lambda: attend(q[:, :3], cache, table, lens), lambda: attend(q.cpu(), cache, table, lens),
                lambda: attend(q[..., :32], cache, table, lens), lambda: attend(q, cache, table[:1], lens),
                lambda: attend(q, cache, table[0], lens), lambda: attend(q, cache, table.float(), lens),
                lambda: attend(q, cache, table, [5]), lambda: attend(q, cache, table, [5.0, 6.0]),
                lambda: attend(q.clone().requires_grad_(True), cache, table, lens),
                lambda: append(cache, table, lens, k, k[:, :1]), lambda: append(cache, table, lens, k[:, :1], k[:, :1]),
                lambda: append(cache, table, lens, k.half(), k.half()), lambda: append(cache, table, lens, k, k.float()),
                lambda: append(cache, table, lens, k, k, q=q.float()), lambda: append(cache, table, lens, k, k, q=q[:1]),
                lambda: append(cache, table, lens, k, k, rotary=pf.rotary_spec(32)),
                lambda: append(cache, table, lens, k.cpu(), k.cpu()),
                lambda: append(cache, table, lens, k.clone().requires_grad_(True), k),
                lambda: pf.PagedKVCache(cache.k, cache.v), lambda: pf.PagedKVCache(cache.k, cache.v, cache.k_scale[:1], cache.v_scale),
                lambda: pf.PagedKVCache(cache.k.cpu(), cache.v.cpu(), cache.k_scale, cache.v_scale),
                lambda: pf.PagedKVCache(cache.k.to(BF16), cache.v.to(BF16), cache.k_scale, cache.v_scale),
                lambda: pf.PagedKVCache(cache.k.float(), cache.v.float()),
                lambda: pf.PagedKVCache(cache.k[:1].expand(8, -1, -1, -1), cache.v, cache.k_scale, cache.v_scale)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: attend(q, cache, table, lens, pf.document_mask([3, 3])),
                lambda: attend(q, cache, table, lens, score_mod=pf.relative_bias_score_mod(torch.zeros(1, 1))),
                lambda: pf.PagedKVCache.empty(4, 1, 24, 64, F8, DEV), lambda: pf.PagedKVCache.empty(4, 1, 16, 96, F8, DEV)):
        with pytest.raises(NotImplementedError):
            bad()
    with pytest.raises(L.FlexAttnError):
        append(cache, table, lens, k, k, rotary=pf.rotary_spec(64, rotary_dim=24))


def test_empty_batches():
    cache = pf.PagedKVCache.empty(4, 1, 16, 64, BF16, DEV)
    table = torch.zeros(2, 1, dtype=torch.int32, device=DEV)
    o, lse = pf.flash_attention_paged(torch.empty(2, 2, 0, 64, device=DEV, dtype=BF16), cache, table, [0, 0])
    assert o.shape == (2, 2, 0, 64) and lse.shape == (2, 2, 0)
    e = torch.empty(2, 1, 0, 64, device=DEV, dtype=BF16)
    assert pf.paged_kv_append(cache, table, [0, 0], e, e) is None
    o, lse = pf.flash_attention_paged(torch.ones(2, 2, 1, 64, device=DEV, dtype=BF16), cache, table, [0, 0])
    assert torch.all(o == 0) and torch.all(lse == -math.inf)
    check_device_status(DEV)
