"""Paged attention where the sizes of probabilities or of value scales lie far apart, against 64 bits."""
import math

import pytest
import torch

import pallas_flexattn as pf
from pallas_flexattn.flash_attn import check_device_status
from paged_reference import U_BF16, U_F32, assert_within, attend64

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0) if torch.cuda.is_available() else None
BF16, F8 = torch.bfloat16, torch.float8_e4m3fn
TILE = 128


# ------------------------------------------------------------------------------- value scales
@pytest.mark.parametrize("G,Tq", [(4, 1), (12, 1), (8, 3), (8, 8)])
@pytest.mark.parametrize("large,small,zeros", [(24, -8, True), (40, -9, True), (30, -90, False), (60, -9, False),
                                               (41, -41, True), (-50, -99, False)])
def test_the_sum_keeps_weights_on_pages_of_small_values(large, small, zeros, G, Tq):
    """One page of large values among many of small ones, or of none at all (as an append of zeros leaves
    them), logits that spread over 20 nats: o and lse by the formula."""
    g = torch.Generator().manual_seed(large * 100 + G)
    ps, pages, D = 16, 60, 128
    k = (torch.randn(pages, 1, ps, D, generator=g) * 32).clamp(-448, 448)
    v = (torch.randn(pages, 1, ps, D, generator=g) * 90).clamp(-448, 448)
    ks = torch.full((pages, 1), 2.0 ** -5)
    vs = torch.full((pages, 1), 2.0 ** small)
    vs[7] = 2.0 ** large
    if zeros:
        v[9:50], vs[9:50] = 0, 2.0 ** -100
    cache = pf.PagedKVCache(k.to(DEV).to(F8), v.to(DEV).to(F8), ks.to(DEV), vs.to(DEV))
    table = torch.randperm(pages, generator=g).to(DEV, torch.int32)[None]
    q = (torch.randn(1, G, Tq, D, generator=g) * 4).to(DEV, BF16)
    for n in (pages * ps, 500):
        o, lse = pf.flash_attention_paged(q, cache, table, [n], pf.causal_mask)
        check_device_status(DEV)
        ro, rl, to, tl = attend64(q, cache, table, [n], [Tq], "causal", 0, None, 0, 1 / math.sqrt(D))
        assert_within("lse", lse, rl, tl)
        assert_within("o", o, ro, to)


# ------------------------------------------------------------------------------- small probabilities
def running_max_from_the_end(x):
    return x.flip(-1).cummax(-1).values.flip(-1)


def bound(p, v, dx, u=U_BF16):
    """Bound of o's error for probabilities p (rows, n), values v (n, D) and logits off by at most dx.

    Each probability is rounded to 8 bits relative (2^-8; for 8-bit pages in two parts), and there to no finer
    than half the parts' smallest step, 2^-10 of a unit in which the row's largest z so far was brought to at
    least 32.  The unit follows the tiles of 128 positions, walked from the end: when the largest of two tiles of
    a set (all tiles, or every other one) were below 1/2, the next one's is brought to 32, at most 2^20 below
    the largest of all.  So a tile's step is 2^-15 of the largest so far at most, and 2^-15 of its own largest,
    or 2^-9 of that of one of the two tiles before it in the set, or 2^-35 of the row's largest."""
    rows, n = p.shape
    nt = -(-n // TILE)
    pad = torch.nn.functional.pad(p, (0, nt * TILE - n)).view(rows, nt, TILE)
    top = pad.amax(-1)
    before = torch.nn.functional.pad(top, (0, 4)).unfold(-1, 5, 1).amax(-1)  # the tile and four before it
    step = torch.maximum(torch.maximum(2.0 ** -15 * top, 2.0 ** -9 * before), 2.0 ** -35 * top.amax(-1, keepdim=True))
    step = torch.minimum(step, 2.0 ** -15 * running_max_from_the_end(top))
    av = v.abs()
    codes = torch.nn.functional.pad(av, (0, 0, 0, nt * TILE - n)).view(nt, TILE, -1).sum(1)
    return (p @ av) * (u + 2.1 * dx + (n + 64) * 2.0 ** -23) + step @ codes + (p @ v).abs() * U_BF16


def peaked_cache(n, D, offsets, peak, g, ps=64, mean=1.0):
    """One sequence of n positions in 8-bit pages (K in units of 1/8, V of 1/64).  The logits of a row q =
    (8, 8, N(0, 1), ...) are N(0, 1) + offsets[position], and `peak` for the newest, about."""
    k = torch.randn(n, D, generator=g) * 8
    unit = math.sqrt(D) / 8  # what one nat of logit takes in k[:, 0]
    k[:, 0] = offsets * unit * 8
    k[:, 1] = 0
    k[-1] = 0
    k[-1, 1] = peak * unit * 8
    v = ((torch.randn(n, D, generator=g) + mean) * 64).clamp(-440, 440)
    k, v = (x.view(n // ps, 1, ps, D).to(DEV).to(F8) for x in (k, v))
    s = torch.full((n // ps, 1), 1 / 64, device=DEV)
    return pf.PagedKVCache(k, v, s * 8, s)


# name: positions, sequences, G, D, offsets of the tiles in nats by tile, peak of the newest key in nats
PEAKED = {
    "r8_8192": (8192, 296, 4, 128, lambda t: t * 0, 11.0),
    "r8_32768": (32768, 148, 4, 128, lambda t: t * 0, 10.5),
    "r8_d64": (8192, 200, 8, 64, lambda t: t * 0, 12.0),
    "r8_d256": (12288, 160, 3, 256, lambda t: t * 0, 11.5),
    "r16_16384": (16384, 148, 16, 128, lambda t: t * 0, 11.0),
    "r32_8192": (8192, 160, 24, 64, lambda t: t * 0, 11.0),
    "r32_d256": (8192, 150, 20, 256, lambda t: t * 0, 11.0),
    "r64_16384": (16384, 148, 64, 128, lambda t: t * 0, 11.0),
    "steps_down_r8": (16384, 148, 4, 128, lambda t: -4.0 * (t % 5 == 0) + 3.0 * (t % 7 == 0), 13.0),
    "steps_down_r64": (8192, 300, 40, 128, lambda t: -4.0 * (t % 5 == 0) + 3.0 * (t % 7 == 0), 13.0),
    "stairs_r8": (8192, 300, 4, 128, lambda t: (t % 8) * 1.0 - 4.0, 11.0),
    "stairs_r16": (8192, 300, 16, 128, lambda t: 4.0 - (t % 8) * 1.0, 11.0),
    "far_below_r32": (8192, 300, 32, 128, lambda t: 7.0 * (t % 3) - 7.0, 30.0),
}


@pytest.mark.parametrize("name", list(PEAKED))
def test_a_dominant_key_leaves_the_rest_its_weight(name):
    """A newest key far above a long rest: the rest keeps its share of o, not only of the sum.  The sequences
    are many copies of one (they share its pages), so that an SM walks whole units."""
    n, B, G, D, off, peak = PEAKED[name]
    g = torch.Generator().manual_seed(sum(map(ord, name)))
    tiles = torch.arange(n // TILE).repeat_interleave(TILE)
    cache = peaked_cache(n, D, off(tiles).float(), peak, g)
    table = torch.arange(n // 64, device=DEV, dtype=torch.int32).expand(B, -1).contiguous()
    q = torch.randn(1, G, 1, D, generator=g)
    q[..., :2] = 8.0
    q = q.to(DEV, BF16)
    o, lse = pf.flash_attention_paged(q.expand(B, -1, -1, -1), cache, table, [n] * B, pf.causal_mask)
    check_device_status(DEV)
    k, v = (x.double()[0] for x in cache.gather(table[0]))
    q64, scale = q.double()[0, :, 0], 1 / math.sqrt(D)
    s = q64 @ k.T * scale
    # S: exact products summed in fp32, q's two parts exact to 2^-17 of its largest, the product with the scale,
    # the exponent's product and sum
    dx = ((q64.abs() @ k.abs().T * scale) * (D + 16) * 2.0 ** -23
          + 2.0 ** -17 * q64.abs().amax(-1, keepdim=True) * k.abs().sum(-1) * scale + s.abs() * 8 * U_F32 + 2.0 ** -20)
    dx = dx.amax(-1, keepdim=True)
    p = torch.softmax(s, -1)
    tol = bound(p, v, dx)
    want = p @ v
    for b in (0, 1, B // 2, B - 1):
        assert_within("lse", lse[b, :, 0], torch.logsumexp(s, -1),
                      (1.1 * dx[:, 0] + (n + 64) * 2.0 ** -23 + 64 * 4 * U_F32 + 2.0 ** -20))
        assert_within("o", o[b, :, 0], want, tol)


def test_zero_values_under_the_largest_weights():
    """Values of zero where nearly all the weight lies: the sum is large in the unit of the others, and stays
    finite when references go down."""
    g = torch.Generator().manual_seed(3)
    n, ps, D, B = 8192, 64, 128, 160
    k = torch.randn(n // ps, 1, ps, D, generator=g) * 8
    k[..., 0] = 0
    k[60:70, ..., 0] = 24 * math.sqrt(D) / 8 * 8  # the logits of ten pages lie 24 nats above the others'
    v = torch.randn(n // ps, 1, ps, D, generator=g) * 64
    vs = torch.full((n // ps, 1), 1 / 64)
    v[60:70], vs[60:70] = 0, 2.0 ** -100
    cache = pf.PagedKVCache(k.to(DEV).to(F8), v.to(DEV).to(F8), torch.full((n // ps, 1), 1 / 8, device=DEV), vs.to(DEV))
    q = torch.randn(1, 4, 1, D, generator=g)
    q[..., 0] = 8
    q = q.to(DEV, BF16)
    table = torch.arange(n // ps, device=DEV, dtype=torch.int32).expand(B, -1).contiguous()
    o, lse = pf.flash_attention_paged(q.expand(B, -1, -1, -1), cache, table, [n] * B, pf.causal_mask)
    check_device_status(DEV)
    ro, rl, to, tl = attend64(q, cache, table[:1], [n], [1], "causal", 0, None, 0, 1 / math.sqrt(D))
    for b in (0, 1, B // 2, B - 1):
        assert_within("lse", lse[b:b + 1], rl, tl)
        assert_within("o", o[b:b + 1], ro, to)
    vs.fill_(2.0 ** -100)
    cache.k.copy_(torch.randn(k.shape, generator=g).to(F8))
    cache.v_scale.copy_(vs)
    o, lse = pf.flash_attention_paged(q.expand(B, -1, -1, -1), cache, table, [n] * B, pf.causal_mask)
    assert torch.all(o == 0)
    _, rl, _, tl = attend64(q, cache, table[:1], [n], [1], "causal", 0, None, 0, 1 / math.sqrt(D))
    assert_within("lse", lse[:1], rl, tl)
