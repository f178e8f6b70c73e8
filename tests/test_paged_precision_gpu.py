"""Paged attention where the sizes of value scales lie far apart, against 64 bits."""
import math

import pytest
import torch

import pallas_flexattn as pf
from pallas_flexattn.flash_attn import check_device_status
from paged_reference import assert_within, attend64

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0) if torch.cuda.is_available() else None
BF16, F8 = torch.bfloat16, torch.float8_e4m3fn


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
