"""Paged caches at the edges of what their calls document: rows that see nothing next to NaN, scales that are
not positive numbers, empty slots, a first call inside a capture, streams."""
import math

import pytest
import torch

import pallas_flexattn as pf
from pallas_flexattn import _lib as L
from pallas_flexattn.flash_attn import check_device_status
from paged_reference import assert_within, attend64

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0) if torch.cuda.is_available() else None
BF16, F8 = torch.bfloat16, torch.float8_e4m3fn


def cache_of(pages, hkv, ps, D, dtype, g):
    pools = [torch.randn(pages, hkv, ps, D, generator=g) for _ in range(2)]
    if dtype == BF16:
        return pf.PagedKVCache(*[x.to(DEV, BF16) for x in pools])
    scales = [torch.full((pages, hkv), 2.0 ** -6, device=DEV) for _ in range(2)]
    return pf.PagedKVCache(*[(x * 64).clamp(-448, 448).to(DEV).to(F8) for x in pools], *scales)


# B, H, Hkv, Tq, D, lens, q_lens: units inside one CTA, and units that are cut
PADDED = {
    "whole_r8": (3, 2, 2, 3, 128, [100, 90, 128], [1, 0, 2]),
    "whole_r32": (2, 8, 2, 6, 64, [60, 120], [2, 5]),
    "whole_r64": (2, 8, 1, 8, 128, [128, 70], [3, 1]),
    "cut_r8": (2, 4, 2, 4, 128, [9000, 5000], [1, 3]),
    "cut_r32": (1, 8, 1, 4, 256, [7000], [2]),
    "cut_r64": (1, 16, 1, 20, 64, [20000], [9]),
    "before_the_start": (2, 4, 1, 5, 128, [3, 2], None),
}


@pytest.mark.parametrize("special", [math.nan, math.inf])
@pytest.mark.parametrize("dtype", [F8, BF16])
@pytest.mark.parametrize("name", list(PADDED))
def test_rows_that_see_nothing_are_zero_next_to_nan(name, dtype, special):
    """A value that every live row sees is NaN or infinite: it reaches its element of those rows, and no row of
    padding or before the sequence's start."""
    B, H, hkv, Tq, D, lens, qlens = PADDED[name]
    g = torch.Generator().manual_seed(len(name))
    cols = -(-max(lens) // 64)
    cache = cache_of(B * cols, hkv, 64, D, dtype, g)
    table = torch.arange(B * cols, device=DEV, dtype=torch.int32).view(B, cols)
    cache.v[table[:, 0].long(), :, 0, 5] = torch.full((1,), special, device=DEV).to(dtype)  # (8 bits have no infinity: NaN)
    q = torch.randn(B, H, Tq, D, generator=g).to(DEV, BF16)
    o, lse = pf.flash_attention_paged(q, cache, table, lens, pf.causal_mask, q_lens=qlens)
    check_device_status(DEV)
    t = torch.tensor(qlens or [Tq] * B, device=DEV)[:, None]
    i = torch.arange(Tq, device=DEV)
    live = ((i < t) & (torch.tensor(lens, device=DEV)[:, None] - t + i >= 0))[:, None].expand(B, H, Tq)
    assert bool(live.any()) and not bool(live.all())
    assert torch.all(o[~live] == 0) and torch.all(lse[~live] == -math.inf)
    hit = torch.zeros(D, dtype=torch.bool, device=DEV)
    hit[5] = True
    assert not torch.isfinite(o[live][:, hit]).any()
    assert torch.isfinite(o[live][:, ~hit]).all() and torch.isfinite(lse[live]).all()
