"""Paged caches at the edges of what their calls document: rows that see nothing next to NaN, scales that are
not positive numbers, empty slots, a first call inside a capture, streams."""
import math

import pytest
import torch

import pallas_flexattn as pf
from pallas_flexattn import _lib as L
from pallas_flexattn.flash_attn import check_device_status
from paged_reference import assert_within, attend64, rotate64, unit

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


@pytest.mark.parametrize("G,Tq,D", [(4, 1, 128), (12, 1, 64), (8, 3, 128), (8, 8, 256)])
def test_value_scales_that_are_not_positive_numbers(G, Tq, D):
    """value = code * scale whatever the scale: negative ones turn the sign, NaN and infinity reach every row that
    sees the page, and no other head or sequence."""
    g = torch.Generator().manual_seed(D + G)
    cache = cache_of(24, 2, 32, D, F8, g)
    table = torch.randperm(24, generator=g).view(2, 12).to(DEV, torch.int32)
    q = torch.randn(2, 2 * G, Tq, D, generator=g).to(DEV, BF16)
    lens = [370, 300]
    cache.v_scale[table[0, 2:5].long(), 0] = -(2.0 ** -5)
    cache.v_scale[table[1, 7].long(), 1] = -(2.0 ** -101)  # counts as zero
    cache.k_scale[table[1, 3].long(), 0] *= -1
    args = (q, cache, table, lens, pf.causal_mask)
    o, lse = pf.flash_attention_paged(*args)
    ro, rl, to, tl = attend64(q, cache, table, lens, [Tq] * 2, "causal", 0, None, 0, 1 / math.sqrt(D))
    # attend64 bounds the logits' sum with log2 vs, of a positive vs: the same for its magnitude
    signed = cache.v_scale.clone()
    cache.v_scale.abs_()
    _, _, to, tl = attend64(q, cache, table, lens, [Tq] * 2, "causal", 0, None, 0, 1 / math.sqrt(D))
    cache.v_scale.copy_(signed)
    assert_within("lse", lse, rl, tl)
    assert_within("o", o, ro, to)
    for bad in (math.nan, math.inf, -math.inf):
        cache.v_scale[table[0, 4].long(), 0] = bad
        o2, lse2 = pf.flash_attention_paged(*args)
        check_device_status(DEV)
        assert torch.isnan(o2[0, :G]).all()
        assert torch.equal(o2[0, G:], o[0, G:]) and torch.equal(o2[1], o[1])
        assert_within("lse", lse2, rl, tl)


CAPTURE_FIRST = """
import torch, pallas_flexattn as pf
from pallas_flexattn import _lib as L
dev = torch.device("cuda", 0)
make = lambda: pf.PagedKVCache(*[torch.randn(4, 1, 16, 64, device=dev).to(torch.bfloat16) for _ in range(2)])
cache = None if {late} else make()
table = torch.tensor([[0, 1]], device=dev, dtype=torch.int32)
lens = torch.tensor([20], device=dev, dtype=torch.int32)
q = torch.randn(1, 2, 1, 64, device=dev).to(torch.bfloat16)
torch.cuda.synchronize()
stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
if {late}:
    pools = [torch.randn(4, 1, 16, 64, device=dev).to(torch.bfloat16) for _ in range(2)]
    try:
        with torch.cuda.graph(graph, stream=stream):
            pf.PagedKVCache(*pools)
    except RuntimeError as e:
        assert "check_device_status" in str(e), e
    else:
        raise SystemExit("made a status word inside a capture")
    torch.cuda.synchronize()
    pf.check_device_status()
    cache, graph = make(), torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, stream=stream):
    out = pf.flash_attention_paged(q, cache, table, lens, pf.causal_mask)
pf.check_device_status()           # nothing has run: nothing is reported
table[0, 1] = 9
graph.replay()                     # a page out of range
table[0, 1] = 1
graph.replay()                     # and one that is fine: the report of the first stays
try:
    pf.check_device_status()
except L.FlexAttnError as e:
    assert "out of range" in str(e)
else:
    raise SystemExit("the report of a replay was lost")
pf.check_device_status()
want = pf.flash_attention_paged(q, cache, table, lens, pf.causal_mask)
assert all(torch.equal(a, b) for a, b in zip(out, want))
print("fine")
"""


@pytest.mark.parametrize("late", [False, True])
def test_a_capture_holds_the_first_call_on_a_device(late):
    """In a fresh process: reports of replays are neither invented nor lost."""
    import subprocess
    import sys

    path = ["pallas-flexattn_b200" if p == "" else p for p in sys.path]
    r = subprocess.run([sys.executable, "-c", f"import sys; sys.path[:0] = {path!r}" + CAPTURE_FIRST.format(late=late)],
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "fine" in r.stdout, r.stdout + r.stderr


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("which", ["q", "k", "both"])
def test_tangents_of_the_rotation(which, dtype):
    """Forward-mode tangents are the rotated tangents, also through a gradient taken backwards."""
    fw = torch.autograd.forward_ad
    g = torch.Generator().manual_seed(1)
    spec = pf.rotary_spec(64, rotary_dim=32, scaling=pf.by_parts_scaling(4.0, 64))
    q, tq, w, tw = (torch.randn(2, 4, 9, 64, generator=g).to(DEV, dtype) for _ in range(4))
    k, tk = (torch.randn(2, 2, 9, 64, generator=g).to(DEV, dtype) for _ in range(2))
    pos = torch.randint(0, 10 ** 6, (9,), generator=g).to(DEV, torch.int32)

    def check(got, x, inverse=False):
        want, err = rotate64(x, spec, pos, inverse)
        assert_within("tangent", got.detach(), want, err + unit(dtype) * want.abs())

    q.requires_grad_(True)
    with fw.dual_level():
        dq = fw.make_dual(q, tq) if which != "k" else q
        dk = fw.make_dual(k, tk) if which != "q" else k
        oq, ok = pf.rotary_embedding(dq, dk, spec, pos)
        check(fw.unpack_dual(oq).primal, q.detach())
        check(fw.unpack_dual(ok).primal, k)
        for o, t, has in ((oq, tq, which != "k"), (ok, tk, which != "q")):
            if has:
                check(fw.unpack_dual(o).tangent.detach(), t)
            else:
                assert fw.unpack_dual(o).tangent is None
        gq, = torch.autograd.grad(oq, q, fw.make_dual(w, tw))
        check(fw.unpack_dual(gq).primal, w, True)
        check(fw.unpack_dual(gq).tangent, tw, True)


def test_a_spec_may_be_dropped_while_another_stream_still_reads_it():
    """The table of a rotary_spec, made by its first call, is not handed out again before calls on other
    streams have read it."""
    g = torch.Generator().manual_seed(2)
    x = torch.randn(1, 2, 16, 128, generator=g).to(DEV, BF16)
    want, _ = pf.rotary_embedding(x, None, pf.rotary_spec(128))
    other = torch.cuda.Stream()
    spec = pf.rotary_spec(128)
    pf.rotary_embedding(x, None, spec)
    torch.empty(64, dtype=torch.int64, device=DEV).fill_(1)  # (a kernel's first launch waits for the device)
    torch.cuda.synchronize()
    at = spec.turns(DEV).data_ptr()
    with torch.cuda.stream(other):
        torch.cuda._sleep(200_000_000)  # some 100 ms
        got, _ = pf.rotary_embedding(x, None, spec)
    del spec
    new = [torch.empty(64, dtype=torch.int64, device=DEV) for _ in range(2000)]  # on the first stream
    for n in new:
        if n.data_ptr() == at:
            n.fill_(1 << 60)
    torch.cuda.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [F8, BF16])
@pytest.mark.parametrize("T", [1, 3, 70])
def test_empty_slots_without_new_lens(T, dtype):
    """kv_lens 0 is an empty slot in both calls of a step, whether or not new_lens says so."""
    g = torch.Generator().manual_seed(T)
    B, lens, spec = 4, [0, T + 5, 0, T], pf.rotary_spec(64)
    q, k, v = (torch.randn(B, h, T, 64, generator=g).to(DEV, BF16) for h in (4, 2, 2))
    table = torch.arange(B * 6, device=DEV, dtype=torch.int32).view(B, 6)
    results = []
    for new in (None, [0, T, 0, T]):
        cache = cache_of(B * 6, 2, 16, 64, dtype, torch.Generator().manual_seed(7))
        before = cache.k.clone()
        rq = pf.paged_kv_append(cache, table, lens, k, v, new_lens=new, rotary=spec, q=q)
        o, lse = pf.flash_attention_paged(rq, cache, table, lens, pf.causal_mask, q_lens=new)
        check_device_status(DEV)
        for b in (0, 2):
            assert torch.all(rq[b] == 0) and torch.all(o[b] == 0) and torch.all(lse[b] == -math.inf)
            assert torch.equal(cache.k[table[b].long()].float(), before[table[b].long()].float())
        results.append((rq, o, lse, cache.k.float(), cache.v.float()))
    assert all(torch.equal(a, b) for a, b in zip(*results))
    pf.paged_kv_append(cache, table, lens, k, v, new_lens=[T] * B)  # tokens for a sequence without a length
    with pytest.raises(L.FlexAttnError, match="out of range"):
        check_device_status(DEV)


# B, H, Hkv, Tq, D, dtype, positions: rings of 5, 3, 5, 3 and 2 slots
FEW_SLOTS = {
    "f8_d256_r32": (8, 64, 2, 1, 256, F8, 16384),
    "f8_d256_r64": (8, 64, 2, 4, 256, F8, 16384),
    "bf16_d128_r32": (8, 64, 2, 1, 128, BF16, 16384),
    "bf16_d256_r16": (8, 16, 2, 1, 256, BF16, 16384),
    "bf16_d256_r32": (8, 64, 2, 1, 256, BF16, 8192),
}


@pytest.mark.parametrize("name", list(FEW_SLOTS))
def test_long_walks_through_rings_of_few_slots(name):
    """Dozens of tiles a CTA where shared memory holds two or three of them, many times: the formula and the same bits."""
    B, H, hkv, Tq, D, dtype, n = FEW_SLOTS[name]
    g = torch.Generator().manual_seed(len(name))
    cols = n // 64
    cache = cache_of(2 * cols, hkv, 64, D, dtype, g)
    table = torch.randperm(2 * cols, generator=g)[:cols].to(DEV, torch.int32).expand(B, -1).contiguous()
    q = torch.randn(1, H, Tq, D, generator=g).to(DEV, BF16)
    qb = q.expand(B, -1, -1, -1).contiguous()
    lens = torch.full((B,), n, dtype=torch.int32, device=DEV)
    o, lse = pf.flash_attention_paged(qb, cache, table, lens, pf.causal_mask)
    ro, rl, to, tl = attend64(q, cache, table[:1], [n], [Tq], "causal", 0, None, 0, 1 / math.sqrt(D))
    for b in range(B):
        assert_within("lse", lse[b:b + 1], rl, tl)
        assert_within("o", o[b:b + 1], ro, to)
    for _ in range(60):
        again = pf.flash_attention_paged(qb, cache, table, lens, pf.causal_mask)
        assert torch.equal(again[0], o) and torch.equal(again[1], lse)
    check_device_status(DEV)


def test_a_score_mod_may_be_dropped_while_another_stream_still_reads_it():
    """The same for the slopes of an ALiBi score mod."""
    g = torch.Generator().manual_seed(4)
    H = 128
    cache = cache_of(8, H, 16, 64, BF16, g)
    table = torch.arange(8, device=DEV, dtype=torch.int32)[None]
    q = torch.randn(1, H, 1, 64, generator=g).to(DEV, BF16)
    lens = torch.tensor([128], device=DEV, dtype=torch.int32)
    attend = lambda mod: pf.flash_attention_paged(q, cache, table, lens, pf.causal_mask, score_mod=mod)  # noqa: E731
    want = attend(pf.alibi_score_mod(H))
    mod = pf.alibi_score_mod(H)
    attend(mod)
    torch.empty(H, device=DEV).fill_(1)
    torch.cuda.synchronize()
    at = mod.__fa_spec__.device_tensors(DEV)["slopes"].data_ptr()
    other = torch.cuda.Stream()
    with torch.cuda.stream(other):
        torch.cuda._sleep(200_000_000)
        got = attend(mod)
    del mod
    new = [torch.empty(H, device=DEV) for _ in range(2000)]
    for n in new:
        if n.data_ptr() == at:
            n.fill_(100.0)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
