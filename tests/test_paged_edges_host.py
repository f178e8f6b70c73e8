"""Paged caches and rotary positions at the edges of what their calls document, without a GPU."""
import ctypes as C
import random
import re
from pathlib import Path

import numpy as np
import pytest
import torch

import pallas_flexattn as pf
from paged_reference import rotate64
from pallas_flexattn import _lib as L
from pallas_flexattn import flash_attn as F
from pallas_flexattn import paged as P
from pallas_flexattn import rotary as R

CSRC = Path(__file__).resolve().parent.parent / "pallas-flexattn_b200" / "csrc"


def test_a_wait_that_gave_up_is_reported_whichever_warp_it_was():
    """No wait can be made to run out from outside, so this reads the source: the timeout is reported behind the
    barrier that all warps of a CTA reach after their last wait, and every wait's failure sets the flag."""
    src = (CSRC / "fa_paged.cu").read_text()
    kernel = src[src.index("paged_attn_kernel("):src.index("int sm_count()")]
    report = kernel.index("report_status(a.status, FA_ERR_TIMEOUT)")
    waits = [m.start() for m in re.finditer(r"\b(?:wait_for|wait_for_w|mbar_wait_w|mbar_try_wait)\(", kernel)]
    assert len(waits) > 15 and kernel.count("FA_ERR_TIMEOUT") == 1
    assert "__syncthreads();" in kernel[max(waits):report]
    for at in waits:
        start = max(kernel.rindex(c, 0, at) for c in ";{}") + 1
        used = kernel[start:at].strip()
        assert used, f"a wait whose result is dropped: {kernel[at:at + 80]}"


def test_a_status_word_of_a_capture_is_not_the_devices(monkeypatch):
    """A word made inside a stream capture is memory of that graph: it is never cached as the device's."""
    on = {"capturing": True}
    zeros = torch.zeros
    monkeypatch.setattr(F, "_STATUS", {})
    monkeypatch.setattr(F, "_STATUS_PTR", {})
    monkeypatch.setattr(F, "_GRAPH_STATUS", {})
    monkeypatch.setattr(F, "_capturing", lambda dev: on["capturing"])
    monkeypatch.setattr(torch, "zeros", lambda *a, device=None, **kw: zeros(*a, **kw))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda dev: type("S", (), {"synchronize": lambda self: None})())
    with pytest.raises(RuntimeError, match="check_device_status"):
        F.status_ptr(0)
    graph = F.device_status("cuda:0")
    on["capturing"] = False
    word = F.device_status("cuda:0")
    assert word is not graph and F.device_status("cuda:0") is word and F.status_ptr(0) == word.data_ptr()
    on["capturing"] = True
    assert F.device_status("cuda:0") is word and F.status_ptr(0) == word.data_ptr()
    for w in (word, graph):
        w.fill_(L.FA_ERR_INVALID)
        with pytest.raises(L.FlexAttnError, match="out of range"):
            F.check_device_status("cuda:0")
        assert int(w) == 0
        F.check_device_status("cuda:0")


def _plain_launch(q, k, spec, positions, inverse):
    pos = positions if positions is not None else torch.arange((q if q is not None else k).shape[2])
    plain = [None if x is None else torch.from_numpy(torch.autograd.forward_ad.unpack_dual(x).primal.detach().numpy().copy())
             for x in (q, k)]  # as opaque to differentiation as a kernel
    return tuple(None if x is None else rotate64(x, spec, pos, inverse)[0].to(x.dtype) for x in plain)


@pytest.mark.parametrize("case", ["q", "k", "both", "no_grad", "requires_grad", "given"])
def test_tangents_of_the_rotation(monkeypatch, case):
    """Forward-mode tangents turn like their primals (the launch is replaced by the formula)."""
    fw = torch.autograd.forward_ad
    monkeypatch.setattr(R, "_launch", _plain_launch)
    monkeypatch.setattr(R, "_check_qk", lambda q, k, spec: None)
    spec = pf.rotary_spec(16, rotary_dim=8, interleaved=True, scaling=pf.by_parts_scaling(4.0, 64))
    g = torch.Generator().manual_seed(0)
    q, k, tq, tk = (torch.randn(1, 2, 5, 16, generator=g, dtype=torch.float64) for _ in range(4))
    pos = torch.tensor([4, 0, 9, 100, 7], dtype=torch.int32) if case == "given" else None
    q.requires_grad_(case == "requires_grad")
    with fw.dual_level(), torch.set_grad_enabled(case != "no_grad"):
        dq = fw.make_dual(q, tq) if case != "k" else q
        dk = fw.make_dual(k, tk) if case != "q" else k
        oq, ok = R.rotary_embedding(dq, dk, spec, pos)
        want = _plain_launch(tq, tk, spec, pos, False)
        for o, d, w in ((oq, dq, want[0]), (ok, dk, want[1])):
            t = fw.unpack_dual(o).tangent
            if fw.unpack_dual(d).tangent is None:
                assert t is None
            else:
                assert torch.allclose(t, w, atol=1e-12)
    if case == "requires_grad":
        gq, = torch.autograd.grad(oq, q, tq)
        assert torch.allclose(gq, _plain_launch(tq, None, spec, pos, True)[0], atol=1e-12)


def test_tangents_are_refused_where_there_is_no_gradient():
    """Appends and paged attention have no gradient, so neither a tangent."""
    fw = torch.autograd.forward_ad
    x = torch.zeros(1, 1, 1, 64, dtype=torch.bfloat16)
    cache = P.PagedKVCache.__new__(P.PagedKVCache)
    cache._shape, cache._device, cache._plans = (1, 1, 16, 64), torch.device("cpu"), {}
    table, lens = torch.zeros(1, 1, dtype=torch.int32), [1]
    with fw.dual_level(), torch.no_grad():
        d = fw.make_dual(x, x)
        for call in (lambda: P.flash_attention_paged(d, cache, table, lens),
                     lambda: P.paged_kv_append(cache, table, lens, d, x),
                     lambda: P.paged_kv_append(cache, table, lens, x, d),
                     lambda: P.paged_kv_append(cache, table, lens, x, x, q=d)):
            with pytest.raises(ValueError, match="tangent"):
                call()


def test_positions_that_are_no_integers_are_refused(monkeypatch):
    monkeypatch.setattr(R, "_launch", lambda q, k, spec, positions, inverse: positions)
    monkeypatch.setattr(R, "_check_qk", lambda q, k, spec: None)
    spec, q = pf.rotary_spec(16), torch.zeros(1, 1, 3, 16)
    for bad in (2.5, "4", [1, 2, 3], 1e20, object(), (1 << 31) - 2, -(1 << 31) - 1):
        with pytest.raises(ValueError, match="positions"):
            R.rotary_embedding(q, None, spec, bad)
    for good in (0, 7, -5, (1 << 31) - 3, -(1 << 31), np.int64(12)):
        assert R.rotary_embedding(q, None, spec, good) == good


@pytest.mark.parametrize("dtype", [torch.int64, torch.uint32, torch.int32, torch.int16])
def test_numbers_beyond_32_bits_stay_out_of_range(dtype):
    """Lengths and page numbers are handed to the kernels as 32 bits: one that does not fit must not wrap into range."""
    cpu = torch.device("cpu")
    values = [0, 5, 300]
    if dtype == torch.int64:
        values += [(1 << 32) + 5, -(1 << 32), 1 << 62, -(1 << 62), (1 << 31) - 1, -1]
    if dtype == torch.uint32:
        values += [(1 << 32) - 2]
    x = torch.tensor(values, dtype=dtype)
    lo, hi = -(1 << 31), (1 << 31) - 1
    want = [min(max(v, lo), hi) for v in values]
    for got in (P._lengths("kv_lens", x, len(values), cpu), P._table(x[:, None], len(values), cpu)[:, 0]):
        assert got.dtype == torch.int32 and got.tolist() == want
    assert P._lengths("kv_lens", values, len(values), cpu).tolist() == want


class _Barrier:
    """An mbarrier: waits see the parity of its completed phases only."""

    def __init__(self):
        self.done = 0

    def passes(self, use):
        return (self.done & 1) == ((use + 1) & 1)


def _walk_the_ring(slots, tiles, sets, apart, rng, loaders=1):
    """Paged attention's ring of K and V tiles with every role at a random pace: the loader (in order, into a slot
    whose last reader has released it; or one for K and one for V), loads that land in any order, the warp that issues S, `sets` of softmax
    groups that take the tiles in turn, the warp that issues P V.  `apart`: a slot's loads of K and of V complete
    on a barrier each.  Returns what went wrong, or None."""
    turn = slots if slots & 1 else slots // 2
    full = [[_Barrier() for _ in range(slots)] for _ in range(2)]
    empty = [_Barrier() for _ in range(slots)]
    holds, landed, flying = [None] * slots, set(), []
    s_done = pv_done = 0
    issued = list(range(loaders))  # the next load of each
    at, ready = list(range(sets)), set()

    def wait(ld):
        return (full[ld & 1][ld % slots], (ld >> 1) // turn) if apart else (full[0][ld % slots], ld // slots)

    def passes(ld):
        bar, use = wait(ld)
        return bar.passes(use)

    while pv_done < tiles:
        steps = [("load", k) for k, ld in enumerate(issued)
                 if ld < 2 * tiles and (ld < slots or empty[ld % slots].passes(ld // slots - 1))]
        steps += ["land"] * bool(flying)
        if s_done < tiles and (s_done < 2 or s_done - 2 in ready) and passes(2 * s_done):
            steps.append("S")
        steps += [k for k in range(sets) if at[k] < s_done and (at[k] < 2 or pv_done > at[k] - 2)]
        if pv_done in ready and passes(2 * pv_done + 1):
            steps.append("PV")
        if not steps:
            return "deadlock"
        step = rng.choice(steps)
        if isinstance(step, tuple):
            ld = issued[step[1]]
            if empty[ld % slots].done < ld // slots:
                return f"load {ld} into a slot in use"
            holds[ld % slots] = ld
            flying.append(ld)
            issued[step[1]] += loaders
        elif step == "land":
            ld = flying.pop(rng.randrange(len(flying)))
            landed.add(ld)
            wait(ld)[0].done += 1
        elif step in ("S", "PV"):
            ld = 2 * s_done if step == "S" else 2 * pv_done + 1
            if ld not in landed or holds[ld % slots] != ld:
                return f"{step} of tile {ld >> 1} before its load has landed"
            empty[ld % slots].done += 1
            s_done, pv_done = s_done + (step == "S"), pv_done + (step == "PV")
        else:
            ready.add(at[step])
            at[step] += sets
    return None


@pytest.mark.parametrize("sets", [1, 2])
def test_the_ring_of_tiles_at_every_depth_and_any_pace(sets):
    """With one barrier a slot, rings of 3 and 5 slots let S start on a tile that has not landed (head dim 256, and
    bf16 of head dim 128 at 32 rows); with one for K and one for V no ring does."""
    def faults(slots, apart, n):
        return sum(_walk_the_ring(slots, 30, sets, apart, random.Random(seed)) is not None for seed in range(n))

    for slots in range(2, 25):
        assert faults(slots, True, 60) == 0
        assert (faults(slots, False, 60) > 0) == (slots in (3, 5))
    for slots in (6, 13, 24):  # two loaders: 8 rows of head dim 256, 128, 64 (odd rings below 9 would not do)
        assert sum(_walk_the_ring(slots, 40, 2, True, random.Random(seed), 2) is not None for seed in range(60)) == 0
    src = (CSRC / "fa_paged.cu").read_text()
    assert "full_k[kMaxSlots], full_v[kMaxSlots]" in src


def test_rotary_offsets_that_leave_32_bits_are_refused():
    """Token t sits at pos_offset + t, a 32-bit sum on the device."""
    p = L.FaRotaryParams()
    p.dtype, p.B, p.H, p.T, p.D = L.FA_DTYPE_BF16, 1, 1, 4, 64
    p.q = p.q_out = L.FaTensor(4096, 256, 256, 64)  # never dereferenced: validation fails first
    p.rotary = L.FaRotarySpec(64, L.FA_ROTARY_HALF, 4096, 1.0)
    p.pos_offset = (1 << 31) - 3
    assert L.lib().fa_rotary(C.byref(p), None) == L.FA_ERR_INVALID and b"32 bits" in L.lib().fa_last_error()
