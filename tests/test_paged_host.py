"""Rotary, paged appends and paged attention without a GPU: structure layouts against the header, refusals
of the C entry points before any CUDA call, the rotary description, and the references themselves."""
import ctypes as C
import math
import shutil
import subprocess
from fractions import Fraction
from pathlib import Path

import pytest
import torch

import pallas_flexattn as pf
from pallas_flexattn import _lib as L
from paged_reference import e4m3_step, rotate64, scale_for, to_e4m3_64

REPO = Path(__file__).resolve().parent.parent
STRUCTS = ["FaRotarySpec", "FaRotaryParams", "FaPagedCache", "FaPagedAppendParams", "FaPagedAttnParams"]


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc not available")
def test_ctypes_layout_matches_header(tmp_path):
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "flexattn.h"', "int main(void) {"]
    for s in STRUCTS:
        lines.append(f'printf("{s} %zu\\n", sizeof({s}));')
        lines += [f'printf("{s}.{f} %zu\\n", offsetof({s}, {f}));' for f, _ in getattr(L, s)._fields_]
    lines += [f'printf("{n} %d\\n", {n});' for n in ("FA_DTYPE_E4M3", "FA_ROTARY_HALF", "FA_ROTARY_INTERLEAVED")]
    (tmp_path / "probe.c").write_text("\n".join(lines + ["return 0;", "}"]))
    exe = tmp_path / "probe"
    subprocess.run(["gcc", "-std=c11", f"-I{REPO / 'include'}", str(tmp_path / "probe.c"), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split("\n")
    got = {k: int(v) for k, v in (line.rsplit(" ", 1) for line in out if line)}
    for s in STRUCTS:
        assert got[s] == C.sizeof(getattr(L, s)), s
        for f, _ in getattr(L, s)._fields_:
            assert got[f"{s}.{f}"] == getattr(getattr(L, s), f).offset, f"{s}.{f}"
    for n in ("FA_DTYPE_E4M3", "FA_ROTARY_HALF", "FA_ROTARY_INTERLEAVED"):
        assert got[n] == getattr(L, n)


def _rotary_params():
    p = L.FaRotaryParams()
    p.dtype, p.B, p.H, p.H_kv, p.T, p.D = L.FA_DTYPE_BF16, 1, 2, 1, 4, 64
    for t in ("q", "k", "q_out", "k_out"):
        setattr(p, t, L.FaTensor(4096, 512, 256, 64))  # never dereferenced: validation fails first
    p.rotary = L.FaRotarySpec(64, L.FA_ROTARY_HALF, 4096, 1.0)
    return p


@pytest.mark.parametrize("change,text", [
    (lambda p: setattr(p, "dtype", L.FA_DTYPE_E4M3), b"dtype"), (lambda p: setattr(p, "T", 0), b"shape"),
    (lambda p: (setattr(p, "H", 0), setattr(p, "H_kv", 0)), b"shape"), (lambda p: setattr(p, "H", -1), b"shape"),
    (lambda p: setattr(p.rotary, "rotary_dim", 66), b"rotary_dim"), (lambda p: setattr(p.rotary, "rotary_dim", 3), b"rotary_dim"),
    (lambda p: setattr(p.rotary, "rotary_dim", -2), b"rotary_dim"), (lambda p: setattr(p.rotary, "layout", 2), b"layout"),
    (lambda p: setattr(p.rotary, "turns", None), b"turns"), (lambda p: setattr(p.rotary, "turns", 4100), b"turns"),
    (lambda p: setattr(p.k_out, "ptr", None), b"NULL"), (lambda p: setattr(p, "H", 70000), b"heads"),
    (lambda p: (setattr(p, "B", 1 << 15), setattr(p, "T", 1 << 15)), b"2^31")])
def test_rotary_refusals(change, text):
    p = _rotary_params()
    change(p)
    assert L.lib().fa_rotary(C.byref(p), None) in (L.FA_ERR_INVALID, L.FA_ERR_UNSUPPORTED)
    assert text in L.lib().fa_last_error()
    assert L.lib().fa_rotary(None, None) == L.FA_ERR_INVALID


def _cache(dtype=L.FA_DTYPE_E4M3):
    c = L.FaPagedCache()
    c.dtype, c.num_pages, c.H_kv, c.page_size, c.D = dtype, 8, 2, 64, 128
    c.k = c.v = L.FaTensor(4096, 2 * 64 * 128, 64 * 128, 128)
    c.k_scale = c.v_scale = c.block_table = 4096
    c.table_cols, c.table_stride = 3, 3
    return c


CACHE_FAULTS = [
    (lambda c: setattr(c, "dtype", L.FA_DTYPE_F32), b"bf16 or e4m3"), (lambda c: setattr(c, "num_pages", 0), b"shape"),
    (lambda c: setattr(c, "table_cols", 0), b"shape"), (lambda c: setattr(c, "page_size", 24), b"page_size"),
    (lambda c: setattr(c, "page_size", 256), b"page_size"), (lambda c: setattr(c, "D", 96), b"head dim"),
    (lambda c: setattr(c, "table_cols", 1 << 26), b"positions"), (lambda c: setattr(c, "block_table", None), b"NULL"),
    (lambda c: setattr(c, "table_stride", -3), b"stride"), (lambda c: setattr(c.v, "stride_t", 64), b"strides"),
    (lambda c: setattr(c.k, "ptr", 4104), b"16 bytes"), (lambda c: setattr(c.k, "stride_h", 8200), b"16 bytes"),
    (lambda c: setattr(c, "v_scale", None), b"k_scale"), (lambda c: setattr(c.k, "ptr", None), b"NULL")]


@pytest.mark.parametrize("change,text", CACHE_FAULTS + [
    (lambda c: setattr(c, "H_kv", 3), b"multiple")])
def test_attention_refusals_of_caches(change, text):
    p = L.FaPagedAttnParams()
    p.B, p.H, p.Tq, p.cache = 2, 8, 1, _cache()
    change(p.cache)
    size = C.c_size_t(0)
    assert L.lib().fa_paged_attn_workspace_size(C.byref(p), C.byref(size)) in (L.FA_ERR_INVALID, L.FA_ERR_UNSUPPORTED)
    assert text in L.lib().fa_last_error()


@pytest.mark.parametrize("change,text", CACHE_FAULTS)
def test_append_refusals_of_caches(change, text):
    p = L.FaPagedAppendParams()
    p.dtype, p.B, p.T, p.cache = L.FA_DTYPE_BF16, 2, 1, _cache()
    p.k = p.v = L.FaTensor(4096, 512, 256, 128)
    p.kv_lens = 4096
    change(p.cache)
    assert L.lib().fa_paged_append(C.byref(p), None) in (L.FA_ERR_INVALID, L.FA_ERR_UNSUPPORTED)
    assert text in L.lib().fa_last_error()


def test_append_and_attention_refusals():
    lib, size = L.lib(), C.c_size_t(0)
    good = L.FaPagedAppendParams()
    good.dtype, good.B, good.T, good.H, good.cache = L.FA_DTYPE_BF16, 2, 1, 4, _cache()
    good.q = good.k = good.v = good.q_out = L.FaTensor(4096, 512, 256, 128)
    good.kv_lens = 4096
    for change, text in [(lambda p: setattr(p, "dtype", 7), b"dtype"), (lambda p: setattr(p, "T", 0), b"T"),
                         (lambda p: setattr(p, "kv_lens", None), b"NULL"), (lambda p: setattr(p.q_out, "ptr", None), b"NULL"),
                         (lambda p: setattr(p, "rotary", L.FaRotarySpec(24, 0, 4096, 1.0)), b"multiple of 16"),
                         (lambda p: setattr(p, "rotary", L.FaRotarySpec(256, 0, 4096, 1.0)), b"rotary_dim"),
                         (lambda p: (setattr(p, "T", 1 << 20), setattr(p, "B", 1 << 10)), b"too many")]:
        p = L.FaPagedAppendParams.from_buffer_copy(good)
        change(p)
        assert lib.fa_paged_append(C.byref(p), None) in (L.FA_ERR_INVALID, L.FA_ERR_UNSUPPORTED)
        assert text in lib.fa_last_error(), lib.fa_last_error()
    good = L.FaPagedAttnParams()
    good.B, good.H, good.Tq, good.cache = 2, 8, 1, _cache()
    assert lib.fa_paged_attn_workspace_size(C.byref(good), C.byref(size)) == 0 and size.value > 0
    for change, text in [(lambda p: setattr(p, "Tq", 0), b"shape"), (lambda p: setattr(p.mask, "flags", L.FA_MASK_DOCUMENT), b"masks"),
                         (lambda p: setattr(p.mask, "q_offset", 4), b"offsets"),
                         (lambda p: setattr(p.score, "flags", L.FA_SCORE_REL_BIAS), b"score"),
                         (lambda p: setattr(p.score, "flags", L.FA_SCORE_ALIBI), b"slopes"),
                         (lambda p: setattr(p.score, "flags", L.FA_SCORE_SOFTCAP), b"softcap"),
                         (lambda p: (setattr(p, "Tq", 1 << 24), setattr(p, "B", 1 << 12)), b"too many")]:
        p = L.FaPagedAttnParams.from_buffer_copy(good)
        change(p)
        assert lib.fa_paged_attn_workspace_size(C.byref(p), C.byref(size)) in (L.FA_ERR_INVALID, L.FA_ERR_UNSUPPORTED)
        assert text in lib.fa_last_error(), lib.fa_last_error()
    assert lib.fa_paged_attn(C.byref(good), None, 0, None) == L.FA_ERR_INVALID and b"NULL" in lib.fa_last_error()
    good.q = good.o = L.FaTensor(4096, 1024, 128, 128)
    good.lse = good.kv_lens = 4096
    assert lib.fa_paged_attn(C.byref(good), 4096, 16, None) == L.FA_ERR_INVALID and b"workspace" in lib.fa_last_error()


def test_workspace_does_not_grow_with_lengths():
    """At most two partial results per CTA, whatever the table's width."""
    size, p = C.c_size_t(0), L.FaPagedAttnParams()
    p.B, p.H, p.Tq, p.cache = 64, 8, 1, _cache()
    got = []
    for cols in (300, 3000, 300000):
        p.cache.table_cols = cols
        assert L.lib().fa_paged_attn_workspace_size(C.byref(p), C.byref(size)) == 0
        got.append(size.value)
    assert got[0] == got[1] == got[2] == 2 * 148 * 8 * 129 * 4 + 256


def test_rotary_spec_turns_are_exact():
    spec = pf.rotary_spec(128, base=500000.0)
    pi = Fraction("3.14159265358979323846264338327950288419716939937510582097494459")
    turns = spec.turns(torch.device("cpu"))
    for f, bits in zip(spec.frequencies, turns.tolist()):
        want = Fraction(f) / (2 * pi)
        assert abs(Fraction(bits % (1 << 64), 1 << 64) - want) <= Fraction(1, 1 << 65)
    # the phase of a far position, as the kernel forms it, against exact arithmetic
    pos = (1 << 31) - 5
    for f, bits in zip(spec.frequencies[::9], turns.tolist()[::9]):
        phase = Fraction(pos * bits % (1 << 64), 1 << 64)
        want = pos * Fraction(f) / (2 * pi) % 1
        d = abs(phase - want)
        assert min(d, 1 - d) <= Fraction(pos, 1 << 65)
    # frequencies above a turn per position, or negative, wrap
    odd = pf.rotary_spec(4, frequencies=[10.0, -0.25])
    t = odd.turns(torch.device("cpu")).tolist()
    assert abs(t[0] % (1 << 64) / 2 ** 64 - (10 / (2 * math.pi)) % 1) < 1e-12
    assert abs(t[1] % (1 << 64) / 2 ** 64 - (-0.25 / (2 * math.pi)) % 1) < 1e-12


def test_scalings():
    rd, base = 64, 10000.0
    plain = pf.rotary_spec(rd).frequencies
    lin = pf.rotary_spec(rd, scaling=pf.linear_scaling(4.0))
    assert all(math.isclose(a / 4, b) for a, b in zip(plain, lin.frequencies)) and lin.magnitude == 1.0
    ntk = pf.rotary_spec(rd, scaling=pf.ntk_scaling(4.0)).frequencies
    assert ntk[0] == 1.0 and math.isclose(ntk[-1], plain[-1] / 4)
    parts = pf.rotary_spec(rd, scaling=pf.by_parts_scaling(8.0, 4096))
    assert math.isclose(parts.magnitude, 0.1 * math.log(8) + 1)
    for f, g in zip(plain, parts.frequencies):
        turns = 4096 * f / (2 * math.pi)
        assert f / 8 * (1 - 1e-12) <= g <= f * (1 + 1e-12)
        if turns > 32 * base ** (2 / rd):
            assert g == f
        if turns < base ** (-2 / rd):
            assert math.isclose(g, f / 8)
    for bad in (lambda: pf.linear_scaling(0), lambda: pf.ntk_scaling(-1), lambda: pf.by_parts_scaling(2, 0),
                lambda: pf.by_parts_scaling(2, 10, 1, 1), lambda: pf.rotary_spec(64, rotary_dim=65),
                lambda: pf.rotary_spec(64, rotary_dim=66), lambda: pf.rotary_spec(64, rotary_dim=-2),
                lambda: pf.rotary_spec(64, base=1.0), lambda: pf.rotary_spec(64, frequencies=[1.0]),
                lambda: pf.rotary_spec(4, frequencies=[1.0, math.nan]),
                lambda: pf.rotary_spec(4, frequencies=[1.0, 1.0], scaling=pf.linear_scaling(2)),
                lambda: pf.rotary_spec(2, scaling=pf.ntk_scaling(2))):
        with pytest.raises(ValueError):
            bad()


def test_cpu_tensors_are_refused():
    x = torch.zeros(1, 1, 16, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        pf.rotary_embedding(x, None, pf.rotary_spec(64))
    with pytest.raises(ValueError):
        pf.PagedKVCache(x, x)


def test_reference_of_rotation_and_gradient():
    """The reference turns pairs by the angle (against complex arithmetic), and its inverse is its transpose."""
    g = torch.Generator().manual_seed(0)
    for inter in (False, True):
        spec = pf.rotary_spec(16, rotary_dim=8, interleaved=inter, scaling=pf.by_parts_scaling(4.0, 64))
        x, y = (torch.randn(2, 5, 16, generator=g, dtype=torch.float64) for _ in range(2))
        pos = torch.tensor([0, 1, 7, 100, 65536])
        rx, _ = rotate64(x, spec, pos)
        by, _ = rotate64(y, spec, pos, inverse=True)
        assert abs(float((rx * y).sum() - (x * by).sum())) < 1e-9
        i = 2
        a, b = (2 * i, 2 * i + 1) if inter else (i, i + 4)
        z = torch.complex(x[..., a], x[..., b]) * torch.polar(
            torch.full((5,), spec.magnitude, dtype=torch.float64), pos.double() * spec.frequencies[i])
        assert torch.allclose(z.real, rx[..., a], atol=1e-9) and torch.allclose(z.imag, rx[..., b], atol=1e-9)


def test_reference_of_e4m3():
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    codes = codes[torch.isfinite(codes)].double()
    assert torch.equal(to_e4m3_64(codes), codes)
    x = torch.cat((torch.linspace(-500, 500, 20001), torch.linspace(-0.05, 0.05, 20001))).double()
    want = x.clamp(-448, 448).float().to(torch.float8_e4m3fn).double()
    assert torch.equal(to_e4m3_64(x), want)
    assert float(e4m3_step(torch.tensor(1.0))) == 0.125 and float(e4m3_step(torch.tensor(1e-9))) == 2.0 ** -9
    for top, s in ((448.0, 1.0), (448.001, 2.0), (1.0, 2.0 ** -8), (0.0, 2.0 ** -100), (1e-35, 2.0 ** -100)):
        assert float(scale_for(torch.tensor(top, dtype=torch.float64))) == s
