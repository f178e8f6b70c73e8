"""64-bit references of rotary positions, paged appends and paged attention, and the error that the
kernels may make against them, derived from their roundings.

A rounding to a type is off by at most half a step: eps / 2 relative, with eps / 2 = 2^-8 for
bf16, 2^-24 for fp32 and 2^-4 for e4m3.
"""
import math

import torch

U_BF16, U_F32, U_E4M3 = 2.0 ** -8, 2.0 ** -24, 2.0 ** -4


def unit(dtype):
    return {torch.bfloat16: U_BF16, torch.float32: U_F32}[dtype]


# ------------------------------------------------------------------ rotary
def rotate64(x, spec, pos, inverse=False):
    """x (..., T, D) turned by pos (T,) in 64 bits, and the error bound of the kernel's result.

    The phase is exact; its conversion to fp32 is off by 2^-24 relative, at most 2^-24 pi in the
    angle.  fp32: sincospi is within 2 ulp (2^-22).  bf16: the angle's product with pi adds 2^-23 pi, and
    the hardware's sine and cosine are within 2^-21 on [-pi, pi].  The magnitude's product adds 2^-24.
    Two products and a sum round at most three times (3 * 2^-24 of m (|a| + |b|)), then the result is
    rounded once to x's type."""
    rd, m = spec.rotary_dim, spec.magnitude
    x64 = x.double()
    f = torch.tensor(spec.frequencies, dtype=torch.float64, device=x.device)
    ang = torch.remainder(pos.double()[:, None] * f, 2 * math.pi) * (-1 if inverse else 1)
    c, s = torch.cos(ang) * m, torch.sin(ang) * m
    if spec.interleaved:
        a, b = x64[..., 0:rd:2], x64[..., 1:rd:2]
    else:
        a, b = x64[..., : rd // 2], x64[..., rd // 2: rd]
    ra, rb = a * c - b * s, b * c + a * s
    turn = 2.0 ** -22 + (2.0 ** -22 if x.dtype == torch.float32 else 2.0 ** -21 + 2.0 ** -21) + 2.0 ** -24
    e = (a.abs() + b.abs()) * m * (turn + 3 * U_F32)
    # the reference's own angle: a 64-bit product of a position below 2^31 is off by 2^-53 * 2^31 = 2^-22
    if pos.numel():
        e = e + (a.abs() + b.abs()) * m * pos.double().abs().max().item() * 2.0 ** -52
    if spec.interleaved:
        out, err = torch.stack((ra, rb), -1).flatten(-2), torch.stack((e, e), -1).flatten(-2)
    else:
        out, err = torch.cat((ra, rb), -1), torch.cat((e, e), -1)
    out = torch.cat((out, x64[..., rd:]), -1)
    err = torch.cat((err, torch.zeros_like(x64[..., rd:])), -1)
    return out, err


def assert_within(name, got, ref, tol):
    got, ref = got.double(), ref.double()
    assert got.shape == ref.shape, (name, got.shape, ref.shape)
    fin = torch.isfinite(ref)
    assert torch.equal(torch.isnan(ref), torch.isnan(got)), f"{name}: NaN in other places"
    assert torch.equal(ref[~fin & ~ref.isnan()], got[~fin & ~ref.isnan()]), f"{name}: infinities differ"
    over = ((got - ref).abs() - tol)[fin]
    if over.numel():
        k = int(over.argmax())
        assert float(over.max()) <= 0, (f"{name}: {got[fin][k].item()} for {ref[fin][k].item()}, "
                                        f"{float(over.max()):.3e} beyond the bound")


# ------------------------------------------------------------------ e4m3 and appends
def e4m3_step(x):
    """Distance of neighbouring e4m3 values at |x| (three fraction bits, exponents from -6)."""
    return torch.exp2((torch.frexp(x.double())[1] - 1).clamp(min=-6).double() - 3)


def to_e4m3_64(x):
    s = e4m3_step(x)
    return (torch.round(x.double() / s) * s).clamp(-448.0, 448.0)


def scale_for(top):
    """The least power of two s (from 2^-100) with top <= 448 s, elementwise."""
    m, e = torch.frexp(top.double())
    e = torch.where(top > 0, e - 9 + (m > 0.875).to(e.dtype), torch.full_like(e, -100)).clamp(min=-100)
    return torch.exp2(e.double())


# ------------------------------------------------------------------ attention
def attend64(q, cache, table, lens, qlens, kind, window, slopes, cap, scale, hidden_page=lambda p: False):
    """o, lse of paged attention in 64 bits and their error bounds, by the formula, one sequence and
    K/V head at a time."""
    B, H, Tq, D = q.shape
    n_pages, hkv, ps, _ = cache.k.shape
    G = H // hkv
    f8 = cache.k_scale is not None
    o = torch.zeros(B, H, Tq, D, dtype=torch.float64, device=q.device)
    lse = torch.full((B, H, Tq), -math.inf, dtype=torch.float64, device=q.device)
    to, tl = torch.zeros_like(o), torch.zeros_like(lse)
    for b in range(B):
        n, t = min(lens[b], table.shape[1] * ps), qlens[b]
        if n == 0 or t == 0:
            continue
        ids = table[b, : -(-n // ps)].long()
        hide_page = torch.tensor([not 0 <= int(p) < n_pages or hidden_page(int(p)) for p in ids], device=q.device)
        ids = torch.where(hide_page, torch.zeros_like(ids), ids)
        gone = hide_page.repeat_interleave(ps)[:n]
        for hk in range(hkv):
            kc, vc = (c[ids, hk].double().flatten(0, 1)[:n] for c in (cache.k, cache.v))
            ks, vs = ((s[ids, hk].double().repeat_interleave(ps)[:n] if f8 else torch.ones(n, device=q.device).double())
                      for s in (cache.k_scale, cache.v_scale))
            qq = q[b, hk * G:(hk + 1) * G, :t].double()
            kk = kc * ks[:, None]
            pos = torch.arange(n, device=q.device)
            qpos = torch.arange(n - t, n, device=q.device)
            see = torch.ones(t, n, dtype=torch.bool, device=q.device)
            if kind in ("causal", "window"):
                see = pos[None] <= qpos[:, None]
            if kind == "window":
                see = see & (qpos[:, None] - pos[None] <= window)
            if kind == "band":  # a window to both sides
                see = (qpos[:, None] - pos[None] <= window[0]) & (pos[None] - qpos[:, None] <= window[1])
            see = see & ~gone[None]
            s = torch.einsum("gtd,nd->gtn", qq, kk) * scale
            # S: D exact products summed in fp32 (each addition off by 2^-23 of the terms' sum at most), an
            # 8-bit q split exact down to 2^-17 of its largest element, three fp32 products after it
            mag = torch.einsum("gtd,nd->gtn", qq.abs(), kk.abs()) * scale
            err = mag * (D + 16) * 2.0 ** -23 + s.abs() * 4 * U_F32
            if f8:
                err = err + 2.0 ** -17 * qq.abs().amax(-1, keepdim=True) * kk.abs().sum(-1) * scale
            if slopes is not None:
                al = slopes[hk * G:(hk + 1) * G].double()[:, None, None] * (pos[None] - qpos[:, None]).double()
                s = s + al
                err = err + al.abs() * 2 * U_F32
            if cap:
                s = cap * torch.tanh(s / cap)
                err = err + cap * 2.0 ** -21  # 1 - 2 / (1 + e^z): exponential, quotient and sum, 2^-23 each at most
            # into log2 units and back, the exponential itself, and the sum with log2 vs
            err = err + s.abs() * 2 * U_F32 + 2.0 ** -22 + vs.clamp(min=2.0 ** -100).log2().abs() * 2 * U_F32
            s = s.masked_fill(~see, -math.inf)
            top = s.amax(-1, keepdim=True)
            top = torch.where(top == -math.inf, torch.zeros_like(top), top)
            p = torch.exp(s - top)
            z = p.sum(-1)
            some = z > 0
            p = p / torch.where(some, z, torch.ones_like(z))[..., None]
            v = vc * vs[:, None]
            v0 = torch.where(see.any(0)[:, None], v, torch.zeros_like(v))  # what no row sees does not count
            dx = torch.where(see, err, torch.zeros_like(err)).amax(-1)
            oo = p @ v0
            pv = p @ v0.abs()
            # the probability's rounding (bf16, or two e4m3 parts: 2^-4 * 2^-4), the logits' error in
            # numerator and denominator, sums of n terms in fp32, and the output's rounding
            rel = U_BF16 + 2.1 * dx[..., None] + (n + 64) * 2.0 ** -23
            tol = pv * rel + oo.abs() * U_BF16
            if f8:
                # parts below e4m3's smallest step: 2^-10 of P, where the largest p vs is at least 2^5
                big = (p * vs).amax(-1, keepdim=True)
                tol = tol + 2.0 ** -15 * big * v0.div(vs.clamp(min=2.0 ** -100)[:, None]).abs().sum(0)
            sl = slice(hk * G, (hk + 1) * G)
            o[b, sl, :t] = oo
            lse[b, sl, :t] = torch.where(some, top[..., 0] + torch.log(z), torch.full_like(z, -math.inf))
            to[b, sl, :t] = tol + 1e-30
            tl[b, sl, :t] = 1.1 * dx + (n + 64) * 2.0 ** -23 + lse[b, sl, :t].abs().nan_to_num(0, 0, 0) * 4 * U_F32 + 2.0 ** -20
    return o, lse, to, tl
