"""The serving operators around a paged K/V cache, as cases to be timed and compared.

Three operators of one decode or prompt step:

* ``rotary``: the rotary position embedding of q and k, forward, and forward with its gradients;
* ``append``: new keys (rotated on the way) and values written into the pages of a cache, with the
  step's q rotated in the same call.  The cache is bf16, or 8-bit (e4m3) with one power-of-two
  scale for each page and head;
* ``attend``: attention of the step's query rows against that cache.

``own`` picks between the plain form (elementary torch operations) and the framework's calls.

Shapes follow the framework: q (B, H, T, D), k and v (B, H_kv, T, D), caches (pages, H_kv,
page_size, D), scales (pages, H_kv), a block table (B, pages of a sequence).  ``kv_lens`` counts
the cached positions of a sequence with its new tokens, ``new_lens`` the valid ones among its T
new tokens: token i < new_lens[b] sits at position kv_lens[b] - new_lens[b] + i.
"""
import math
import random
import sys

import torch

own = False

DEV = "cuda"
E4M3_MAX = 448.0
SCALE_FLOOR = -100  # smallest exponent of a page's scale: an all-zero page gets 2^-100
FAR = 1 << 20       # positions of a long context


# ------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one decode step of 64 users with far positions: a few KB each way, the launch counts
        {"name": "rotary_step_b64", "op": "rotary", "B": 64, "H": 32, "Hkv": 8, "T": 1, "D": 128, "rd": 128,
         "inter": False, "dtype": "bf16", "layout": "bhtd", "pos": "far", "scaling": "none", "grad": False},
        # a training step's q and k, forward and gradients, at the length of the window benchmark
        {"name": "rotary_train_s8192", "op": "rotary", "B": 2, "H": 32, "Hkv": 8, "T": 8192, "D": 128, "rd": 128,
         "inter": False, "dtype": "bf16", "layout": "bthd", "pos": "range", "scaling": "none", "grad": True},
        # part of the head, interleaved pairs, stretched for a long context, odd length, fp32
        {"name": "rotary_part_fp32_s4097", "op": "rotary", "B": 1, "H": 16, "Hkv": 16, "T": 4097, "D": 64, "rd": 32,
         "inter": True, "dtype": "fp32", "layout": "bhtd", "pos": "packed", "scaling": "parts", "grad": True},
        # one decode step of 64 users into an 8-bit cache: the page's scale may have to grow
        {"name": "append_step_b64_e4m3", "op": "append", "B": 64, "H": 32, "Hkv": 8, "T": 1, "D": 128, "rd": 128,
         "inter": False, "cache": "e4m3", "ps": 64, "ctx": 500, "mix": 1},
        # prompts of eight users, up to 2048 tokens each behind what they have cached
        {"name": "append_prompt_b8_e4m3", "op": "append", "B": 8, "H": 32, "Hkv": 8, "T": 2048, "D": 128, "rd": 128,
         "inter": False, "cache": "e4m3", "ps": 64, "ctx": 300, "mix": 2},
        # an odd prompt into a bf16 cache of small pages, interleaved pairs in half of the head
        {"name": "append_prompt_odd_bf16", "op": "append", "B": 3, "H": 16, "Hkv": 16, "T": 1111, "D": 64, "rd": 32,
         "inter": True, "cache": "bf16", "ps": 16, "ctx": 77, "mix": 3},
        # one user with a short context: the latency of one token
        {"name": "attend_one_l1000", "op": "attend", "B": 1, "H": 32, "Hkv": 8, "Tq": 1, "L": 1000, "D": 128,
         "cache": "e4m3", "ps": 64, "mask": "causal", "window": 0, "score": "none", "mix": 4},
        # the decode benchmark's batch of 64 with lengths up to 4096, in 8 bits
        {"name": "attend_b64_l4096", "op": "attend", "B": 64, "H": 32, "Hkv": 8, "Tq": 1, "L": 4096, "D": 128,
         "cache": "e4m3", "ps": 64, "mask": "causal", "window": 0, "score": "none", "mix": 5},
        # a few users with long contexts (the length of the sparse benchmark), large pages
        {"name": "attend_b8_l32768", "op": "attend", "B": 8, "H": 32, "Hkv": 8, "Tq": 1, "L": 32768, "D": 128,
         "cache": "e4m3", "ps": 128, "mask": "causal", "window": 0, "score": "none", "mix": 6},
        # the decode benchmark's head dim 64 without grouping, a bf16 cache in small pages, ALiBi in a window
        {"name": "attend_window_d64_bf16", "op": "attend", "B": 32, "H": 16, "Hkv": 16, "Tq": 1, "L": 8192, "D": 64,
         "cache": "bf16", "ps": 16, "mask": "window", "window": 1024, "score": "alibi", "mix": 7},
        # five drafted tokens to check at once, head dim 256, softcap, odd lengths
        {"name": "attend_draft_d256", "op": "attend", "B": 5, "H": 16, "Hkv": 2, "Tq": 5, "L": 2777, "D": 256,
         "cache": "e4m3", "ps": 32, "mask": "causal", "window": 0, "score": "softcap", "mix": 8},
        # a chunk of the prompts of four users behind what they have cached
        {"name": "attend_prompt_chunk", "op": "attend", "B": 4, "H": 32, "Hkv": 8, "Tq": 512, "L": 4096, "D": 128,
         "cache": "e4m3", "ps": 64, "mask": "causal", "window": 0, "score": "none", "mix": 9},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["rotary", "append", "attend", "attend"])
    D = rng.choice([64, 128, 128, 256])
    Hkv, G = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 2, 3, 4, 7, 8])
    if op == "rotary":
        B, T = _log(rng, 1, 64), _log(rng, 1, 8192)
        while B * T * (G + 1) * Hkv * D > 2 * 8192 * 40 * 128:
            B, T = max(1, B // 2), max(1, T * 2 // 3)
        return {"op": op, "B": B, "H": G * Hkv, "Hkv": Hkv, "T": T, "D": D, "rd": rng.choice([D, D, D // 2, D // 4]),
                "inter": rng.random() < 0.5, "dtype": rng.choice(["bf16", "bf16", "fp32"]),
                "layout": rng.choice(["bhtd", "bthd"]), "pos": rng.choice(["far", "range", "packed"]),
                "scaling": rng.choice(["none", "linear", "ntk", "parts"]), "grad": rng.random() < 0.5}
    cache, ps = rng.choice(["e4m3", "e4m3", "bf16"]), rng.choice([16, 32, 64, 128])
    if op == "append":
        B, T, ctx = _log(rng, 1, 64), _log(rng, 1, 2048), _log(rng, 1, 600)
        while B * (T + 2 * ctx) * (G + 4) * Hkv * D > 8 * 2048 * 48 * 128:
            B, T = max(1, B // 2), max(1, T * 2 // 3)
        return {"op": op, "B": B, "H": G * Hkv, "Hkv": Hkv, "T": T, "D": D, "rd": rng.choice([D, D, D // 2]),
                "inter": rng.random() < 0.5, "cache": cache, "ps": ps, "ctx": ctx, "mix": rng.randrange(1 << 20)}
    B, L = _log(rng, 1, 64), _log(rng, 1, 32768)
    Tq = rng.choice([1, 1, 1, 1, 2, 3, 5, 17, 130])
    while B * L * Hkv * D > 64 * 4096 * 8 * 128 or B * L * Hkv * G * Tq * max(D, 128) > 4 * 4096 * 32 * 512 * 128:
        B, L = max(1, B // 2), max(1, L * 2 // 3)
    mask = rng.choice(["none" if Tq == 1 else "causal", "causal", "window"])
    return {"op": op, "B": B, "H": G * Hkv, "Hkv": Hkv, "Tq": Tq, "L": L, "D": D, "cache": cache, "ps": ps,
            "mask": mask, "window": _log(rng, 16, 4096) if mask == "window" else 0,
            "score": rng.choice(["none", "none", "softcap", "alibi"]), "mix": rng.randrange(1 << 20)}


def _lens(case):
    """Cached lengths and new tokens of each sequence: a function of the case alone."""
    r, B = random.Random(case["mix"]), case["B"]
    if case["op"] == "append":
        T = case["T"]
        new = [T if b == 0 else r.randint(max(1, T // 3), T) for b in range(B)]
        return [n + r.randint(0, 2 * case["ctx"]) for n in new], new
    L, Tq = case["L"], case["Tq"]
    lens = [L if b == 0 else r.randint(max(1, L // 2), L) for b in range(B)]
    return lens, [min(n, Tq if b == 0 or Tq < 16 else r.randint(Tq // 2, Tq)) for b, n in enumerate(lens)]


def _pairs(case):
    """Visible (query row, key) pairs of one head, and cached positions that some row sees."""
    pairs = keys = 0
    for n, t in zip(*_lens(case)):
        first = n
        for p in range(n - t, n):
            lo = max(0, p - case["window"]) if case["mask"] == "window" else 0
            hi = n - 1 if case["mask"] == "none" else p
            pairs += hi - lo + 1
            first = min(first, lo)
        keys += n - first
    return pairs, keys


def work(case):
    D, H, Hkv, op = case["D"], case["H"], case["Hkv"], case["op"]
    if op == "rotary":
        n = case["B"] * case["T"] * (H + Hkv)
        es, passes = (4 if case["dtype"] == "fp32" else 2), (2 if case["grad"] else 1)
        return {"bytes": passes * 2 * n * D * es, "flops": passes * 3 * n * case["rd"]}
    es = 1 if case["cache"] == "e4m3" else 2
    if op == "append":
        new = sum(_lens(case)[1])
        scales = 0 if es == 2 else 8 * Hkv * sum(-(-n // case["ps"]) for n in _lens(case)[1])
        return {"bytes": new * D * (2 * 2 * H + 2 * Hkv * (2 + es)) + scales, "flops": 3 * new * (H + Hkv) * case["rd"]}
    pairs, keys = _pairs(case)
    rows = sum(_lens(case)[1]) * H
    scales = 0 if es == 2 else 8 * Hkv * -(-keys // case["ps"])
    return {"bytes": 2 * keys * Hkv * D * es + scales + rows * (4 * D + 4), "flops": 4 * D * H * pairs}


# ------------------------------------------------------------------------------------- the inputs
def _scaling(case):
    """What the rotary frequencies are stretched by."""
    return {"none": None, "linear": ("linear", 4.0), "ntk": ("ntk", 4.0),
            "parts": ("parts", 8.0, 4096)}[case.get("scaling", "none")]


def _frequencies(case):
    """Radians a position for each pair, in 64 bits, and the factor on the rotated values."""
    rd, base, s = case["rd"], 10000.0, _scaling(case)
    i = torch.arange(rd // 2, dtype=torch.float64)
    if s and s[0] == "ntk":  # the base grows so that the slowest pair turns as under linear scaling
        base *= s[1] ** (rd / (rd - 2))
    f = base ** (-2.0 * i / rd)
    if s and s[0] == "linear":
        f = f / s[1]
    if s and s[0] == "parts":
        # pairs that turn over 32 times within the original length stay, those under once are divided
        # by the factor, and a ramp joins the two
        factor, length = s[1], s[2]
        lo, hi = (rd * math.log(length / (t * 2 * math.pi)) / (2 * math.log(base)) for t in (32.0, 1.0))
        lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), rd - 1)
        ramp = ((i - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        return f * (1 - ramp) + f / factor * ramp, 0.1 * math.log(factor) + 1.0
    return f, 1.0


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEV)


def _activations(g, dtype, layout, *shape):
    """(B, H, T, D) activations as a projection leaves them: some channels larger than others."""
    B, H, T, D = shape
    amp = torch.exp(0.5 * _randn(g, D))
    x = _randn(g, B, T, H, D) if layout == "bthd" else _randn(g, B, H, T, D)
    x = (x * amp).to(dtype)
    return x.transpose(1, 2) if layout == "bthd" else x


def _pages(case, g, cols):
    """A pool of pages and a block table that deals them out in random order."""
    B, ps = case["B"], case["ps"]
    n = B * cols + 3
    table = torch.randperm(n, generator=g, device=DEV)[: B * cols].view(B, cols).to(torch.int32)
    shape = (n, case["Hkv"], ps, case["D"])
    pools = []
    for _ in range(2):
        if case["cache"] == "bf16":
            pools.append((torch.randn(shape, generator=g, device=DEV, dtype=torch.bfloat16), None))
        else:
            # e4m3 values, and a power-of-two scale for each page and head as an append leaves them
            codes = (torch.randn(shape, generator=g, device=DEV, dtype=torch.bfloat16) * 96).clamp_(-448, 448)
            e = torch.randint(-9, -5, shape[:2], generator=g, device=DEV)
            pools.append((codes.to(torch.float8_e4m3fn), torch.exp2(e.float())))
    (k, ks), (v, vs) = pools
    return k, v, ks, vs, table


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    op, B, H, Hkv, D = case["op"], case["B"], case["H"], case["Hkv"], case["D"]
    st = {"case": dict(case)}
    if op != "attend":
        st["freq"], st["factor"] = _frequencies(case)
        st["freq"] = st["freq"].to(DEV)
    if op == "rotary":
        T, dtype = case["T"], torch.float32 if case["dtype"] == "fp32" else torch.bfloat16
        st["q"] = _activations(g, dtype, case["layout"], B, H, T, D)
        st["k"] = _activations(g, dtype, case["layout"], B, Hkv, T, D)
        if case["pos"] == "far":     # each sequence at a place of its own in a long context
            st["pos"] = torch.randint(0, FAR, (B, 1), generator=g, device=DEV) + torch.arange(T, device=DEV)
        elif case["pos"] == "packed":  # documents behind one another, each from position 0
            cut = torch.randint(64, 2048, (1,), generator=g, device=DEV)
            st["pos"] = torch.arange(T, device=DEV) % cut
        else:
            st["pos"] = torch.arange(T, device=DEV)
        st["pos"] = st["pos"].to(torch.int32)
        if case["grad"]:
            st["dq"] = _activations(g, dtype, "bhtd", B, H, T, D)
            st["dk"] = _activations(g, dtype, "bhtd", B, Hkv, T, D)
            st["q"].requires_grad_(True)
            st["k"].requires_grad_(True)
    else:
        lens, new = _lens(case)
        st["k_cache"], st["v_cache"], st["k_scale"], st["v_scale"], st["table"] = _pages(
            case, g, -(-max(lens) // case["ps"]))
        st["kv_lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
        st["new_lens"] = torch.tensor(new, dtype=torch.int32, device=DEV)
        T = case["T"] if op == "append" else case["Tq"]
        st["q"] = _activations(g, torch.bfloat16, "bthd", B, H, T, D) if op == "append" else _randn(
            g, B, H, T, D).to(torch.bfloat16)
        if op == "append":
            st["k"] = _activations(g, torch.bfloat16, "bthd", B, Hkv, T, D)
            st["v"] = _activations(g, torch.bfloat16, "bthd", B, Hkv, T, D)
        elif case["score"] == "alibi":
            st["slopes"] = torch.exp2(-8.0 * torch.arange(1, H + 1, device=DEV) / H)
    if own:
        _prepare_own(st)
    return st


def _prepare_own(st):
    """The handles that a user's program keeps: the rotary description, the cache, the mods."""
    if "pallas-flexattn_b200" not in sys.path:
        sys.path.insert(0, "pallas-flexattn_b200")
    import pallas_flexattn as pf

    case = st["case"]
    st["pf"] = pf
    if case["op"] != "attend":
        s = _scaling(case)
        kind = {"linear": pf.linear_scaling, "ntk": pf.ntk_scaling, "parts": pf.by_parts_scaling}
        st["rotary"] = pf.rotary_spec(case["D"], rotary_dim=case["rd"], base=10000.0, interleaved=case["inter"],
                                      scaling=kind[s[0]](*s[1:]) if s else None)
    if case["op"] != "rotary":
        st["cache"] = pf.PagedKVCache(st["k_cache"], st["v_cache"], st["k_scale"], st["v_scale"])
    if case["op"] == "attend":
        st["mask_mod"] = {"none": None, "causal": pf.causal_mask,
                          "window": pf.sliding_window_mask(case["window"], 0)}[case["mask"]]
        st["score_mod"] = (pf.softcap_score_mod(20.0) if case["score"] == "softcap" else
                           pf.alibi_score_mod(case["H"]) if case["score"] == "alibi" else None)


# -------------------------------------------------------------------------- one pass through each
def run(st):
    return {"rotary": _run_rotary, "append": _run_append, "attend": _run_attend}[st["case"]["op"]](st)


def _run_rotary(st):
    grad = st["case"]["grad"]
    if own:
        q, k = st["pf"].rotary_embedding(st["q"], st["k"], st["rotary"], st["pos"])
        return (q, k, *torch.autograd.grad((q, k), (st["q"], st["k"]), (st["dq"], st["dk"]))) if grad else (q, k)
    turn = _turn(st, st["pos"])
    with torch.no_grad():
        out = [_rotate(st["q"], st, turn), _rotate(st["k"], st, turn)]
        if grad:  # the transpose of a rotation turns back
            out += [_rotate(st["dq"], st, turn, back=True), _rotate(st["dk"], st, turn, back=True)]
    return tuple(out)


def _run_append(st):
    if own:
        q = st["pf"].paged_kv_append(st["cache"], st["table"], st["kv_lens"], st["k"], st["v"],
                                     new_lens=st["new_lens"], rotary=st["rotary"], q=st["q"])
    else:
        q = _plain_append(st)
    return (q, st["k_cache"], st["v_cache"]) + ((st["k_scale"], st["v_scale"]) if st["k_scale"] is not None else ())


def _run_attend(st):
    if own:
        return st["pf"].flash_attention_paged(st["q"], st["cache"], st["table"], st["kv_lens"], st["mask_mod"],
                                              q_lens=st["new_lens"], score_mod=st["score_mod"])
    return _plain_attend(st)


# ------------------------------------------------------------------------------- the plain forms
def _turn(st, pos):
    """cos and sin at each position, (..., T, rd / 2): the angles in 64 bits, far positions lose in 32."""
    a = pos.double()[..., None] * st["freq"]
    a = a - 2 * math.pi * torch.round(a / (2 * math.pi))
    return (torch.cos(a) * st["factor"]).float(), (torch.sin(a) * st["factor"]).float()


def _rotate32(x, st, turn, back=False):
    rd, inter = st["case"]["rd"], st["case"]["inter"]
    cos, sin = (t[:, None] if t.dim() == 3 else t for t in turn)  # (B, 1, T, rd / 2) or (T, rd / 2)
    if back:
        sin = -sin
    x = x.float()
    a, b = (x[..., 0:rd:2], x[..., 1:rd:2]) if inter else (x[..., : rd // 2], x[..., rd // 2: rd])
    ra, rb = a * cos - b * sin, b * cos + a * sin
    r = torch.stack((ra, rb), -1).flatten(-2) if inter else torch.cat((ra, rb), -1)
    return torch.cat((r, x[..., rd:]), -1)


def _rotate(x, st, turn, back=False):
    return _rotate32(x, st, turn, back).to(x.dtype)


def _plain_append(st):
    case = st["case"]
    ps, (B, _, T, D), Hkv = case["ps"], st["k"].shape, case["Hkv"]
    start = (st["kv_lens"] - st["new_lens"]).long()
    pos = start[:, None] + torch.arange(T, device=DEV)
    turn = _turn(st, pos)
    valid = torch.arange(T, device=DEV) < st["new_lens"][:, None]
    q = torch.where(valid[:, None, :, None], _rotate32(st["q"], st, turn), 0.0).to(st["q"].dtype)
    knew, vnew = _rotate32(st["k"], st, turn), st["v"].float()
    if case["cache"] == "bf16":
        b, t = valid.nonzero(as_tuple=True)
        page, at = st["table"][b, pos[b, t] // ps].long(), pos[b, t] % ps
        st["k_cache"][page, :, at] = knew[b, :, t].to(torch.bfloat16)
        st["v_cache"][page, :, at] = vnew[b, :, t].to(torch.bfloat16)
        return q
    # the pages that each sequence's new tokens touch, as (sequence, page) pairs
    first = start // ps
    cols = first[:, None] + torch.arange(T // ps + 2, device=DEV)
    touched = cols * ps < st["kv_lens"].long()[:, None]
    b, c = touched.nonzero(as_tuple=True)
    page, col = st["table"][b, cols[b, c]].long(), cols[b, c]
    row = col[:, None] * ps + torch.arange(ps, device=DEV)           # positions of the page's rows
    t = row - start[b][:, None]
    new = (t >= 0) & (t < st["new_lens"].long()[b][:, None])         # rows that a new token takes
    old = t < 0                                                      # rows cached before
    some = old.any(1)
    t = t.clamp(0, T - 1)
    for_scale = new[:, None, :, None]
    for x, cache, scale in ((knew, st["k_cache"], st["k_scale"]), (vnew, st["v_cache"], st["v_scale"])):
        rows = x[b[:, None], :, t].transpose(1, 2)                    # (pairs, H_kv, ps, D)
        top = torch.where(for_scale & torch.isfinite(rows), rows.abs(), 0.0).amax((2, 3))
        m, e = torch.frexp(top)                                       # the least e with top <= 448 * 2^e
        e = torch.where(top > 0, (e - 9 + (m > 0.875)).clamp(min=SCALE_FLOOR), SCALE_FLOOR)
        s = torch.exp2(e.float())
        was = scale[page]
        s = torch.where(some[:, None], torch.maximum(s, was), s)      # a page's scale only grows
        codes = cache[page]
        again = (codes.float() * (was / s)[..., None, None]).to(torch.float8_e4m3fn)
        fresh = (rows / s[..., None, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
        codes = torch.where(for_scale, fresh.float(), torch.where(old[:, None, :, None], again.float(), codes.float()))
        cache[page] = codes.to(torch.float8_e4m3fn)
        scale[page] = s
    return q


def _plain_attend(st):
    case = st["case"]
    B, H, Tq, D = st["q"].shape
    Hkv, ps, cols = case["Hkv"], case["ps"], st["table"].shape[1]
    page = st["table"].long()

    def whole(cache, scale):  # (B, H_kv, cached positions, D)
        x = cache[page].float()
        if scale is not None:
            x = x * scale[page][..., None, None]
        return x.transpose(1, 2).reshape(B, Hkv, cols * ps, D)

    k, v = whole(st["k_cache"], st["k_scale"]), whole(st["v_cache"], st["v_scale"])
    q = st["q"].float().reshape(B, Hkv, H // Hkv * Tq, D)
    x = (q @ k.transpose(-1, -2)).view(B, H, Tq, cols * ps) * (1 / math.sqrt(D))
    i = torch.arange(Tq, device=DEV)
    qpos = ((st["kv_lens"] - st["new_lens"])[:, None] + i)[:, None, :, None]   # (B, 1, Tq, 1)
    kpos = torch.arange(cols * ps, device=DEV)
    if case["score"] == "alibi":
        x += st["slopes"][:, None, None] * (kpos - qpos)
    elif case["score"] == "softcap":
        x = 20.0 * torch.tanh(x / 20.0)
    see = (kpos < st["kv_lens"][:, None, None, None]) & (i < st["new_lens"][:, None])[:, None, :, None]
    if case["mask"] != "none":
        d = qpos - kpos
        see = see & (d >= 0)
        if case["mask"] == "window":
            see = see & (d <= case["window"])
    x = torch.where(see, x, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = (p.view(B, Hkv, -1, cols * ps) @ v).view(B, H, Tq, D) / torch.where(total > 0, total, 1.0)
    return o.to(st["q"].dtype), (top + torch.log(total))[..., 0]


# ------------------------------------------------------------------ the definitions, in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    return {"rotary": _exact_rotary, "append": _exact_append, "attend": _exact_attend}[case["op"]](case, st)


def _exact_turn(x, pos, case, st, sign=1.0):
    """x (H, T, D) as complex pairs times e^(i angle), in 64 bits."""
    rd, x = case["rd"], x.detach().double()
    head = x[..., :rd].unflatten(-1, (-1, 2) if case["inter"] else (2, -1))
    z = torch.view_as_complex((head if case["inter"] else head.transpose(-1, -2)).contiguous())
    angle = torch.remainder(pos.double()[:, None] * st["freq"], 2 * math.pi) * sign
    z = torch.view_as_real(z * torch.polar(torch.full_like(angle, st["factor"]), angle))
    z = z if case["inter"] else z.transpose(-1, -2)
    return torch.cat((z.flatten(-2), x[..., rd:]), -1)


def _exact_rotary(case, st):
    out = []
    for name, sign in (("q", 1.0), ("k", 1.0)) + ((("dq", -1.0), ("dk", -1.0)) if case["grad"] else ()):
        pos = st["pos"].expand(case["B"], -1)
        out.append(torch.stack([_exact_turn(x, p, case, st, sign) for x, p in zip(st[name], pos)]))
    return tuple(out)


def _to_e4m3(x):
    """The nearest e4m3 values of x in 64 bits: three fraction bits, exponents from -6, ties to even."""
    step = torch.exp2((torch.frexp(x)[1] - 1).clamp(min=-6).double() - 3)
    return (torch.round(x / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def _exact_append(case, st):
    q = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
    k_cache, v_cache = st["k_cache"].double(), st["v_cache"].double()
    scales = [s.double() for s in (st["k_scale"], st["v_scale"]) if s is not None]
    ps = case["ps"]
    for b, (n, t) in enumerate(zip(*_lens(case))):
        pos = torch.arange(n - t, n, device=DEV)
        q[b, :, :t] = _exact_turn(st["q"][b, :, :t], pos, case, st)
        news = (_exact_turn(st["k"][b, :, :t], pos, case, st), st["v"][b, :, :t].double())
        for c in range((n - t) // ps, -(-n // ps)):
            page, lo, hi = int(st["table"][b, c]), max(c * ps, n - t), min(n, c * ps + ps)
            for j, (cache, new) in enumerate(zip((k_cache, v_cache), news)):
                rows = new[:, lo - (n - t): hi - (n - t)]
                if not scales:
                    cache[page, :, lo - c * ps: hi - c * ps] = rows
                    continue
                top = rows.abs().amax((1, 2))
                e = torch.ceil(torch.log2(top / E4M3_MAX))   # the logarithm of a power of two may be just off
                e = torch.where(top <= E4M3_MAX * torch.exp2(e - 1), e - 1, e)
                s = torch.exp2(e.clamp(min=SCALE_FLOOR))
                if lo > c * ps:
                    s = torch.maximum(s, scales[j][page])
                    earlier = cache[page, :, : lo - c * ps] * (scales[j][page] / s)[:, None, None]
                    cache[page, :, : lo - c * ps] = _to_e4m3(earlier)
                cache[page, :, lo - c * ps: hi - c * ps] = _to_e4m3(rows / s[:, None, None])
                scales[j][page] = s
    return (q, k_cache, v_cache, *scales)


def _exact_attend(case, st):
    B, H, Tq, D = st["q"].shape
    Hkv, G = case["Hkv"], H // case["Hkv"]
    o = torch.zeros(B, H, Tq, D, dtype=torch.float64, device=DEV)
    lse = torch.full((B, H, Tq), -math.inf, dtype=torch.float64, device=DEV)
    for b, (n, t) in enumerate(zip(*_lens(case))):
        pages = st["table"][b, : -(-n // case["ps"])].long()
        kv = []
        for cache, scale in ((st["k_cache"], st["k_scale"]), (st["v_cache"], st["v_scale"])):
            x = cache[pages].double()
            x = x if scale is None else x * scale[pages].double()[:, :, None, None]
            kv.append(x.transpose(0, 1).flatten(1, 2)[:, :n])
        for h in range(Hkv):
            q = st["q"][b, h * G: h * G + G, :t].double()
            s = torch.einsum("gtd,nd->gtn", q, kv[0][h]) / math.sqrt(D)
            back = (torch.arange(n - t, n, device=DEV)[:, None] - torch.arange(n, device=DEV)).double()
            if case["score"] == "alibi":
                s = s - st["slopes"][h * G: h * G + G].double()[:, None, None] * back
            elif case["score"] == "softcap":
                s = torch.tanh(s / 20.0) * 20.0
            hide = torch.zeros_like(back, dtype=torch.bool)
            if case["mask"] != "none":
                hide = back < 0
                if case["mask"] == "window":
                    hide = hide | (back > case["window"])
            s = s.masked_fill(hide, -math.inf)
            l = torch.logsumexp(s, -1)
            lse[b, h * G: h * G + G, :t] = l
            o[b, h * G: h * G + G, :t] = torch.exp(s - l[..., None]) @ kv[1][h]
    return o, lse
