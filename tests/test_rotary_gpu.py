"""Rotary positions on the GPU (rotary_embedding -> fa_rotary) against the formula in 64 bits, with the
bound that the kernel's roundings allow (paged_reference.rotate64), and their gradients."""
import math

import pytest
import torch

import pallas_flexattn as pf
from paged_reference import assert_within, rotate64, unit

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0) if torch.cuda.is_available() else None
BF16, F32 = torch.bfloat16, torch.float32

# B, H, Hkv, T, D, rotary_dim, interleaved, dtype, positions
CASES = {
    "one_token": (1, 4, 1, 1, 128, 128, False, BF16, "far"),
    "step_b7": (7, 3, 3, 1, 64, 64, True, BF16, "far"),
    "odd_t_half": (2, 5, 1, 257, 128, 128, False, BF16, None),
    "part_inter_fp32": (1, 2, 2, 65, 64, 32, True, F32, "packed"),
    "part_half_fp32_d256": (2, 2, 1, 33, 256, 64, False, F32, "batch"),
    "d96": (1, 3, 1, 19, 96, 96, False, BF16, 1000),
    "rd_not_16": (2, 3, 1, 9, 64, 24, False, BF16, "batch"),
    "rd_2": (1, 1, 1, 5, 8, 2, True, F32, None),
    "odd_d": (1, 2, 1, 5, 7, 6, False, F32, "far"),
    "rd_0_copies": (1, 2, 1, 5, 64, 0, False, BF16, None),
    "many_heads": (3, 40, 8, 31, 128, 128, True, BF16, "negative"),
    "q_only": (2, 6, 0, 12, 64, 64, False, BF16, None),
}


def _positions(kind, B, T, g):
    if kind == "far":
        return (torch.randint(0, 1 << 30, (B, 1), generator=g) + torch.arange(T)).int()
    if kind == "batch":
        return torch.randint(0, 5000, (B, T), generator=g).int()
    if kind == "packed":
        return torch.arange(T) % 13
    if kind == "negative":
        return torch.randint(-3000, 3000, (T,), generator=g)
    return kind


def _case(name):
    B, H, Hkv, T, D, rd, inter, dtype, kind = CASES[name]
    g = torch.Generator().manual_seed(sum(map(ord, name)))
    q = torch.randn(B, H, T, D, generator=g).to(DEV, dtype)
    k = torch.randn(B, Hkv, T, D, generator=g).to(DEV, dtype) if Hkv else None
    pos = _positions(kind, B, T, g)
    pos = pos.to(DEV) if isinstance(pos, torch.Tensor) else pos
    full = pos if isinstance(pos, torch.Tensor) else torch.arange(T, device=DEV) + (pos or 0)
    return q, k, pf.rotary_spec(D, rotary_dim=rd, interleaved=inter), pos, full.expand(B, T)


def _ref(x, spec, pos, inverse=False):
    out = [rotate64(x[b], spec, pos[b], inverse) for b in range(x.shape[0])]
    ref, err = torch.stack([o for o, _ in out]), torch.stack([e for _, e in out])
    return ref, err + unit(x.dtype) * ref.abs() + 1e-37


@pytest.mark.parametrize("name", list(CASES))
def test_rotation_matches_the_formula(name):
    q, k, spec, pos, full = _case(name)
    before = q.clone()
    rq, rk = pf.rotary_embedding(q, k, spec, pos)
    assert_within("q", rq, *_ref(q, spec, full))
    assert rq.dtype == q.dtype and torch.equal(q, before)
    if k is None:
        assert rk is None
    else:
        assert_within("k", rk, *_ref(k, spec, full))


@pytest.mark.parametrize("name", [n for n in CASES if n != "q_only"])
def test_gradient_is_the_rotation_back(name):
    q, k, spec, pos, full = _case(name)
    q.requires_grad_(True), k.requires_grad_(True)
    rq, rk = pf.rotary_embedding(q, k, spec, pos)
    dq, dk = torch.randn_like(rq), torch.randn_like(rk)
    gq, gk = torch.autograd.grad((rq, rk), (q, k), (dq, dk))
    assert_within("dq", gq, *_ref(dq, spec, full, inverse=True))
    assert_within("dk", gk, *_ref(dk, spec, full, inverse=True))


@pytest.mark.parametrize("inter", [False, True])
def test_gradient_against_differences(inter):
    # linear in x: (f(x + h) - f(x - h)) / 2h is exact but for fp32's rounding of values up to |x| + h,
    # each difference off by at most 4 * 2^-24 * max|y| / h
    spec = pf.rotary_spec(16, rotary_dim=8, interleaved=inter, scaling=pf.by_parts_scaling(4.0, 64))
    g = torch.Generator().manual_seed(3)
    x = torch.randn(1, 2, 3, 16, generator=g).to(DEV).requires_grad_(True)
    w = torch.randn(1, 2, 3, 16, generator=g).to(DEV)
    y, _ = pf.rotary_embedding(x, None, spec, 5)
    grad, = torch.autograd.grad((y * w).sum(), x)
    h = 0.25
    for j in range(0, 96, 7):
        e = torch.zeros(96, device=DEV)
        e[j] = h
        e = e.view_as(x)
        with torch.no_grad():
            up, dn = (pf.rotary_embedding(x + s * e, None, spec, 5)[0].double() for s in (1, -1))
        num = ((up - dn) * w.double()).sum().item() / (2 * h)
        tol = 96 * 8 * 2.0 ** -24 * float(up.abs().max() + 1) * float(w.abs().max()) / h
        assert abs(num - grad.flatten()[j].item()) <= tol


def test_second_gradient_and_unused_outputs():
    spec = pf.rotary_spec(64)
    q = torch.randn(1, 2, 4, 64, device=DEV, requires_grad=True)
    k = torch.randn(1, 1, 4, 64, device=DEV, requires_grad=True)
    rq, rk = pf.rotary_embedding(q, k, spec)
    gq, gk = torch.autograd.grad((rq * rq).sum(), (q, k), create_graph=True, allow_unused=True)
    assert gk is None  # k's output was not used: nothing was launched for it
    v = torch.randn_like(q)
    hv, = torch.autograd.grad((gq * v).sum(), q)
    # |rq|^2 has the gradient 2 q and the Hessian 2: rotations there and back, 5 roundings each of
    # values up to 2 |pair|
    assert_within("hv", hv, 2 * v.double(), torch.full_like(v, 64 * 2.0 ** -22 * float(v.abs().max())).double())


def test_positions_changed_before_the_gradient_are_an_error():
    spec = pf.rotary_spec(64)
    q = torch.randn(1, 2, 4, 64, device=DEV, requires_grad=True)
    pos = torch.arange(4, device=DEV, dtype=torch.int32)
    r, _ = pf.rotary_embedding(q, None, spec, pos)
    pos += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        r.sum().backward()


def test_expanded_gradient():
    spec = pf.rotary_spec(64, interleaved=True)
    q = torch.randn(1, 2, 4, 64, device=DEV, requires_grad=True)
    r, _ = pf.rotary_embedding(q, None, spec, 9)
    r.sum().backward()
    full = (torch.arange(4, device=DEV) + 9).expand(1, -1)
    assert_within("dq", q.grad, *_ref(torch.ones_like(q), spec, full, inverse=True))


def test_strided_broadcast_and_misaligned_inputs():
    spec = pf.rotary_spec(64, interleaved=True)
    base = torch.randn(2, 9, 6, 64, device=DEV).to(BF16)
    for q in (base.transpose(1, 2), base.transpose(1, 2)[:, ::2], base.transpose(1, 2)[:, :, 1::3],
              torch.randn(2 * 6 * 9 * 64 + 3, device=DEV).to(BF16)[3:].view(2, 6, 9, 64),
              torch.randn(1, 1, 9, 64, device=DEV).to(BF16).expand(2, 6, 9, 64),
              torch.randn(2, 6, 64, 9, device=DEV).to(BF16).transpose(2, 3)):
        rq, _ = pf.rotary_embedding(q, None, spec, 77)
        full = (torch.arange(q.shape[2], device=DEV) + 77).expand(2, -1)
        assert_within("q", rq, *_ref(q, spec, full))


def test_scalings_and_given_frequencies():
    q = torch.randn(1, 2, 50, 64, device=DEV)
    for spec in (pf.rotary_spec(64, scaling=pf.linear_scaling(4.0)), pf.rotary_spec(64, scaling=pf.ntk_scaling(8.0)),
                 pf.rotary_spec(64, scaling=pf.by_parts_scaling(16.0, 4096)),
                 pf.rotary_spec(64, frequencies=[0.5 ** i for i in range(32)], magnitude=0.7)):
        rq, _ = pf.rotary_embedding(q, None, spec, 100000)
        assert_within("q", rq, *_ref(q, spec, (torch.arange(50, device=DEV) + 100000).expand(1, -1)))


def test_other_stream_capture_and_empty():
    spec = pf.rotary_spec(128)
    q = torch.randn(2, 4, 16, 128, device=DEV).to(BF16)
    k = torch.randn(2, 1, 16, 128, device=DEV).to(BF16)
    want = pf.rotary_embedding(q, k, spec)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = pf.rotary_embedding(q, k, spec)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    pos = torch.arange(16, device=DEV, dtype=torch.int32)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gq, gk = pf.rotary_embedding(q, k, spec, pos)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(gq, want[0]) and torch.equal(gk, want[1])
    pos += 5
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(gq, pf.rotary_embedding(q, k, spec, 5)[0])
    e, _ = pf.rotary_embedding(q[:, :, :0], None, spec)
    assert e.shape == (2, 4, 0, 128)


def test_nan_and_infinity_stay_in_their_pair():
    spec = pf.rotary_spec(64)
    q = torch.randn(1, 1, 2, 64, device=DEV)
    q[0, 0, 0, 3] = math.nan
    q[0, 0, 1, 40] = math.inf
    r, _ = pf.rotary_embedding(q, None, spec, 3)
    bad = ~torch.isfinite(r[0, 0])
    assert bad[0].nonzero().flatten().tolist() == [3, 35] and bad[1].nonzero().flatten().tolist() == [8, 40]


def test_refusals():
    q = torch.randn(1, 2, 4, 64, device=DEV)
    spec = pf.rotary_spec(64)
    for bad in (lambda: pf.rotary_embedding(q[0], None, spec), lambda: pf.rotary_embedding(q.half(), None, spec),
                lambda: pf.rotary_embedding(q, q.to(BF16), spec), lambda: pf.rotary_embedding(q.cpu(), None, spec),
                lambda: pf.rotary_embedding(q, q[:, :, :2], spec), lambda: pf.rotary_embedding(q, None, pf.rotary_spec(32)),
                lambda: pf.rotary_embedding(q, None, spec, torch.zeros(4, device=DEV)),
                lambda: pf.rotary_embedding(q, None, spec, torch.zeros(3, device=DEV, dtype=torch.int32)),
                lambda: pf.rotary_embedding(q, None, spec, 1 << 31)):
        with pytest.raises(ValueError):
            bad()
