"""Differential attention: the float64 oracle against autograd and differences, the public
call's refusals, and the kernels against the oracle element by element.

Tolerances are the oracle's bounds (oracle/diff.py): each rounding that the kernels make
counted once at half a unit in the last place, carried through absolute values. They hold for
every order of summation, so they are loose where errors average and tight where they cannot.
"""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from machinelearning_amd import _capi
from machinelearning_amd import flash_cuda as fc
from oracle import diff as orc

gpu = pytest.mark.gpu
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.float16: 2.0 ** -25}


def draw(B, S, H, Hkv, E, dtype, seed=0, std=1.0):
    g = torch.Generator().manual_seed(seed)
    q, k, v, do = (torch.randn(B, S, h, E, generator=g) * s
                   for h, s in ((H, std), (Hkv, 1.0), (Hkv, 1.0), (H, 1.0)))
    lam = 0.2 + 0.6 * torch.rand(H, generator=g)
    return [t.to(dtype) for t in (q, k, v, do)] + [lam.to(dtype)]


def case_of(q, k, v, lam, causal, scale=None):
    S, E = q.shape[1], q.shape[3]
    return orc.Case(q, k, v, lam, math.sqrt(2.0 / E) if scale is None else scale,
                    orc.causal_keep(S, S, causal))


def within(name, got, ref, bound):
    got, ref = got.detach().double().cpu(), ref.double()
    assert got.shape == ref.shape, (name, got.shape, ref.shape)
    if ref.numel() == 0:
        return
    assert torch.isfinite(got).all(), name
    ratio = ((got - ref).abs() / bound.clamp(min=1e-30)).max().item()
    print(f"{name}: max|err|={(got - ref).abs().max():.2e} of max|ref|={ref.abs().max():.2e}, "
          f"worst err/bound={ratio:.3f}", flush=True)
    assert ratio <= 1.0, (name, ratio)


def check_all(q, k, v, do, lam, causal, scale=None, lam_dtype=None):
    """Forward and gradients of the public call against the oracle."""
    dtype = q.dtype
    u, tiny = HALF[dtype], TINY.get(dtype, 0.0)
    lam = lam if lam_dtype is None else lam.to(lam_dtype)
    leaves = [t.cuda().requires_grad_() for t in (q, k, v, lam)]
    out = fc.diff_attn(*leaves, scale, causal=causal)
    assert out.dtype == dtype
    grads = torch.autograd.grad(out, leaves, do.cuda())
    ref = case_of(q, k, v, lam, causal, scale)
    within("out", out, ref.out(), ref.out_bound(u, tiny))
    for name, leaf, g, r, b in zip(("dq", "dk", "dv", "dlam"), leaves, grads, ref.grads(do),
                                   ref.grad_bounds(do, u, tiny)):
        assert g.dtype == leaf.dtype and g.shape == leaf.shape
        if name == "dlam":
            # Stored in lam's own type, computed from what the inputs' type left of O2.
            b = b + HALF[lam.dtype] * r.abs() + TINY.get(lam.dtype, 0.0)
        within(name, g, r, b)
    return out, grads


# ---------------------------------------------------------------------------
# the oracle (CPU)
# ---------------------------------------------------------------------------
def plain(q, k, v, lam, scale, keep):
    """Autograd's view of the formula, dense."""
    H, E = q.shape[2], q.shape[3]
    qh = q.transpose(1, 2)
    kh, vh = (t.transpose(1, 2).repeat_interleave(H // t.shape[2], 1) for t in (k, v))

    def attend(m):
        s = scale * qh[..., m] @ kh[..., m].transpose(-1, -2)
        return torch.softmax(s.masked_fill(~keep, float("-inf")), -1)
    P = attend(slice(0, E // 2)) - lam[:, None, None] * attend(slice(E // 2, E))
    return (P @ vh).transpose(1, 2)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("S,H,Hkv,E", [(7, 2, 1, 32), (33, 4, 4, 64), (1, 3, 3, 32), (40, 6, 2, 32)])
def test_oracle_matches_autograd(S, H, Hkv, E, causal):
    q, k, v, do, lam = draw(2, S, H, Hkv, E, torch.float64)
    ref = case_of(q, k, v, lam, causal)
    leaves = [t.requires_grad_() for t in (q, k, v, lam)]
    out = plain(*leaves, math.sqrt(2.0 / E), orc.causal_keep(S, S, causal))
    torch.testing.assert_close(out.detach(), ref.out(), rtol=0, atol=1e-12)
    for got, want in zip(torch.autograd.grad(out, leaves, do), ref.grads(do)):
        torch.testing.assert_close(got, want, rtol=0, atol=1e-11)


def test_oracle_gradients_match_differences():
    q, k, v, do, lam = draw(1, 9, 2, 1, 32, torch.float64, seed=3)
    args = [q, k, v, lam]
    grads = case_of(*args, True).grads(do)
    h = 1e-6
    for n, (x, g) in enumerate(zip(args, grads)):
        step = torch.randn(x.shape, generator=torch.Generator().manual_seed(n), dtype=torch.float64)
        up, down = list(args), list(args)
        up[n], down[n] = x + h * step, x - h * step
        num = ((case_of(*up, True).out() - case_of(*down, True).out()) * do).sum() / (2 * h)
        assert abs(num - (g * step).sum()) < 1e-6 * max(1.0, abs(num))


def test_oracle_special_cases():
    q, k, v, do, lam = draw(2, 12, 4, 2, 32, torch.float64, seed=1)
    # lam = 0 leaves the first map; equal halves leave (1 - lam) of one.
    one = case_of(q, k, v, torch.zeros(4, dtype=torch.float64), True)
    torch.testing.assert_close(one.out(), (one.P[0] @ one.vh).transpose(1, 2))
    q2, k2 = (torch.cat([t[..., :16]] * 2, -1) for t in (q, k))
    same = case_of(q2, k2, v, lam, True)
    torch.testing.assert_close(same.out(), (1 - lam)[:, None] * (same.P[0] @ same.vh).transpose(1, 2))


# ---------------------------------------------------------------------------
# refusals (no GPU: everything is refused before the library is asked to run)
# ---------------------------------------------------------------------------
def diff_shape(**kw):
    base = dict(B=1, S=8, H=2, Hkv=1, E=64, causal=1, scale=0.1, dtype=_capi.MI_BF16,
                lam_dtype=_capi.MI_F32)
    base.update(kw)
    return _capi.MiDiffShape(*(base[f] for f, _ in _capi.MiDiffShape._fields_))


@pytest.mark.parametrize("kw,code", [
    (dict(B=-1), 2), (dict(S=-1), 2), (dict(H=3, Hkv=2), 2), (dict(Hkv=0), 2), (dict(E=48), 4),
    (dict(E=256), 4), (dict(dtype=7), 3), (dict(lam_dtype=-1), 3), (dict(scale=0.0), 9),
    (dict(scale=float("nan")), 9), (dict(scale=float("inf")), 9), (dict(S=1 << 25, H=64), 7), (dict(S=1 << 24, dtype=_capi.MI_F32), 7)])
def test_abi_refuses_shapes(kw, code):
    lib, s, n = _capi.load(), diff_shape(**kw), ctypes.c_longlong(-1)
    assert lib.mi_attn_diff_bwd_workspace(ctypes.byref(s), ctypes.byref(n)) == code
    assert lib.mi_attn_diff_fwd(*[None] * 7, ctypes.byref(s), None) == code
    assert lib.mi_attn_diff_bwd(*[None] * 13, ctypes.byref(s), None) == code
    assert n.value == -1


def test_abi_refuses_pointers():
    lib, s = _capi.load(), diff_shape()
    assert lib.mi_attn_diff_fwd(*[None] * 7, ctypes.byref(s), None) == 1
    assert lib.mi_attn_diff_bwd(*[None] * 13, ctypes.byref(s), None) == 1
    assert lib.mi_attn_diff_bwd_workspace(ctypes.byref(s), None) == 1
    assert lib.mi_attn_diff_fwd(*[None] * 7, None, None) == 1
    # Misaligned pointers are refused before anything is launched.
    fwd = [0x1000, 0x1000, 0x1000, 0x1004, 0x1000, 0x1000, 0x1004]
    for i in (0, 1, 2, 4, 5):
        bad = list(fwd)
        bad[i] += 8
        assert lib.mi_attn_diff_fwd(*bad, ctypes.byref(s), None) == 6, i
    bwd = [0x1000] * 13
    for i in (0, 1, 2, 4, 5, 6, 8, 9, 10, 11):
        bad = list(bwd)
        bad[i] += 8
        assert lib.mi_attn_diff_bwd(*bad, ctypes.byref(s), None) == 6, i
    empty = diff_shape(S=0)
    assert lib.mi_attn_diff_fwd(*[None] * 7, ctypes.byref(empty), None) == 0
    assert lib.mi_attn_diff_bwd(*[None] * 13, ctypes.byref(empty), None) == 0


def test_public_call_refuses_cpu_tensors_and_bad_scales():
    q, k, v, _, lam = draw(1, 4, 2, 1, 64, torch.float32)
    with pytest.raises(ValueError, match="unsupported inputs"):
        fc.diff_attn(q, k, v, lam)


@gpu
def test_public_call_refusals():
    q, k, v, _, lam = (t.cuda() for t in draw(1, 4, 4, 2, 64, torch.bfloat16))
    with pytest.raises(ValueError, match="scale must be finite"):
        fc.diff_attn(q, k, v, lam, float("nan"))
    for bad in (lam[:3], lam.double(), lam.cpu(), 0.5, lam[:, None]):
        with pytest.raises(ValueError, match="lam must be"):
            fc.diff_attn(q, k, v, bad)
    for bad in ((q[..., :48], k[..., :48], v[..., :48]), (q, k[:, :3], v), (q, k, v[:, :, :1]),
                (q.float(), k, v), (q[:, :, :3], k, v)):
        with pytest.raises(ValueError, match="unsupported inputs"):
            fc.diff_attn(*bad, lam[:bad[0].shape[2]])
    with pytest.raises(RuntimeError, match="once_differentiable"):
        x = q.clone().requires_grad_()
        g, = torch.autograd.grad(fc.diff_attn(x, k, v, lam).float().square().sum(), x,
                                create_graph=True)
        g.sum().backward()


# ---------------------------------------------------------------------------
# the kernels
# ---------------------------------------------------------------------------
LENGTHS = [1, 2, 31, 32, 33, 64, 65, 127, 128, 129, 200]


@gpu
@pytest.mark.parametrize("E", [32, 64, 128])
@pytest.mark.parametrize("dtype", list(HALF), ids=lambda d: str(d)[6:])
@pytest.mark.parametrize("causal", [True, False])
def test_lengths(E, dtype, causal):
    """Lengths round the tiles' edges."""
    for n, S in enumerate(LENGTHS):
        print(f"S={S}", flush=True)
        check_all(*draw(1, S, 2, 1, E, dtype, seed=n), causal)


@gpu
@pytest.mark.parametrize("dtype", list(HALF), ids=lambda d: str(d)[6:])
@pytest.mark.parametrize("B,S,H,Hkv,E,causal", [
    (2, 300, 4, 4, 64, True), (3, 257, 6, 2, 32, True), (1, 700, 8, 1, 128, True),
    (8, 130, 8, 8, 64, False), (2, 513, 12, 4, 64, True), (5, 77, 9, 3, 32, False),
    (1, 1500, 2, 2, 128, False),
    # Enough key blocks for a workgroup each (the others share theirs out).
    (64, 130, 16, 16, 32, True), (64, 200, 32, 16, 64, False), (32, 129, 16, 16, 128, True)])
def test_shapes(B, S, H, Hkv, E, causal, dtype):
    check_all(*draw(B, S, H, Hkv, E, dtype, seed=S), causal)


@gpu
def test_peaked_scores():
    """Sharp maps: nearly all of a row's weight on a few keys, maxima that move between tiles."""
    for dtype in HALF:
        check_all(*draw(1, 400, 2, 2, 64, dtype, seed=5, std=4.0), True)


@gpu
@pytest.mark.parametrize("scale", [0.3, -0.2, 0.0, 1e-30])
def test_scales(scale):
    q, k, v, do, lam = draw(2, 90, 4, 2, 64, torch.bfloat16, seed=9)
    check_all(q, k, v, do, lam, True, scale)


@gpu
@pytest.mark.parametrize("lam_dtype", list(HALF), ids=lambda d: str(d)[6:])
def test_lam_types_and_broadcast(lam_dtype):
    q, k, v, do, lam = draw(2, 150, 6, 3, 64, torch.float16, seed=2)
    check_all(q, k, v, do, lam.float(), True, lam_dtype=lam_dtype)
    # One weight for every head: its gradient is the heads' sum.
    for one in (torch.tensor(0.4), torch.tensor([0.4])):
        one = one.to(lam_dtype).cuda().requires_grad_()
        leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
        out = fc.diff_attn(*leaves, one)
        g, = torch.autograd.grad(out, one, do.cuda())
        assert g.shape == one.shape and g.dtype == lam_dtype
        each = one.detach().reshape(-1).expand(6).contiguous().requires_grad_()
        per, = torch.autograd.grad(fc.diff_attn(*leaves, each), each, do.cuda())
        torch.testing.assert_close(g.float().reshape(()), per.float().sum(),
                                   rtol=8 * HALF[lam_dtype], atol=8 * HALF[lam_dtype] * 6)


@gpu
def test_lam_of_zero_and_of_any_sign():
    q, k, v, do, _ = draw(1, 130, 4, 4, 32, torch.bfloat16, seed=4)
    check_all(q, k, v, do, torch.tensor([0.0, -0.7, 1.0, 3.0]).bfloat16(), True)


@gpu
def test_empty_inputs():
    for B, S in ((0, 5), (2, 0)):
        leaves = [torch.empty(B, S, 2, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
                  for _ in range(3)]
        lam = torch.ones(2, device="cuda", requires_grad=True)
        out = fc.diff_attn(*leaves, lam)
        grads = torch.autograd.grad(out, leaves + [lam], torch.empty_like(out))
        assert out.shape == (B, S, 2, 64) and grads[0].shape == out.shape
        assert grads[3].tolist() == [0.0, 0.0]


@gpu
def test_strides_autocast_and_no_grad():
    q, k, v, do, lam = (t.cuda() for t in draw(2, 100, 4, 2, 64, torch.bfloat16, seed=6))
    base = fc.diff_attn(q, k, v, lam)
    for t in (q, k, v, lam):
        assert not t.requires_grad
    # Views in other orders: heads before rows, a slice of wider rows, a reversed copy.
    swapped = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    assert torch.equal(fc.diff_attn(*swapped, lam), base)
    wide = [torch.cat([t, t], -1)[..., :64] for t in (q, k, v)]
    assert torch.equal(fc.diff_attn(*wide, torch.stack([lam, lam], 1)[:, 0]), base)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        auto = fc.diff_attn(q.float(), k.float(), v, lam.float())
    assert auto.dtype == torch.bfloat16
    assert torch.equal(auto, fc.diff_attn(q, k, v, lam.float()))
    leaves = [t.clone().requires_grad_() for t in (q, k, v, lam)]
    strided = torch.stack([do, do], 0).transpose(0, 1).select(1, 0)
    a = torch.autograd.grad(fc.diff_attn(*leaves), leaves, strided)
    b = torch.autograd.grad(fc.diff_attn(*leaves), leaves, do)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    with torch.no_grad():
        assert torch.equal(fc.diff_attn(*leaves), base)


@gpu
@pytest.mark.parametrize("need", ["q", "k", "v", "lam"])
def test_one_leaf_alone(need):
    names = ("q", "k", "v", "lam")
    q, k, v, do, lam = (t.cuda() for t in draw(1, 70, 2, 2, 64, torch.float16, seed=8))
    every = [t.clone().requires_grad_() for t in (q, k, v, lam)]
    want = dict(zip(names, torch.autograd.grad(fc.diff_attn(*every), every, do)))
    args = [t.clone().requires_grad_(n == need) for n, t in zip(names, (q, k, v, lam))]
    got, = torch.autograd.grad(fc.diff_attn(*args), [args[names.index(need)]], do)
    assert torch.equal(got, want[need])


@gpu
def test_reproducible_and_the_python_node_agrees(monkeypatch):
    q, k, v, do, lam = (t.cuda() for t in draw(2, 333, 6, 2, 64, torch.bfloat16, seed=11))

    def once():
        leaves = [t.clone().requires_grad_() for t in (q, k, v, lam)]
        out = fc.diff_attn(*leaves)
        return (out,) + torch.autograd.grad(out, leaves, do)
    first = once()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, once()))
    monkeypatch.setattr(fc, "_ext", None)
    assert all(torch.equal(a, b) for a, b in zip(first, once()))


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=lambda d: str(d)[6:])
@pytest.mark.parametrize("S,E,causal", [(2, 64, True), (3, 64, False), (9, 128, True), (64, 32, False),
                                        (65, 64, True), (200, 128, False), (333, 64, True)])
def test_dlam_has_no_rounding_to_16_bits(S, E, causal, dtype):
    """With 16-bit inputs and a float32 lam, dlam = -sum P_2 G: G's products are exact in float32
    and its sum of E of them is off by at most E 2^-24 of sum_d |dout_d v_d| =: A; P_2 is off by
    the score's sum (E / 2 terms), its scale and the LSE, each a few 2^-24 of numbers below 16
    here, and the exponential's 2^-22: below 2^-18 of P_2, and the rows' sums of P_2 are as near
    to 1. With the sums over keys and rows (S^2 <= 2^17 terms in short chains: below 2^-18) that
    is under 2^-15 sum P_2 A."""
    q, k, v, do, lam = (t.cuda() for t in draw(2, S, 4, 2, E, dtype, seed=S))
    w = lam.float().requires_grad_()
    got, = torch.autograd.grad(fc.diff_attn(q, k, v, w, causal=causal), [w], do)
    qd, kd, vd, dd = (t.cpu().double().transpose(1, 2) for t in (q, k, v, do))
    kd, vd = (t.repeat_interleave(2, 1) for t in (kd, vd))
    s = qd[..., E // 2:] @ kd[..., E // 2:].transpose(2, 3).contiguous() * (2 / E) ** 0.5
    if causal:
        s = s.masked_fill(torch.ones(S, S).triu(1).bool(), float("-inf"))
    p2 = torch.softmax(s, -1)
    want = -(p2 * (dd @ vd.transpose(2, 3).contiguous())).sum((0, 2, 3))
    bound = 2.0 ** -15 * (p2 * (dd.abs() @ vd.abs().transpose(2, 3).contiguous())).sum((0, 2, 3))
    worst = ((got.cpu().double() - want).abs() / bound).max().item()
    print(f"worst err/bound={worst:.3f}", flush=True)
    assert worst <= 1.0


@gpu
@pytest.mark.parametrize("plain_node", [False, True], ids=["cpp", "python"])
def test_unaligned_tensors(plain_node, monkeypatch):
    """Dense pieces of larger tensors that begin anywhere: inputs, and the gradient that a
    concatenation hands back."""
    if plain_node:
        assert fc._load() is not None
        monkeypatch.setattr(fc, "_ext", None)
    g = torch.Generator().manual_seed(5)
    q, k, v = (torch.randn(2, 33, h, 64, generator=g).to("cuda", torch.bfloat16) for h in (4, 2, 2))
    lam = torch.rand(4, generator=g).cuda()
    weight = torch.randn(1 + q.numel(), generator=g).to("cuda", torch.bfloat16)

    def step(shift):
        leaves, seen = [], []
        for t in (q, k, v):
            leaf = torch.cat([t.new_zeros(shift), t.reshape(-1)]).requires_grad_()
            leaves.append(leaf)
            seen.append(leaf[shift:].view(t.shape))
        if shift:
            assert all(t.is_contiguous() and t.data_ptr() % 16 != 0 for t in seen)
        w = lam.clone().requires_grad_()
        y = fc.diff_attn(*seen, w)
        flat = torch.cat([y.new_zeros(shift), y.reshape(-1)])      # its gradient: a shifted piece
        grads = torch.autograd.grad(flat, leaves + [w], weight[1 - shift:])
        return [y, grads[3]] + [t[shift:] for t in grads[:3]]
    assert all(torch.equal(a, b) for a, b in zip(step(0), step(1)))


@gpu
def test_other_stream_and_graph():
    q, k, v, do, lam = (t.cuda() for t in draw(2, 260, 4, 2, 64, torch.bfloat16, seed=12))
    leaves = [t.clone().requires_grad_() for t in (q, k, v, lam)]
    out = fc.diff_attn(*leaves)
    want = (out.detach(),) + torch.autograd.grad(out, leaves, do)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = fc.diff_attn(*leaves)
        got = (out.detach(),) + torch.autograd.grad(out, leaves, do)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    del out, got
    # Captured, then replayed on other values; every replay against the eager call.
    static = [t.clone().requires_grad_() for t in (q, k, v, lam)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cap = fc.diff_attn(*static)
        cap = (cap.detach(),) + torch.autograd.grad(cap, static, do)
    for n in range(4):
        new = [t.cuda() for t in draw(2, 260, 4, 2, 64, torch.bfloat16, seed=20 + n)]
        with torch.no_grad():
            for s, x in zip(static, (new[0], new[1], new[2], new[4])):
                s.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        eager = [t.detach().clone().requires_grad_() for t in static]
        out = fc.diff_attn(*eager)
        ref = (out.detach(),) + torch.autograd.grad(out, eager, do)
        assert all(torch.equal(a, b) for a, b in zip(cap, ref))


@gpu
def test_16_bit_inputs_without_the_mfma_path(monkeypatch):
    """Where the 16-bit probe failed, float32 arithmetic on upcast copies."""
    q, k, v, do, lam = draw(1, 80, 2, 1, 64, torch.bfloat16, seed=13)
    monkeypatch.setattr(fc, "_mma_ok", False)
    check_all(q, k, v, do, lam, True)
