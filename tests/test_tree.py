"""Draft trees over caches of different lengths, the cached step of differential attention, and
the commit of accepted nodes: the oracle's own checks, refusals, and the kernels against the
oracle element by element (its bounds: oracle/diff.py)."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from machinelearning_amd import _capi
from machinelearning_amd import decode as dec
from machinelearning_amd import flash_cuda as fc
from oracle import diff as orc
from oracle import tree as ort
from tests.test_diff import HALF, TINY, within

gpu = pytest.mark.gpu


def draft(B, T, seed, pad=False, shape="mixed"):
    """Parents of B random trees."""
    g = torch.Generator().manual_seed(seed)
    t = torch.arange(T)
    if shape == "chain":
        up = (t - 1).expand(B, T).clone()
    elif shape == "star":
        up = torch.where(t > 0, 0, -1).expand(B, T).clone()
    elif shape == "roots":
        up = torch.full((B, T), -1)
    else:
        up = (torch.rand(B, T, generator=g) * (t + 1)).long().clamp(max=T - 1) - 1
        up = torch.where(torch.rand(B, T, generator=g) < 0.5, t - 1, up)
    if pad:
        n = torch.randint(0, T + 1, (B, 1), generator=g)
        up = torch.where(t < n, up, -2)
    return up.to(torch.int32)


def draw(B, T, H, Hkv, D, rows, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    q, k, v, ck, cv = (torch.randn(*s, generator=g).to(dtype) for s in (
        (B, T, H, D), (B, T, Hkv, D), (B, T, Hkv, D), (B, Hkv, rows, D), (B, Hkv, rows, D)))
    return q, k, v, ck, cv, (0.2 + 0.6 * torch.rand(H, generator=g)).to(dtype)


def check(out, lse, q, k, v, ck, cv, lens, parents, lam=None, scale=None, causal=True, gate=None):
    B, T, H, D = q.shape
    dtype = q.dtype
    scale = math.sqrt((1 if lam is None else 2) / D) if scale is None else scale
    out = out.cpu()
    worst = 0.0
    for b, (live, case) in enumerate(ort.cases(q, k, v, ck, cv, lens, parents, scale, lam, causal)):
        away = [t for t in range(T) if t not in live]
        assert (out[b, away] == 0).all(), "rows outside the tree are 0"
        if lse is not None:
            assert (lse[b, :, away] == float("-inf")).all()
        if case is None:
            continue
        ref, bound = case.out()[0], case.out_bound(HALF[dtype], TINY.get(dtype, 0.0))[0]
        if gate is not None:
            sig = torch.sigmoid(gate[b, live].double())[..., None]
            ref, bound = ref * sig, bound + 2.0 ** -20 * ref.abs()
        got = out[b, live].double()
        assert torch.isfinite(got).all(), b
        worst = max(worst, ((got - ref).abs() / bound).max().item())
        if lse is not None:
            err = (lse[b].cpu().double()[:, live] - case.lse[0][0]).abs()
            assert (err <= case.lse_bound()[0]).all(), (b, err.max())
    print(f"worst err/bound={worst:.3f}", flush=True)
    assert worst <= 1.0


def run(q, k, v, ck, cv, lens, parents, lam=None, check_lse=True, **kw):
    """attn_tree on the GPU, against the oracle. Rows behind the lengths are poison."""
    ck, cv = ck.clone(), cv.clone()
    for b, n in enumerate(lens.tolist()):
        ck[b, :, n:] = float("nan")
        cv[b, :, n:] = float("inf")
    cache = {"k": ck.cuda(), "v": cv.cuda(), "lens": lens.cuda()}
    res = dec.attn_tree(*(t.cuda() for t in (q, k, v)), cache, parents.cuda(),
                        lam=None if lam is None else lam.cuda(), return_lse=lam is None and check_lse,
                        gate=kw["gate"].cuda() if kw.get("gate") is not None else None,
                        scale=kw.get("scale"))
    out, lse = res if isinstance(res, tuple) else (res, None)
    assert out.dtype == q.dtype and out.shape == q.shape
    check(out, lse, q, k, v, ck, cv, lens, parents, lam, **kw)
    return out


# ---------------------------------------------------------------------------
# the oracle, and refusals (CPU)
# ---------------------------------------------------------------------------
def test_lines_of_descent():
    assert ort.lines([-1, 0, 0, 2, -1, 4, -2, 6, 9, 8, 3]) == [
        [0], [0, 1], [0, 2], [0, 2, 3], [4], [4, 5], None, None, None, None, [0, 2, 3, 10]]


def test_a_chain_is_causal_attention():
    q, k, v, ck, cv, lam = draw(2, 5, 4, 2, 32, 9, torch.float64)
    lens = torch.tensor([9, 4], dtype=torch.int32)
    for maps in (None, lam):
        trees = ort.cases(q, k, v, ck, cv, lens, torch.arange(5) - 1, 0.2, maps)
        plain = ort.cases(q, k, v, ck, cv, lens, None, 0.2, maps)
        for (a, x), (b, y) in zip(trees, plain):
            assert a == b
            torch.testing.assert_close(x.out(), y.out(), rtol=0, atol=1e-14)


def test_one_map_is_softmax_attention():
    q, k, v, _, _, _ = draw(1, 6, 2, 2, 32, 1, torch.float64)
    case = orc.Case(q, k, v, None, 0.2, orc.causal_keep(6, 6, True))
    qh, kh, vh = (t.transpose(1, 2) for t in (q, k, v))
    want = torch.nn.functional.scaled_dot_product_attention(qh, kh, vh, is_causal=True, scale=0.2)
    torch.testing.assert_close(case.out(), want.transpose(1, 2), rtol=0, atol=1e-12)


def step_shape(**kw):
    base = dict(B=2, T=4, H=4, Hkv=2, D=64, rows=100, causal=1, one_tree=0, maps=1, scale=0.125,
                dtype=_capi.MI_BF16, lam_dtype=0, k_batch_stride=12800, k_head_stride=6400,
                v_batch_stride=12800, v_head_stride=6400)
    base.update(kw)
    return _capi.MiStepShape(**base)


@pytest.mark.parametrize("kw,code", [
    (dict(B=-1), 2), (dict(T=-1), 2), (dict(rows=-1), 2), (dict(H=3), 2), (dict(Hkv=0), 2),
    (dict(D=48), 4), (dict(dtype=3), 3), (dict(maps=0), 14), (dict(maps=3), 14),
    (dict(maps=2, lam_dtype=9), 3), (dict(scale=0.0), 9), (dict(scale=float("nan")), 9),
    (dict(k_head_stride=12), 6), (dict(v_batch_stride=-8), 6), (dict(rows=0x7fffffff), 7),
    (dict(T=1 << 20, H=1 << 12, Hkv=1 << 12), 7)])
def test_abi_refuses_shapes(kw, code):
    lib, s, n = _capi.load(), step_shape(**kw), ctypes.c_longlong(-1)
    assert lib.mi_attn_step_workspace(ctypes.byref(s), ctypes.byref(n)) == code
    assert lib.mi_attn_step(*[None] * 12, ctypes.byref(s), None) == code
    assert lib.mi_attn_tree_commit(*[None] * 8, 1, ctypes.byref(s), None) == code
    assert n.value == -1


def test_abi_refuses_pointers():
    lib, s = _capi.load(), step_shape(rows=5000)     # enough for a workspace
    good = [0x1000] * 5 + [0x1004, 0x1004, None, None, 0x1000, None, 0x1000]

    def step(**kw):
        args = list(good)
        for i, x in kw.items():
            args[int(i[1:])] = x
        return lib.mi_attn_step(*args, ctypes.byref(kw.pop("s", s)), None)
    for i in (0, 1, 2, 3, 4, 9, 11):
        assert step(**{f"a{i}": None}) == 1, i
        assert step(**{f"a{i}": 0x1008}) == 6, i
    two = step_shape(maps=2, rows=5000)
    assert lib.mi_attn_step(*good, ctypes.byref(two), None) == 1          # no lam
    with_lse = list(good)
    with_lse[7], with_lse[10] = 0x1000, 0x1000
    assert lib.mi_attn_step(*with_lse, ctypes.byref(two), None) == 14
    big = step_shape(T=257)
    assert lib.mi_attn_step(*good, ctypes.byref(big), None) == 13
    commit = [0x1000, 0x1000, 0x1000, 0x1000, 0x1004, 0x1004, 0x1004, 0x2004]

    def put(P=3, s=s, **kw):
        args = list(commit)
        for i, x in kw.items():
            args[int(i[1:])] = x
        return lib.mi_attn_tree_commit(*args, P, ctypes.byref(s), None)
    for i in range(8):
        assert put(**{f"a{i}": None}) == 1, i
    for i in range(4):
        assert put(**{f"a{i}": 0x1008}) == 6, i
    assert put(a7=commit[4]) == 1                                        # lens_out is lens
    assert put(P=-1) == 2
    for shared in ("k_batch_stride", "k_head_stride", "v_batch_stride", "v_head_stride"):
        assert put(s=step_shape(**{shared: 0})) == 2
    empty = step_shape(B=0)
    assert lib.mi_attn_step(*[None] * 12, ctypes.byref(empty), None) == 0
    assert lib.mi_attn_tree_commit(*[None] * 8, 1, ctypes.byref(empty), None) == 0


def test_public_calls_refuse_cpu_tensors():
    q, k, v, ck, cv, lam = draw(1, 2, 2, 1, 64, 4, torch.float32)
    cache = {"k": ck, "v": cv, "lens": torch.tensor([2], dtype=torch.int32)}
    one = torch.zeros(1, 1, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU tensor"):
        dec.attn_tree(q, k, v, cache, torch.tensor([-1, 0]))
    with pytest.raises(ValueError, match="GPU tensor"):
        dec.diff_attn_cached(q, k, v, lam, {}, False)
    with pytest.raises(ValueError, match="GPU tensor"):
        dec.tree_commit(k, v, cache, one, one[0])


def test_ragged_cache_on_the_cpu():
    _, _, _, ck, cv, _ = draw(3, 1, 2, 2, 32, 5, torch.float32)
    new = dec.ragged_cache({"k": ck, "v": cv}, 9)
    assert new["k"].shape == (3, 2, 9, 32) and torch.equal(new["k"][:, :, :5], ck)
    assert torch.equal(new["v"][:, :, :5], cv) and new["lens"].tolist() == [5, 5, 5]
    assert new["lens"].dtype == torch.int32
    fewer = dec.ragged_cache({"k": ck, "v": cv}, 5, torch.tensor([2, 7, -1]))
    assert fewer["lens"].tolist() == [2, 5, 0]
    for bad in ({}, {"k": ck}, {"k": ck, "v": cv, "pos": 0}, {"k": ck, "v": cv, "lens": 0},
                {"k": ck, "v": cv[:, :1]}):
        with pytest.raises(ValueError, match="ragged_cache"):
            dec.ragged_cache(bad, 9)
    with pytest.raises(ValueError, match="rows must be at least"):
        dec.ragged_cache({"k": ck, "v": cv}, 4)
    with pytest.raises(ValueError, match="lens must be"):
        dec.ragged_cache({"k": ck, "v": cv}, 9, torch.tensor([1.0, 2.0, 3.0]))


@gpu
def test_refusals():
    q, k, v, ck, cv, lam = (t.cuda() for t in draw(2, 3, 4, 2, 64, 8, torch.bfloat16))
    lens = torch.tensor([3, 8], dtype=torch.int32, device="cuda")
    cache = {"k": ck, "v": cv, "lens": lens}
    up = torch.tensor([-1, 0, 1], device="cuda")

    def refused(match, call, *a, error=ValueError, **kw):
        with pytest.raises(error, match=match):
            call(*a, **kw)
    tree = dec.attn_tree
    refused("H a multiple", tree, q[:, :, :3], k, v, cache, up)
    refused("head_dim", tree, q[..., :48], k[..., :48], v[..., :48], cache, up)
    refused("dtypes", tree, q.float(), k, v, cache, up)
    refused("parents must be", tree, q, k, v, cache, up[:2])
    refused("parents must be", tree, q, k, v, cache, up.float())
    refused("parents must be", tree, q, k, v, cache, up.cpu())
    refused("parents must be", tree, q, k, v, cache, [-1, 0, 1])
    refused("parents must be", tree, q, k, v, cache, None)
    refused("lam must be", dec.diff_attn_cached, q, k, v, None, {}, False)
    refused("lens'\\] must be", tree, q, k, v, {**cache, "lens": lens[:1]}, up)
    refused("lens'\\] must be", tree, q, k, v, {**cache, "lens": lens.float()}, up)
    refused("only one of", tree, q, k, v, {"k": ck}, up)
    refused("lengths differ", tree, q, k, v, {**cache, "v": cv[:, :, :4]}, up)
    refused("must be \\(B, Hkv", tree, q, k, v, {**cache, "k": ck[:1]}, up)
    refused("windowed cache", tree, q, k, v, {**cache, "pos": lens}, up)
    refused("scale must be", tree, q, k, v, cache, up, scale=-1.0)
    refused("gate logits", tree, q, k, v, cache, up, gate=lam)
    refused("lam must be", tree, q, k, v, cache, up, lam=lam[:3])
    refused("no lse", tree, q, k, v, cache, up, lam=lam, return_lse=True)
    long = [t[:, :1].expand(-1, 257, -1, -1) for t in (q, k, v)]
    refused("at most 256", tree, *long, cache, torch.full((257,), -1, device="cuda"))
    refused("inference-only", tree, q.clone().requires_grad_(), k, v, cache, up, error=RuntimeError)
    refused("inference-only", tree, q, k, v, cache, up, lam=lam.clone().requires_grad_(),
            error=RuntimeError)
    refused("'lens'", dec.attn_cached, q, k, v, cache, False)
    refused("'lens'", dec.diff_attn_cached, q, k, v, lam, cache, False)
    refused("'pos'", dec.diff_attn_cached, q, k, v, lam, {"k": ck, "v": cv, "pos": lens}, False)
    path, count = torch.zeros(2, 1, dtype=torch.int32, device="cuda"), lens * 0
    put = dec.tree_commit
    refused("no 'lens'", put, k, v, {"k": ck, "v": cv}, path, count)
    refused("path must be", put, k, v, cache, path[0], count)
    refused("path must be", put, k, v, cache, path[:1], count)
    refused("count must be", put, k, v, cache, path, count[:1])
    refused("cache\\['k'\\] must be", put, k, v, {**cache, "k": ck.float()}, path, count)
    refused("cache\\['v'\\] must be", put, k, v, {**cache, "v": cv.transpose(2, 3)}, path, count)
    refused("cache\\['v'\\] must be", put, k, v, {**cache, "v": None}, path, count)
    refused("lengths differ", put, k, v, {**cache, "v": cv[:, :, :4]}, path, count)
    refused("share their rows", put, k, v, {**cache, "v": cv[:1].expand_as(cv)}, path, count)
    refused("share their rows", put, k, v, {**cache, "k": ck[:, :1].expand_as(ck)}, path, count)
    assert torch.equal(cache["lens"], lens)


# ---------------------------------------------------------------------------
# the kernels
# ---------------------------------------------------------------------------
DT = list(HALF)
name = lambda d: str(d)[6:]  # noqa: E731


@gpu
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("dtype", DT, ids=name)
@pytest.mark.parametrize("two", [False, True], ids=["one", "two"])
def test_small_trees(D, dtype, two):
    """Sizes round the blocks' edges, empty caches, padded and empty trees."""
    for n, (T, rep, lens) in enumerate([
            (1, 1, [0, 1, 31, 32]), (1, 4, [33, 64, 100, 0]), (3, 2, [5, 0, 64, 95]),
            (16, 2, [0, 63, 65, 1]), (17, 3, [96, 7, 130, 50]), (33, 1, [31, 32, 33, 0]),
            (40, 4, [12, 77, 128, 3])]):
        print((T, rep, lens), flush=True)
        q, k, v, ck, cv, lam = draw(4, T, 2 * rep, 2, D, max(lens) + 3, dtype, seed=n)
        run(q, k, v, ck, cv, torch.tensor(lens, dtype=torch.int32), draft(4, T, n, pad=n % 2 == 1),
            lam if two else None)


@gpu
@pytest.mark.parametrize("dtype", DT, ids=name)
@pytest.mark.parametrize("B,T,H,Hkv,D,longest", [
    (8, 1, 8, 8, 64, 3000), (3, 1, 32, 8, 128, 2500), (2, 32, 32, 8, 128, 1500),
    (1, 64, 8, 2, 64, 5000), (5, 27, 9, 3, 64, 700), (2, 200, 4, 1, 32, 900),
    (1, 256, 2, 2, 128, 300), (16, 2, 12, 12, 64, 1000)])
def test_long_caches(B, T, H, Hkv, D, longest, dtype):
    g = torch.Generator().manual_seed(T)
    lens = torch.randint(0, longest + 1, (B,), generator=g).to(torch.int32)
    lens[0] = longest
    q, k, v, ck, cv, lam = draw(B, T, H, Hkv, D, longest, dtype, seed=B)
    up = draft(B, T, B + T)
    run(q, k, v, ck, cv, lens, up)
    run(q, k, v, ck, cv, lens, up, lam)


@gpu
@pytest.mark.parametrize("B", [63, 64, 65, 128, 200])
def test_many_sequences(B):
    """The prefix sum over the lengths, 64 sequences a round."""
    g = torch.Generator().manual_seed(B)
    for T, H in ((1, 4), (5, 16)):
        lens = torch.randint(0, 150, (B,), generator=g).to(torch.int32)
        q, k, v, ck, cv, lam = draw(B, T, H, 2, 32, 150, torch.bfloat16, seed=T)
        run(q, k, v, ck, cv, lens, draft(B, T, B, pad=True), lam if T > 1 else None)


@gpu
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("dtype", DT, ids=name)
def test_room_to_spare(D, dtype):
    """Short sequences in a cache that could hold long ones: the steps' work is dealt out by
    what it could hold (the tests of short caches run a workgroup for each unit)."""
    for n, (B, T, rep, lens) in enumerate([
            (4, 1, 1, [0, 1, 31, 32]), (4, 1, 4, [33, 1399, 100, 0]), (4, 16, 2, [0, 63, 65, 1]),
            (4, 17, 3, [96, 7, 1400, 50]), (3, 33, 1, [31, 320, 0]), (2, 40, 8, [12, 777]),
            (70, 3, 2, [11 * i % 150 for i in range(70)])]):
        print((B, T, rep, lens), flush=True)
        q, k, v, ck, cv, lam = draw(B, T, 2 * rep, 2, D, 1400, dtype, seed=n)
        at = torch.tensor(lens, dtype=torch.int32)
        for maps in (None, lam):
            run(q, k, v, ck, cv, at, draft(B, T, n, pad=n % 2 == 1), maps)


@gpu
@pytest.mark.parametrize("shape", ["chain", "star", "roots"])
@pytest.mark.parametrize("T", [31, 64, 130, 256])
def test_tree_shapes(shape, T):
    """The deepest line (log2 T rounds of doubling), the widest, and no edge at all."""
    q, k, v, ck, cv, _ = draw(2, T, 4, 2, 64, 50, torch.bfloat16, seed=T)
    run(q, k, v, ck, cv, torch.tensor([50, 17], dtype=torch.int32), draft(2, T, 0, shape=shape))


@gpu
def test_strange_parents():
    """Later nodes, itself, far and negative numbers, and what hangs from such a node."""
    bad = torch.tensor([[-1, 0, 5, 2, 4, -3, 5, 1, 7], [8, -1, 1, 1 << 30, 3, 2, -(1 << 31), 0, 5]],
                       dtype=torch.int32)
    q, k, v, ck, cv, lam = draw(2, 9, 4, 2, 64, 40, torch.float16, seed=1)
    lens = torch.tensor([40, 11], dtype=torch.int32)
    a = run(q, k, v, ck, cv, lens, bad)
    run(q, k, v, ck, cv, lens, bad, lam)
    wide = bad.long()
    wide[1, 3] = 1 << 40
    assert torch.equal(run(q, k, v, ck, cv, lens, wide), a)
    # One tree for every sequence; lengths in 64 bits and past the cache's ends.
    one = torch.tensor([-1, 0, 0, 1, -2, 2, 3, 4, 1])
    b = run(q, k, v, ck, cv, lens, one)
    cache = {"k": ck.cuda(), "v": cv.cuda(), "lens": torch.tensor([1 << 33, 11], device="cuda")}
    each = one.to(torch.int32).expand(2, 9).cuda()
    assert torch.equal(dec.attn_tree(q.cuda(), k.cuda(), v.cuda(), cache, each), b)


@gpu
@pytest.mark.parametrize("T,rep", [(6, 1), (40, 2)])
@pytest.mark.parametrize("dtype", DT, ids=name)
def test_values_that_are_not_finite(T, rep, dtype):
    """Nodes outside the tree may hold anything. A node inside whose v is not finite makes the
    rows that see it NaN, and no others."""
    q, k, v, ck, cv, lam = draw(2, T, 2 * rep, 2, 64, 45, dtype, seed=3)
    lens = torch.tensor([45, 20], dtype=torch.int32)
    up = draft(2, T, 5)
    up[0, T - 2] = -2
    up[:, T - 1] = 0                        # a leaf
    clean = ort.lines(up[0])
    assert clean[T - 2] is None
    dirty = v.clone()
    dirty[0, T - 2] = float("nan")
    keys = k.clone()
    keys[0, T - 2] = float("inf")
    for maps in (None, lam):
        a = run(q, k, v, ck, cv, lens, up, maps)
        cache = {"k": ck.cuda(), "v": cv.cuda(), "lens": lens.cuda()}
        more = {} if maps is None else {"lam": maps.cuda()}
        b = dec.attn_tree(q.cuda(), keys.cuda(), dirty.cuda(), cache, up.cuda(), **more)
        assert torch.equal(a, b)
        for bad in (float("nan"), float("inf"), float("-inf")):
            worse = v.clone()
            worse[1, T - 1, 1, 7] = bad     # a leaf's: its own row alone sees it
            c = dec.attn_tree(q.cuda(), k.cuda(), worse.cuda(), cache, up.cuda(), **more)
            assert torch.isnan(c[1, T - 1, rep:]).all()
            c[1, T - 1, rep:] = a[1, T - 1, rep:]
            assert torch.equal(a, c)


@gpu
@pytest.mark.parametrize("two", [False, True], ids=["one", "two"])
def test_gate_scale_strides_and_types(two):
    q, k, v, ck, cv, lam = draw(3, 11, 6, 2, 64, 70, torch.bfloat16, seed=7)
    lam = lam if two else None
    lens, up = torch.tensor([70, 0, 33], dtype=torch.int32), draft(3, 11, 2, pad=True)
    gate = torch.randn(3, 11, 6, generator=torch.Generator().manual_seed(1))
    run(q, k, v, ck, cv, lens, up, lam, gate=gate)
    a = run(q, k, v, ck, cv, lens, up, lam, scale=0.7)
    # The same through views: a cache inside a larger buffer, heads before tokens.
    more = {"scale": 0.7} if lam is None else {"scale": 0.7, "lam": lam.float().cuda()}
    big = torch.full((3, 2, 200, 64), float("nan"), dtype=torch.bfloat16, device="cuda")
    big[:, :, 8:78] = ck.cuda()
    cache = {"k": big[:, :, 8:78], "v": cv.cuda().transpose(1, 2).contiguous().transpose(1, 2),
             "lens": lens.cuda()}
    moved = [t.cuda().transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    assert torch.equal(dec.attn_tree(*moved, cache, up.cuda().t().contiguous().t(), **more), a)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        b = dec.attn_tree(q.float().cuda(), k.cuda(), v.cuda(), cache, up.cuda(), **more)
    assert torch.equal(a, b)


@gpu
def test_cache_past_32_bits():
    """Rows whose byte offsets pass 32 bits (4.3 GB of keys). Keys of zero give every row the same
    weight, so the output is the values' mean: those of the last row alone are not zero. In
    float32 the weights' sum L + 1 is exact to 2^-24 L per addition of a few thousand partial
    sums, and the mean is rounded to bf16: 2^-8 covers both."""
    D, rows = 128, (1 << 24) + 104
    L = rows - 4
    ck = torch.zeros(1, 1, rows, D, dtype=torch.bfloat16, device="cuda")
    cv = torch.zeros_like(ck)
    cv[0, 0, L - 1] = torch.arange(D, device="cuda") * 2.0 ** 18
    cv[0, 0, L:] = float("nan")
    lens = torch.tensor([L], dtype=torch.int32, device="cuda")
    q, k, v = (torch.randn(1, 2, h, D, device="cuda").to(torch.bfloat16) for h in (4, 1, 1))
    want = cv[0, 0, L - 1].double() / L
    cache = {"k": ck, "v": cv, "lens": lens}
    up = torch.tensor([-1, -1], device="cuda")
    for lam, share in ((None, 1.0), (torch.full((4,), 0.25, device="cuda"), 0.75)):
        out = dec.attn_tree(q, k * 0, v * 0, cache, up, lam=lam).double()
        assert ((out - share * want).abs() <= 2.0 ** -8 * want).all()
    path, count = torch.tensor([[1, 0]], device="cuda"), torch.tensor([2], device="cuda")
    dec.tree_commit(k, v, cache, path, count)
    assert cache["lens"].item() == L + 2
    assert torch.equal(ck[0, 0, L:L + 2], k[0, [1, 0], 0]) and torch.equal(cv[0, 0, L:L + 2], v[0, [1, 0], 0])
    assert torch.isnan(cv[0, 0, L + 2:]).all() and not ck[0, 0, :L].any()


def off_by_one(t):
    """The same values, dense, one element behind a 16-byte boundary."""
    flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    flat[1:] = t.reshape(-1)
    return flat[1:].view(t.shape)


@gpu
@pytest.mark.parametrize("dtype", DT, ids=name)
def test_unaligned_blocks_and_shared_caches(dtype):
    q, k, v, ck, cv, lam = (t.cuda() for t in draw(3, 6, 4, 2, 64, 90, dtype, seed=3))
    cache = {"k": ck, "v": cv, "lens": torch.tensor([90, 4, 31], dtype=torch.int32, device="cuda")}
    up = draft(3, 6, 1).cuda()
    assert off_by_one(q).is_contiguous() and off_by_one(q).data_ptr() % 16 != 0
    for maps in (None, lam):
        want = dec.attn_tree(q, k, v, cache, up, lam=maps)
        assert torch.equal(dec.attn_tree(*map(off_by_one, (q, k, v)), cache, up, lam=maps), want)
        moved = {**cache, "k": off_by_one(ck), "v": off_by_one(cv)}
        assert torch.equal(dec.attn_tree(q, k, v, moved, up, lam=maps), want)
    want = dec.diff_attn_cached(q, k, v, lam, {"k": ck, "v": cv}, False, True)
    got = dec.diff_attn_cached(*map(off_by_one, (q, k, v)), lam, {"k": ck, "v": cv}, False, True)
    assert torch.equal(got, want)
    # One prompt's rows for every sequence of the batch.
    one = {**cache, "k": ck[:1].expand_as(ck), "v": cv[:1].expand_as(cv)}
    own = {**cache, "k": one["k"].contiguous(), "v": one["v"].contiguous()}
    assert torch.equal(dec.attn_tree(q, k, v, one, up), dec.attn_tree(q, k, v, own, up))
    a, b = ({n: t.clone() for n, t in cache.items()} for _ in range(2))
    path = torch.tensor([[0, 2], [1, 1], [5, 0]], dtype=torch.int32, device="cuda")
    dec.tree_commit(k, v, a, path, torch.tensor([2, 2, 1], dtype=torch.int32, device="cuda"))
    dec.tree_commit(off_by_one(k), off_by_one(v), b, path, torch.tensor([2, 2, 1], device="cuda"))
    assert all(torch.equal(a[n], b[n]) for n in a)


@gpu
@pytest.mark.parametrize("dtype", DT, ids=name)
@pytest.mark.parametrize("B,T,H,Hkv,E,L,causal", [
    (4, 1, 4, 4, 64, 300, True), (2, 1, 8, 2, 128, 1, False), (3, 7, 6, 3, 32, 0, True),
    (2, 33, 4, 1, 64, 130, True), (2, 33, 4, 1, 64, 130, False), (1, 300, 2, 2, 128, 95, True),
    (1, 70, 4, 2, 32, 1000, False), (4, 1, 48, 48, 32, 1500, True), (4, 5, 96, 48, 32, 1301, False)])
def test_diff_cached(B, T, H, Hkv, E, L, causal, dtype):
    q, k, v, ck, cv, lam = draw(B, T, H, Hkv, E, L, dtype, seed=L)
    cache = {"k": ck.cuda(), "v": cv.cuda()} if L else {}
    out = dec.diff_attn_cached(*(t.cuda() for t in (q, k, v, lam)), cache, False, causal)
    check(out, None, q, k, v, ck, cv, torch.full((B,), L), None, lam, causal=causal)


@gpu
@pytest.mark.parametrize("dtype", DT, ids=name)
def test_diff_cached_stream_is_the_training_call(dtype):
    """Blocks committed one after another give the rows of one causal call."""
    B, S, H, Hkv, E = 2, 60, 4, 2, 64
    q, k, v, _, _, lam = (t.cuda() for t in draw(B, S, H, Hkv, E, 1, dtype, seed=4))
    want = fc.diff_attn(q, k, v, lam)
    cache, at, outs = {}, 0, []
    for n in (7, 1, 1, 20, 1, 30):
        blk = slice(at, at + n)
        outs.append(dec.diff_attn_cached(q[:, blk], k[:, blk], v[:, blk], lam, cache, True, True))
        at += n
        assert cache["k"].shape == (B, Hkv, at, E)
    assert torch.equal(cache["k"], k.transpose(1, 2)) and torch.equal(cache["v"], v.transpose(1, 2))
    got = torch.cat(outs, 1)
    case = orc.Case(q, k, v, lam, math.sqrt(2 / E), orc.causal_keep(S, S, True))
    within("stream", got, case.out(), case.out_bound(HALF[dtype], TINY.get(dtype, 0.0)))
    within("call", want, case.out(), case.out_bound(HALF[dtype], TINY.get(dtype, 0.0)))


def committed(k, v, cache, path, count):
    """tree_commit's definition on the host."""
    k, v, path, count = (t.cpu() for t in (k, v, path, count))
    ck, cv, lens = (cache[n].cpu().clone() for n in ("k", "v", "lens"))
    rows = ck.shape[2]
    for b in range(k.shape[0]):
        n = min(max(int(lens[b]), 0), rows)
        take = min(max(int(count[b]), 0), path.shape[1], rows - n)
        for i in range(take):
            t = int(path[b, i])
            if 0 <= t < k.shape[1]:
                ck[b, :, n + i], cv[b, :, n + i] = k[b, t], v[b, t]
        lens[b] = n + take
    return ck, cv, lens


@gpu
@pytest.mark.parametrize("dtype", DT, ids=name)
@pytest.mark.parametrize("B,T,Hkv,D,P,rows", [(1, 1, 1, 32, 1, 4), (5, 9, 3, 64, 6, 40),
                                              (64, 64, 8, 128, 16, 80), (3, 4, 2, 64, 7, 3),
                                              (2, 5, 2, 128, 0, 9)])
def test_commit(B, T, Hkv, D, P, rows, dtype):
    """Every row that is not committed keeps its bits, behind the last one too."""
    g = torch.Generator().manual_seed(P)
    _, k, v, ck, cv, _ = draw(B, T, Hkv, Hkv, D, rows, dtype, seed=P)
    path = torch.randint(-1, T + 1, (B, P), generator=g)
    count = torch.randint(-1, P + 2, (B,), generator=g)
    lens = torch.randint(0, rows + 1, (B,), generator=g).to(torch.int32)
    for whole in (torch.int32, torch.int64):
        cache = {"k": ck.cuda(), "v": cv.cuda(), "lens": lens.cuda()}
        old = dict(cache)
        want = committed(k, v, cache, path, count)
        dec.tree_commit(k.cuda(), v.cuda(), cache, path.to(whole).cuda(), count.to(whole).cuda())
        for x, y in zip((cache["k"], cache["v"], cache["lens"]), want):
            assert torch.equal(x.cpu(), y)
        assert torch.equal(old["lens"].cpu(), lens) and cache["k"] is old["k"]


@gpu
@pytest.mark.parametrize("two", [False, True], ids=["one", "two"])
def test_speculative_rounds(two):
    """Prompt, then drafted rounds with different acceptance, then single tokens: the set as it
    is used. Every row against the oracle over the tokens that its sequence really holds."""
    B, H, Hkv, D, dtype = 3, 6, 2, 64, torch.bfloat16
    g = torch.Generator().manual_seed(0)

    def rand(*s):
        return torch.randn(*s, generator=g).to(dtype)
    lam = (0.2 + 0.6 * torch.rand(H, generator=g)).to(dtype) if two else None
    prompt = [rand(B, 21, h, D) for h in (H, Hkv, Hkv)]
    cache: dict = {}
    with torch.no_grad():
        if two:
            dec.diff_attn_cached(*(t.cuda() for t in prompt), lam.cuda(), cache, True, True)
        else:
            dec.attn_cached(*(t.cuda() for t in prompt), cache, True, True)
    cache = dec.ragged_cache(cache, 64)
    held = [(prompt[1][b], prompt[2][b]) for b in range(B)]     # each sequence's own k, v
    for T in (8, 13, 1, 5, 1):
        q, k, v = rand(B, T, H, D), rand(B, T, Hkv, D), rand(B, T, Hkv, D)
        up = draft(B, T, T, pad=T > 5)
        up[:, 0] = -1
        out = dec.attn_tree(q.cuda(), k.cuda(), v.cuda(), cache, up.cuda(),
                            lam=None if lam is None else lam.cuda())
        n = [h[0].shape[0] for h in held]
        ck = torch.zeros(B, Hkv, max(n), D, dtype=dtype)
        cv = torch.zeros_like(ck)
        for b, (hk, hv) in enumerate(held):
            ck[b, :, :n[b]], cv[b, :, :n[b]] = hk.transpose(0, 1), hv.transpose(0, 1)
        check(out, None, q, k, v, ck, cv, torch.tensor(n), up, lam)
        # Accept a random node's line of descent in each sequence, a different length each.
        ls = [ort.lines(up[b]) for b in range(B)]
        take = [max((x for x in s if x), key=lambda x: (len(x) * 7 + b) % 5) for b, s in enumerate(ls)]
        P = max(map(len, take))
        path = torch.tensor([x + [0] * (P - len(x)) for x in take], dtype=torch.int32)
        count = torch.tensor([len(x) for x in take], dtype=torch.int32)
        dec.tree_commit(k.cuda(), v.cuda(), cache, path.cuda(), count.cuda())
        held = [(torch.cat([hk, k[b, x]]), torch.cat([hv, v[b, x]]))
                for b, ((hk, hv), x) in enumerate(zip(held, take))]
        assert cache["lens"].tolist() == [h[0].shape[0] for h in held]


@gpu
def test_the_python_path_gives_the_same_bits(monkeypatch):
    """Arguments that need no conversion are launched by the C++ extension, any others (and all
    of them without it) by decode.py."""
    assert fc._load() is not None and fc._ext is not None
    q, k, v, ck, cv, lam = (t.cuda() for t in draw(3, 10, 4, 2, 64, 90, torch.bfloat16, seed=2))
    cache = {"k": ck, "v": cv, "lens": torch.tensor([90, 4, 31], dtype=torch.int32, device="cuda")}
    up = draft(3, 10, 1, pad=True).cuda()
    gate = torch.randn(3, 10, 4, device="cuda")
    path = torch.randint(0, 10, (3, 3), device="cuda", dtype=torch.int32)
    count = torch.tensor([0, 3, 1], device="cuda", dtype=torch.int32)

    def everything():
        mine = {n: t.clone() for n, t in cache.items()}
        out = [*dec.attn_tree(q, k, v, mine, up, return_lse=True),
               dec.attn_tree(q, k, v, mine, up[0], lam=lam, gate=gate, scale=0.3),
               dec.diff_attn_cached(q, k, v, lam, {"k": ck, "v": cv}, False, True),
               dec.diff_attn_cached(q, k, v, lam, {}, False, gate=gate)]
        dec.tree_commit(k, v, mine, path, count)
        return out + [mine[n] for n in ("k", "v", "lens")]
    fast = everything()
    for call in ("step", "tree_commit"):
        assert getattr(fc._ext, call) is not None
    monkeypatch.setattr(fc, "_ext", None)
    assert all(torch.equal(a, b) for a, b in zip(fast, everything()))


@gpu
@pytest.mark.parametrize("two", [False, True], ids=["one", "two"])
def test_reproducible_streams_and_graphs(two):
    """Twice the same bits, on another stream too, and as captured graphs replayed side by side:
    each has a workspace of its own."""
    B, T, H, Hkv, D, rows = 4, 12, 8, 2, 64, 3000
    lens = torch.tensor([3000, 1, 700, 0], dtype=torch.int32, device="cuda")
    sets = []
    for n in range(2):
        q, k, v, ck, cv, lam = (t.cuda() for t in draw(B, T, H, Hkv, D, rows, torch.bfloat16, seed=n))
        sets.append((q, k, v, {"k": ck, "v": cv, "lens": lens.clone()}, draft(B, T, n).cuda(),
                     lam if two else None))

    def call(s):
        return dec.attn_tree(*s[:5], lam=s[5])
    want = [call(s) for s in sets]
    assert all(torch.equal(call(s), w) for s, w in zip(sets, want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [call(s) for s in sets]
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graphs, outs, news, inputs = [], [], [], []      # a graph's inputs outlive it
    for s in sets:
        graph = torch.cuda.CUDAGraph()
        path = torch.zeros(B, 2, dtype=torch.int32, device="cuda")
        count = torch.ones(B, dtype=torch.int32, device="cuda")
        kept = dict(s[3])
        inputs.append((path, count))
        with torch.cuda.graph(graph):
            outs.append(call(s))
            dec.tree_commit(s[1], s[2], kept, path, count)
            news.append(kept["lens"])
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    for n in range(4):
        for s in sets:
            s[3]["lens"].copy_(torch.tensor([2900 + n, n, 700, 31 * n], dtype=torch.int32))
            s[0].mul_(-1.0 if n % 2 else 1.0)
        torch.cuda.synchronize()
        for st, graph in zip(streams, graphs):
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        for s, out, new in zip(sets, outs, news):
            # The commit wrote behind the lengths only: the step's result is as before it.
            assert torch.equal(out, call(s))
            assert torch.equal(new, s[3]["lens"] + 1)


@gpu
def test_empty_steps():
    q, k, v, ck, cv, lam = (t.cuda() for t in draw(2, 3, 4, 2, 64, 5, torch.bfloat16))
    up = torch.tensor([-1, 0, 0], device="cuda")
    cache = {"k": ck, "v": cv, "lens": torch.zeros(2, dtype=torch.int32, device="cuda")}
    assert dec.attn_tree(q[:, :0], k[:, :0], v[:, :0], cache, up[:0]).shape == (2, 0, 4, 64)
    none = {n: t[:0] for n, t in cache.items()}
    assert dec.attn_tree(q[:0], k[:0], v[:0], none, up).shape == (0, 3, 4, 64)
    # No cache at all, and a cache with no rows.
    a = dec.attn_tree(q, k, v, {}, up)
    assert torch.equal(a, dec.attn_tree(q, k, v, {"k": ck[:, :, :0], "v": cv[:, :, :0]}, up))
    assert torch.equal(a, dec.attn_tree(q, k, v, cache, up))
    check(a, None, *(t.cpu() for t in (q, k, v, ck, cv)), torch.zeros(2), up.cpu())
