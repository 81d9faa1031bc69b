"""Rotary positions on the GPU against the 64-bit form: values, gradients, strides, refusals."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwAD

import paged_ref as ref
from helpers import require_gpu
from tasft_amd.exceptions import KernelError
from tasft_amd.kernels import append_paged, apply_rotary, rotary_frequencies

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]


def _check(got, x, positions, inv, scale, inter, inverse=False, what=""):
    want = ref.rotate(x.cpu(), positions.cpu(), inv.cpu(), scale, inter, inverse)
    bound = ref.rotate_bound(x.cpu(), want, inv.cpu(), scale, inter, x.dtype)
    err = (got.detach().cpu().double() - want).abs()
    assert bool((err <= bound).all()), f"{what}: {float((err - bound).max()):.3e} over the bound"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize(("D", "R"), [(128, 128), (64, 32), (128, 16), (80, 20), (96, 24), (64, 64), (256, 256),
                                      (6, 2), (40, 8)])
def test_values(D, R, inter, dtype):
    dev = require_gpu()
    print(f"rotary D={D} R={R} interleaved={inter} {dtype}", flush=True)
    g = torch.Generator().manual_seed(D + R)
    inv, scale = rotary_frequencies(R, 10000.0, device=dev)
    for B, S, hq, hkv in ((2, 37, 6, 3), (1, 1, 1, 1), (3, 1500, 2, 2)):
        q = torch.randn((B, hq, S, D), generator=g).to(dtype).to(dev)
        k = torch.randn((B, hkv, S, D), generator=g).to(dtype).to(dev)
        pos = torch.randint(0, 100000, (B, S), generator=g).to(dev)
        a, b = apply_rotary(q, k, pos, inv, interleaved=inter, scale=1.25)
        _check(a, q, pos[:, None], inv, 1.25, inter, what="q")
        _check(b, k, pos[:, None], inv, 1.25, inter, what="k")
        a2, none = apply_rotary(q, None, pos, inv, interleaved=inter, scale=1.25)
        assert none is None and torch.equal(a, a2)


@pytest.mark.parametrize("dtype", DTYPES)
def test_positions_and_layouts(dtype):
    """int32 and int64 positions of any size, shared by the batch or not; packed rows; transposed,
    expanded, sliced and misaligned inputs give what contiguous ones give."""
    dev = require_gpu()
    g = torch.Generator().manual_seed(3)
    B, S, H, D = 2, 33, 4, 64
    inv, scale = rotary_frequencies(D, 500000.0, {"rope_type": "linear", "factor": 4.0}, device=dev)
    base = torch.randn((B, S, H, D), generator=g).to(dtype).to(dev)
    q = base.transpose(1, 2)
    far = torch.arange(S, dtype=torch.int64, device=dev) + 2 ** 31 - 7
    print("rotary layouts", flush=True)
    out, _ = apply_rotary(q, None, far, inv)
    _check(out, q, far, inv, scale, False)
    near = torch.arange(S, device=dev)
    want, _ = apply_rotary(q.contiguous(), None, near, inv)
    for pos in (near.to(torch.int32), near.expand(B, S), near.view(1, S), near.to(torch.int32).expand(B, S)):
        got, kk = apply_rotary(q, q, pos, inv)
        assert torch.equal(got, want) and torch.equal(kk, want)
        assert got.stride() == q.stride()
    packed, _ = apply_rotary(base[0], None, near, inv)
    assert torch.equal(packed, want[0].transpose(0, 1))
    wide = torch.zeros((B, S, H, D + 3), dtype=dtype, device=dev)
    wide[..., 1:D + 1] = base
    odd = wide[..., 1:D + 1].transpose(1, 2)  # rows of 67 elements, two bytes off: no vectors
    assert torch.equal(apply_rotary(odd, None, near, inv)[0], want)
    every2 = torch.empty((B, H, S, 2 * D), dtype=dtype, device=dev)[..., ::2].copy_(q)
    assert torch.equal(apply_rotary(every2, None, near, inv)[0], want)
    one = q[:, :1, :1].expand(B, H, S, D)
    assert torch.equal(apply_rotary(one, None, near, inv)[0], apply_rotary(one.contiguous(), None, near, inv)[0])
    assert torch.equal(apply_rotary(q, None, near, inv.float())[0].float().isfinite().all().cpu(), torch.tensor(True))
    empty, _ = apply_rotary(q[:, :, :0], None, near[:0], inv)
    assert empty.shape == (B, H, 0, D)
    # Infinities and NaN stay with their pair; position 0 keeps every value.
    same, _ = apply_rotary(q, None, torch.zeros(S, dtype=torch.int64, device=dev), inv)
    assert torch.equal(same, q)
    bad = q.contiguous()
    bad[0, 1, 5, 3] = float("nan")
    got, _ = apply_rotary(bad, None, near, inv)
    spoiled = torch.isnan(got)
    assert spoiled.sum() == 2 and spoiled[0, 1, 5, 3] and spoiled[0, 1, 5, 3 + D // 2]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("inter", [False, True])
def test_gradients(inter, dtype):
    dev = require_gpu()
    print(f"rotary gradients interleaved={inter} {dtype}", flush=True)
    g = torch.Generator().manual_seed(11)
    B, S, D, R = 2, 70, 128, 64
    inv, scale = rotary_frequencies(R, 10000.0, {"rope_type": "yarn", "factor": 4.0,
                                                 "original_max_position_embeddings": 4096}, device=dev)
    q = torch.randn((B, 4, S, D), generator=g).to(dtype).to(dev).requires_grad_(True)
    k = torch.randn((B, 2, S, D), generator=g).to(dtype).to(dev).requires_grad_(True)
    gq, gk = torch.randn(q.shape, generator=g).to(dtype).to(dev), torch.randn(k.shape, generator=g).to(dtype).to(dev)
    pos = torch.randint(0, 5000, (B, S), generator=g).to(dev)
    a, b = apply_rotary(q, k, pos, inv, interleaved=inter, scale=scale)
    dq, dk = torch.autograd.grad((a, b), (q, k), (gq, gk), retain_graph=True)
    _check(dq, gq, pos[:, None], inv, scale, inter, inverse=True, what="dq")
    _check(dk, gk, pos[:, None], inv, scale, inter, inverse=True, what="dk")
    # One output alone, one input alone, a gradient of stride 0.
    assert torch.equal(torch.autograd.grad(b, k, gk, retain_graph=True)[0], dk)
    only, _ = apply_rotary(q, k.detach(), pos, inv, interleaved=inter, scale=scale)
    assert torch.equal(torch.autograd.grad(only, q, gq)[0], dq)
    ones = torch.ones((), dtype=dtype, device=dev).expand(a.shape)
    assert torch.equal(torch.autograd.grad(a, q, ones, retain_graph=True)[0],
                       torch.autograd.grad(a, q, ones.contiguous(), retain_graph=True)[0])
    # Against differences: the operator is linear, <g, R(x + d) - R(x)> = <R^T g, d>, in 64 bits of
    # the rounded values; every factor carries roundings of half a step.
    d = torch.randn(q.shape, generator=g).to(dtype).to(dev)
    moved, _ = apply_rotary(d, None, pos, inv, interleaved=inter, scale=scale)
    left = (gq.double() * moved.double()).sum()
    right = (dq.double() * d.double()).sum()
    size = (gq.double().abs() * moved.double().abs()).sum() + (dq.double().abs() * d.double().abs()).sum()
    assert abs(float(left - right)) <= 1.01 * ref.half_step(dtype) * float(size) + 1e-3
    # A second derivative: the gradient of the gradient with respect to its own input.
    gq2 = gq.clone().requires_grad_(True)
    (dq2,) = torch.autograd.grad(a, q, gq2, create_graph=True)
    (back,) = torch.autograd.grad(dq2, gq2, d)
    assert torch.equal(back, moved)


def test_graph_replay_and_streams():
    dev = require_gpu()
    inv, _ = rotary_frequencies(128, device=dev)
    q = torch.randn(2, 8, 50, 128, device=dev).bfloat16()
    k = torch.randn(2, 2, 50, 128, device=dev).bfloat16()
    pos = torch.arange(50, device=dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    print("rotary graph", flush=True)
    with torch.cuda.stream(side):
        on_side = apply_rotary(q, k, pos, inv)
        on_side = apply_rotary(q, k, pos, inv)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = apply_rotary(q, k, pos, inv)
    for step in range(3):
        q.normal_()
        pos += 17
        want = apply_rotary(q, k, pos, inv)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
    assert on_side[0].shape == q.shape


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("inter", [False, True])
def test_forward_mode(inter, dtype):
    """Forward-mode derivatives: the operator is linear, so a tangent is rotated as its value is; with
    and without gradients recorded, and of a gradient."""
    dev = require_gpu()
    print(f"rotary forward mode interleaved={inter} {dtype}", flush=True)
    g = torch.Generator().manual_seed(21)
    B, S, D, R = 2, 19, 64, 32
    inv, _ = rotary_frequencies(R, device=dev)
    q, k, tq, tk = (torch.randn((B, h, S, D), generator=g).to(dtype).to(dev) for h in (4, 2, 4, 2))
    pos = torch.randint(0, 5000, (B, S), generator=g).to(dev)
    kw = {"interleaved": inter, "scale": 1.25}
    want = apply_rotary(q, k, pos, inv, **kw)
    moved = apply_rotary(tq, tk, pos, inv, **kw)
    _check(moved[0], tq, pos[:, None], inv, 1.25, inter, what="tangent")
    for grads in (False, True):
        a, b = q.clone().requires_grad_(grads), k.clone().requires_grad_(grads)
        for on in ((True, True), (True, False), (False, True)):
            with fwAD.dual_level():
                da, db = (fwAD.make_dual(x, t) if yes else x for x, t, yes in ((a, tq, on[0]), (b, tk, on[1])))
                got = [fwAD.unpack_dual(x) for x in apply_rotary(da, db, pos, inv, **kw)]
                for yes, (value, tangent), x, t in zip(on, got, want, moved):
                    assert torch.equal(value, x)
                    assert torch.equal(tangent, t) if yes else tangent is None or not tangent.any()
            with fwAD.dual_level(), torch.no_grad():
                only, none = apply_rotary(fwAD.make_dual(q, tq), None, pos, inv, **kw)
                assert none is None and torch.equal(fwAD.unpack_dual(only).tangent, moved[0])
    # Reverse over forward: a tangent that needs a gradient.
    t = tq.clone().requires_grad_(True)
    with fwAD.dual_level():
        out, _ = apply_rotary(fwAD.make_dual(q, t), None, pos, inv, **kw)
        (back,) = torch.autograd.grad(fwAD.unpack_dual(out).tangent, t, tq)
    _check(back, tq, pos[:, None], inv, 1.25, inter, inverse=True, what="gradient of the tangent")
    # Forward over reverse: a gradient's tangent.
    x = q.clone().requires_grad_(True)
    out, _ = apply_rotary(x, None, pos, inv, **kw)
    with fwAD.dual_level():
        (gx,) = torch.autograd.grad(out, x, fwAD.make_dual(q, tq))
        tangent = fwAD.unpack_dual(gx).tangent
    assert tangent is not None and torch.equal(tangent, back)


def test_more_tokens_than_one_launch_takes():
    """A launch holds fewer than 2^32 threads, 2^24 tokens of a workgroup each."""
    dev = require_gpu()
    t, d = (1 << 24) + 700, 8
    inv, _ = rotary_frequencies(d, device=dev)
    q = torch.randn((t, 1, d), device=dev).bfloat16()
    k = torch.randn((t, 1, d), device=dev).bfloat16()
    pos = torch.arange(t, device=dev) * 3 + 1
    print("rotary of 2^24 + 700 tokens", flush=True)
    a, b = apply_rotary(q, k, pos, inv)
    for part in (slice(0, 1000), slice((1 << 24) - 1500, (1 << 24) + 600), slice(t - 50, t)):
        x, y = apply_rotary(q[part], k[part], pos[part], inv)
        assert torch.equal(a[part], x) and torch.equal(b[part], y)
        _check(x, q[part], pos[part][:, None], inv, 1.0, False)
    # Appended: two sequences, the second's tokens in the second launch.
    page, first = 1 << 12, (1 << 24) + 100
    lens = [first, t - first]
    per = -(-first // page)
    table = torch.arange(2 * per, dtype=torch.int32, device=dev).view(2, per)
    kp = torch.zeros((2 * per, page, 1, d), dtype=q.dtype, device=dev)
    vp = torch.zeros_like(kp)
    cu = torch.tensor([0, first, t], dtype=torch.int32, device=dev)
    kvl = torch.tensor(lens, dtype=torch.int32, device=dev)
    print("append of 2^24 + 700 tokens", flush=True)
    out = append_paged(q, k, q, kp, vp, table, kvl, cu, inv, positions=pos)
    assert torch.equal(out, a)
    for n, (s0, s1) in enumerate(((0, first), (first, t))):
        rows = slice(n * per * page, n * per * page + s1 - s0)
        assert torch.equal(kp.view(-1, 1, d)[rows], b[s0:s1]) and torch.equal(vp.view(-1, 1, d)[rows], q[s0:s1])


@pytest.mark.parametrize("dtype", DTYPES)
def test_overlapping_rows(dtype):
    """Rows that overlap (windows one element apart), and heads or tokens one element apart: torch lays a
    tensor like such a one out with another dim innermost."""
    dev = require_gpu()
    g = torch.Generator().manual_seed(4)
    base = torch.randn(20000, generator=g).to(dtype).to(dev)
    inv, _ = rotary_frequencies(64, device=dev)
    for shape, strides in (((1, 2, 37, 64), (0, 128, 1, 1)), ((2, 2, 80, 64), (700, 1, 64, 1)), ((5, 4, 64), (1, 96, 1))):
        q = base.as_strided(shape, strides)
        s = shape[-2] if len(shape) == 4 else shape[0]
        pos = torch.arange(s, device=dev)
        print(f"rotary overlapping {shape} {strides}", flush=True)
        want, _ = apply_rotary(q.contiguous(), None, pos, inv)
        a, b = apply_rotary(q, q, pos, inv)
        assert torch.equal(a, want) and torch.equal(b, want)
    # Packed rows as new tokens of a cache.
    q = base.as_strided((5, 4, 64), (1, 96, 1))
    pools = [torch.zeros((2, 8, 4, 64), dtype=dtype, device=dev) for _ in range(4)]
    table = torch.tensor([[1]], dtype=torch.int32, device=dev)
    kvl, cu = torch.tensor([6], dtype=torch.int32, device=dev), torch.tensor([0, 5], dtype=torch.int32, device=dev)
    got = append_paged(q, q, q, *pools[:2], table, kvl, cu, inv)
    want = append_paged(*(q.contiguous() for _ in range(3)), *pools[2:], table, kvl, cu, inv)
    assert torch.equal(got, want) and torch.equal(pools[0], pools[2]) and torch.equal(pools[1], pools[3])


def test_forward_mode_of_frequencies():
    """The rotation has no derivative for its frequencies: a tangent of theirs is refused, not dropped."""
    dev = require_gpu()
    inv, _ = rotary_frequencies(32, device=dev)
    q, t = (torch.randn(2, 3, 9, 32, device=dev).bfloat16() for _ in range(2))
    pos = torch.arange(9, device=dev)
    print("rotary forward mode of frequencies", flush=True)
    for x in (q, None):
        with fwAD.dual_level():
            dual = fwAD.make_dual(inv, torch.ones_like(inv))
            with pytest.raises(KernelError, match="inv_freq"):
                apply_rotary(q if x is None else fwAD.make_dual(x, t), None, pos, dual)
