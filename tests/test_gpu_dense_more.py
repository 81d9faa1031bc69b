"""Dense attention, continued: what autograd hands back, and the forms that large calls take."""
from __future__ import annotations

import pytest
import torch
from torch.autograd.graph import save_on_cpu, saved_tensors_hooks
from torch.utils.checkpoint import checkpoint

import dense_ref as ref
from helpers import require_gpu
from tasft_amd import _native
from tasft_amd.kernels import dense_attention

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


@pytest.mark.parametrize("return_lse", [False, True])
@pytest.mark.parametrize("packed", [False, True])
def test_saved_tensors_may_come_back_with_other_strides(packed, return_lse):
    """Slices of a fused projection saved in host memory, as dense copies, at odd places, or computed again: the
    gradients of a plain step, bit for bit."""
    dev = require_gpu()
    b, s, hq, hkv, d = 2, 150, 4, 2, 64
    g = torch.Generator().manual_seed(0)
    wide = torch.randn((b, s, hq + 2 * hkv, d), generator=g).to(BF).to(dev)
    go = torch.randn((b, s, hq, d), generator=g).to(BF).to(dev)
    slopes = torch.tensor([0.5, 0.25, 0.125, 0.0625], device=dev)
    cu = torch.tensor([0, 100, 290], dtype=torch.int32, device=dev)
    lens = torch.tensor([150, 77], dtype=torch.int32, device=dev)

    def attend(q, k, v):
        if packed:
            return dense_attention(q, k, v, cu_seqlens=cu, max_seqlen=190, alibi_slopes=slopes, return_lse=return_lse)
        return dense_attention(q, k, v, seq_lens=lens, alibi_slopes=slopes, return_lse=return_lse)

    def run(within, call=attend):
        leaf = wide.clone().requires_grad_(True)
        parts = leaf.flatten(0, 1).split((hq, hkv, hkv), 1) if packed else \
            [x.transpose(1, 2) for x in leaf.split((hq, hkv, hkv), 2)]
        with within:
            got = call(*parts)
        out, lse = got if return_lse else (got, None)
        grad = go.flatten(0, 1) if packed else go.transpose(1, 2)
        loss = (out * grad).float().sum()
        if return_lse:
            loss = loss + lse[lse > -1e30].sin().sum()
        return torch.autograd.grad(loss, leaf)[0]

    def odd(t):
        room = torch.empty(t.numel() * t.element_size() + 16, dtype=torch.uint8, device=t.device)
        return room[t.element_size():t.element_size() * (t.numel() + 1)].view(t.dtype).view(t.shape).copy_(t)

    print(f"dense hooks packed={packed} lse={return_lse}", flush=True)
    want = run(saved_tensors_hooks(lambda t: t, lambda t: t))
    for name, hooks in (("host", save_on_cpu()), ("pinned", save_on_cpu(pin_memory=True)),
                        ("dense", saved_tensors_hooks(lambda t: t.contiguous().clone(), lambda t: t)),
                        ("odd", saved_tensors_hooks(lambda t: t, odd))):
        assert torch.equal(run(hooks), want), name
    again = run(saved_tensors_hooks(lambda t: t, lambda t: t), lambda *x: checkpoint(attend, *x, use_reentrant=False))
    assert torch.equal(again, want)


def slopes_of(hq):
    return torch.tensor([2.0 ** (-8.0 * (i + 1) / hq) for i in range(hq)])


def parts_of_ds(rows, hq):
    """Sequences of at most so many tokens take dS in two parts."""
    return max(32, (1 << 24) // (rows * hq))


def head_shares(rows, hkv, group, most):
    """How many workgroups share a KV head's query heads."""
    groups = -(-rows // 128) * hkv
    want = -(-(2048 if most >= 6144 else 1024) // groups)
    return group if 2 * want > group and want > 1 else want


# lens of two kinds of sequences, copies of each, Hq, Hkv, D, dtype, causal, softcap, alibi, prefix lengths, max_seqlen
# (0: the longest), shares of a KV head's query heads
LARGE = [
    ([133, 197], 52, 28, 4, 128, BF, True, 50.0, False, None, 0, 2),        # 3 and 4 heads
    ([133, 197], 36, 28, 4, 128, HF, True, 0, True, [70, 0], 0, 3),         # 2, 2 and 3
    ([150, 77], 76, 28, 4, 64, HF, True, 20.0, True, None, 0, 2),
    ([161, 90], 44, 32, 8, 64, BF, True, 0, False, [100, 90], 0, 2),        # 2 and 2
    ([130, 200], 36, 28, 4, 128, BF, False, 30.0, True, None, 0, 3),
    ([133, 97], 108, 28, 4, 64, BF, True, 200.0, False, None, 7000, 3),     # a length that documents may have
    ([129, 190], 52, 32, 8, 128, HF, True, 0, False, [0, 190], 0, 1),       # whole groups
    ([191, 65], 70, 32, 8, 128, BF, True, 0, True, None, 0, 1),
    ([200, 131], 50, 32, 8, 64, HF, False, 0, False, None, 0, 1),
    ([99, 161], 60, 32, 8, 128, HF, True, 25.0, True, [99, 30], 0, 2),
    ([127, 193], 12, 56, 4, 64, BF, True, 0, False, None, 0, 14),           # single heads
]


@pytest.mark.parametrize(("index", "batched"), [(i, b) for i, c in enumerate(LARGE) for b in (False, True)
                                                if not (b and c[10])])  # (max_seqlen goes with documents)
def test_large_calls(index, batched):
    """dS in one part, and heads shared out unevenly or not at all, as calls of many tokens take them: two kinds of
    sequences, mixed, each copy bit for bit, and a copy of each within the bounds of the 64-bit form."""
    lens, copies, hq, hkv, d, dtype, causal, cap, alibi, prefix, most, shares = LARGE[index]
    dev = require_gpu()
    longest = max(lens) + (5 if batched else 0)
    total = 2 * copies * longest if batched else copies * sum(lens)
    # The branches that are meant, by the rules of the kernels' host code.
    assert parts_of_ds(total, hq) < min(lens)
    if not batched:
        assert head_shares(total, hkv, hq // hkv, most or longest) == shares
    kinds = ref.inputs(lens, hq, hkv, d, dtype, seed=60 + index)
    slopes = slopes_of(hq) if alibi else None
    want = [ref.reference(*r[:4], None if batched else r[4], causal=causal, scale=d ** -0.5, cap=cap, slopes=slopes,
                          prefix=prefix[i] if prefix else 0, dtype=dtype) for i, r in enumerate(kinds)]
    g = torch.Generator().manual_seed(index)
    order = torch.tensor([0, 1] * copies)[torch.randperm(2 * copies, generator=g)].tolist()
    on = [[x.to(dev) for x in r] for r in kinds]
    if batched:
        wide = [torch.stack(tuple(x)).to(dev) for x in zip(*[[ref.batched([y], longest)[0] for y in r[:4]] for r in kinds])]
        q, k, v, go = (x[torch.tensor(order, device=dev)].transpose(1, 2) for x in wide)
        kw = {"seq_lens": torch.tensor([lens[i] for i in order], device=dev)}
    else:
        q, k, v, go, gl = (torch.cat([on[i][j] for i in order]) for j in range(5))
        offs = torch.tensor([0] + [lens[i] for i in order]).cumsum(0).tolist()
        kw = {"cu_seqlens": torch.tensor(offs, dtype=torch.int32, device=dev), "max_seqlen": most or longest}
    q, k, v = (x.requires_grad_(True) for x in (q, k, v))
    if prefix:
        kw["prefix_lens"] = torch.tensor([prefix[i] for i in order], device=dev)
    print(f"dense large {LARGE[index]} batched={batched}", flush=True)
    out, lse = dense_attention(q, k, v, causal=causal, softcap=cap or None, return_lse=True,
                               alibi_slopes=None if slopes is None else slopes.to(dev), **kw)
    grads = torch.autograd.grad(out, (q, k, v), go) if batched else torch.autograd.grad((out, lse), (q, k, v), (go, gl))
    torch.cuda.synchronize()
    for name, x in zip(("out", "lse", "gq", "gk", "gv"), (out, lse, *grads)):
        x = x.detach()
        if batched:
            rows = [x[j].transpose(0, 1)[:lens[i]] for j, i in enumerate(order)]
            if name != "lse":
                assert not any(x[j, :, lens[i]:].any() for j, i in enumerate(order)), name
        else:
            rows = [x[offs[j]:offs[j + 1]] for j in range(len(order))]
        for kind in range(2):
            one = rows[order.index(kind)]
            assert all(torch.equal(r, one) for r, i in zip(rows, order) if i == kind), f"{name}: copies differ"
            err, bound = (one.cpu().double() - want[kind][name]).abs(), want[kind]["e_" + name]
            assert bool((err <= bound).all()), f"{name} of kind {kind}: {float((err / bound).max()):.2f} of its bound"


@pytest.mark.parametrize("d", [64, 128])
def test_an_output_gradient_of_infinity_in_fp16(d):
    """An infinity of a row's output gradient reaches dv of the keys that it sees: -inf where no weight of theirs
    rounds to 0."""
    dev = require_gpu()
    n, hq, hkv, at = 200, 4, 2, 120
    q, k, v, go, _ = ref.inputs([n], hq, hkv, d, HF, seed=9)[0]
    go[at, :, 7] = -float("inf")
    weights = torch.stack([torch.exp(ref.scores(q[:, h].double(), k[:, h // 2].double(), d ** -0.5, 0, 0))[at, :at + 1]
                           for h in range(hq)])
    weights = weights / weights.sum(1, keepdim=True)
    assert float(weights.min()) > 2.0 ** -20  # far above the 2^-25 that rounds to 0
    q, k, v = (x.to(dev).requires_grad_(True) for x in (q, k, v))
    print(f"dense infinite gradient {d}", flush=True)
    for cap in (None, 30.0):
        out = dense_attention(q, k, v, cu_seqlens=torch.tensor([0, n]), softcap=cap)
        gv = torch.autograd.grad(out, v, go.to(dev))[0].cpu()
        assert bool((gv[:at + 1, :, 7] == -float("inf")).all()) and bool(torch.isfinite(gv[at + 1:]).all())
        assert bool(torch.isfinite(gv[:, :, [x for x in range(d) if x != 7]]).all())


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_backward_without_what_the_rounding_left_over(d, dtype):
    """The C entry with out_rest NULL: D_i from the output as it was rounded, whose bound has that error in it."""
    dev = require_gpu()
    n, hq, hkv = 150, 4, 2
    kind = ref.inputs([n], hq, hkv, d, dtype, seed=d)[0]
    want = ref.reference(*kind, causal=True, scale=d ** -0.5, cap=20.0, slopes=None, prefix=0, dtype=dtype)
    q, k, v, go, gl = (x.to(dev) for x in kind)
    out, lse = dense_attention(q, k, v, cu_seqlens=torch.tensor([0, n]), softcap=20.0, return_lse=True)
    grads = [torch.full_like(x, float("nan")) for x in (q, k, v)]
    lib = _native.load_library()
    size = lib.tasft_dense_bwd_workspace_bytes(1, n, hq, hkv, n, d)
    room = torch.empty(size, dtype=torch.uint8, device=dev)
    cu = torch.tensor([0, n], dtype=torch.int32, device=dev)
    four = lambda x: _native.kept_strides((0, x.stride(1), x.stride(0), 1))  # noqa: E731
    three = lambda x: _native.kept_strides((0, x.stride(1), x.stride(0)))  # noqa: E731
    print(f"dense without rest {d} {dtype}", flush=True)
    status = lib.tasft_dense_bwd(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(), None, go.data_ptr(), gl.data_ptr(),
        *(x.data_ptr() for x in grads), room.data_ptr(), size, cu.data_ptr(), None, None, None, 1, n, hq, hkv, n, d,
        four(q), four(k), four(v), four(out), three(lse), four(go), three(gl), *(four(x) for x in grads), d ** -0.5, 20.0, 1,
        0 if dtype == BF else 1, _native.stream_handle(dev))
    _native.check(status, "tasft_dense_bwd")
    for name, x in zip(("gq", "gk", "gv"), grads):
        err, bound = (x.cpu().double() - want[name]).abs(), want["e_" + name]
        assert bool((err <= bound).all()), f"{name}: {float((err / bound).max()):.2f} of its bound"
