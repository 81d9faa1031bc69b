"""Dense attention with capped and biased scores, documents and prefixes, and its gradients, against the
64-bit form."""
from __future__ import annotations

import math

import pytest
import torch

import dense_ref as ref
from helpers import require_gpu
from tasft_amd.kernels import apply_rotary, dense_attention, rotary_frequencies

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16

# lens, Hq, Hkv, D, dtype, causal, softcap, alibi, prefix lengths (or None)
CASES = [
    ([1], 1, 1, 128, BF, True, 0, False, None),
    ([1, 2], 4, 4, 64, HF, True, 30.0, True, [1, 0]),
    ([33], 4, 2, 128, BF, True, 0, False, None),
    ([64, 65, 63], 4, 1, 64, HF, True, 0, True, None),
    ([127, 128, 129], 8, 2, 128, BF, True, 50.0, False, None),
    ([200, 0, 31, 1], 6, 2, 128, HF, True, 20.0, True, [70, 0, 31, 1]),
    ([257, 100], 7, 1, 128, BF, True, 0, False, [130, 100]),
    ([300], 3, 3, 64, BF, True, 5.0, False, [299]),
    ([150, 77], 4, 4, 64, HF, False, 0, True, None),
    ([140, 260], 4, 2, 128, BF, False, 15.0, False, None),
    ([513], 2, 1, 128, HF, True, 1000.0, True, None),
    ([390], 2, 2, 128, BF, True, 0, True, [0]),
]


def slopes_of(hq):
    return torch.tensor([2.0 ** (-8.0 * (i + 1) / hq) for i in range(hq)])


def want_of(case, rows, scale=None, use_glse=True):
    lens, hq, _, d, dtype, causal, cap, alibi, prefix = case
    return [ref.reference(*r[:4], r[4] if use_glse else None, causal=causal, scale=scale or 1 / math.sqrt(d), cap=cap,
                          slopes=slopes_of(hq) if alibi else None, prefix=prefix[i] if prefix else 0, dtype=dtype)
            for i, r in enumerate(rows)]


def options(case, dev):
    _, hq, _, _, _, causal, cap, alibi, prefix = case
    return {"causal": causal, "softcap": cap or None, "alibi_slopes": slopes_of(hq).to(dev) if alibi else None,
            "prefix_lens": None if prefix is None else torch.tensor(prefix, dtype=torch.int32, device=dev)}


def check(got, want, bound, what):
    err = (got.detach().cpu().double() - want).abs()
    assert bool(torch.isfinite(got).all()), f"{what}: not finite"
    assert bool((err <= bound).all()), f"{what}: {float((err - bound).max()):.3e} over the bound, {float((err / bound).max()):.2f} of it"


def check_all(out, lse, grads, want, lens, take):
    """``take(x, n)``: rows of sequence n, [len, H, ...]."""
    for n in range(len(lens)):
        if lens[n] == 0:
            continue
        w = want[n]
        check(take(out, n), w["out"], w["e_out"], f"out of {n}")
        check(take(lse, n), w["lse"], w["e_lse"], f"lse of {n}")
        for name, g in zip(("gq", "gk", "gv"), grads):
            check(take(g, n), w[name], w["e_" + name], f"{name} of {n}")


@pytest.mark.parametrize("index", range(len(CASES)))
def test_packed(index):
    case = CASES[index]
    lens, hq, hkv, d, dtype = case[:5]
    dev = require_gpu()
    rows = ref.inputs(lens, hq, hkv, d, dtype, seed=index)
    want = want_of(case, rows)
    pad = 5
    q, k, v, go, gl = (ref.packed((r[i] for r in rows), pad).to(dev) for i in range(5))
    for x in (q, k, v):
        x.requires_grad_(True)
    offs = torch.tensor([0] + lens).cumsum(0).to(torch.int32)
    print(f"dense packed {case}", flush=True)
    out, lse = dense_attention(q, k, v, cu_seqlens=offs.to(dev), max_seqlen=max(lens), return_lse=True,
                               **options(case, dev))
    grads = torch.autograd.grad((out, lse), (q, k, v), (go, gl))
    torch.cuda.synchronize()
    check_all(out, lse, grads, want, lens, lambda x, n: x[offs[n]:offs[n + 1]])
    for x in (out, *grads):
        assert not x[-pad:].any() and x.shape[0] == sum(lens) + pad
    assert bool((lse[-pad:] == -math.inf).all())
    # The same from host offsets and without gradients, and again: equal bits.
    with torch.no_grad():
        alone = dense_attention(q, k, v, cu_seqlens=offs, **options(case, dev))
    assert torch.equal(alone, out)
    out2, lse2 = dense_attention(q, k, v, cu_seqlens=offs.to(dev), max_seqlen=max(lens) + 300, return_lse=True,
                                 **options(case, dev))
    again = torch.autograd.grad((out2, lse2), (q, k, v), (go, gl))
    assert all(torch.equal(a, b) for a, b in zip((out, lse, *grads), (out2, lse2, *again)))


@pytest.mark.parametrize("index", range(len(CASES)))
def test_batched(index):
    """A padded batch whose padding holds NaN, as transposed views of [B, S, H, D]."""
    case = CASES[index]
    lens, hq, hkv, d, dtype = case[:5]
    dev = require_gpu()
    rows = ref.inputs(lens, hq, hkv, d, dtype, seed=30 + index)
    want = want_of(case, rows, use_glse=False)
    longest = max(lens) + 3
    q, k, v, go = (ref.batched((r[i] for r in rows), longest).to(dev).transpose(1, 2) for i in range(4))
    for x in (q, k, v):
        x.requires_grad_(True)
    print(f"dense batched {case}", flush=True)
    out, lse = dense_attention(q, k, v, seq_lens=torch.tensor(lens, dtype=torch.int32, device=dev), return_lse=True,
                               **options(case, dev))
    grads = torch.autograd.grad(out, (q, k, v), go)
    torch.cuda.synchronize()
    assert out.shape == q.shape and lse.shape == q.shape[:3]
    check_all(out, lse, grads, want, lens, lambda x, n: x[n].transpose(0, 1)[:lens[n]])
    for n, m in enumerate(lens):
        for x in (out, *grads):
            assert not x[n, :, m:].any()
        assert bool((lse[n, :, m:] == -math.inf).all())


@pytest.mark.parametrize("hq", [3, 8])
def test_many_heads_of_a_group(hq):
    """A KV head's query heads shared out over workgroups and joined, or (one head) not."""
    dev = require_gpu()
    for hkv, lens in ((1, [300, 40]), (hq, [130])):
        case = (lens, hq, hkv, 64, BF, True, 0, False, None)
        rows = ref.inputs(lens, hq, hkv, 64, BF, seed=hq)
        want = want_of(case, rows)
        q, k, v, go, gl = (ref.packed(r[i] for r in rows).to(dev) for i in range(5))
        for x in (q, k, v):
            x.requires_grad_(True)
        offs = torch.tensor([0] + lens).cumsum(0).to(torch.int32)
        print(f"dense heads {hq}/{hkv}", flush=True)
        out, lse = dense_attention(q, k, v, cu_seqlens=offs, return_lse=True)
        grads = torch.autograd.grad((out, lse), (q, k, v), (go, gl))
        check_all(out, lse, grads, want, lens, lambda x, n: x[offs[n]:offs[n + 1]])


def test_enough_workgroups_for_whole_groups():
    """So many KV heads that a workgroup takes all the query heads of one."""
    dev = require_gpu()
    lens, hq, hkv, d = [130] * 130, 16, 8, 64
    g = torch.Generator().manual_seed(0)
    # Eight different sequences, repeated: the same bits for each, and one of each kind checked.
    kinds = ref.inputs([130] * 2, hq, hkv, d, BF, seed=1)
    rows = [kinds[int(torch.randint(2, (1,), generator=g))] for _ in lens]
    case = (lens, hq, hkv, d, BF, True, 0, False, None)
    want = want_of((lens[:2], *case[1:]), kinds)
    q, k, v, go, gl = (ref.packed(r[i] for r in rows).to(dev) for i in range(5))
    for x in (q, k, v):
        x.requires_grad_(True)
    offs = torch.tensor([0] + lens).cumsum(0).to(torch.int32)
    print("dense whole groups", flush=True)
    out, lse = dense_attention(q, k, v, cu_seqlens=offs, return_lse=True)
    grads = torch.autograd.grad((out, lse), (q, k, v), (go, gl))
    check_all(out, lse, grads, [want[0] if r is kinds[0] else want[1] for r in rows], lens,
              lambda x, n: x[offs[n]:offs[n + 1]])


@pytest.mark.parametrize("d", [64, 128])
def test_layouts(d):
    """A fused projection's slices, expanded heads and values, rows that need a copy, a gradient that is an
    expanded scalar: as contiguous tensors, bit for bit."""
    dev = require_gpu()
    b, s, hq, hkv = 2, 150, 4, 2
    g = torch.Generator().manual_seed(d)
    wide = torch.randn((b, s, (hq + 2 * hkv), d), generator=g).to(BF).to(dev)

    def run(q, k, v):
        q, k, v = (x.detach().requires_grad_(True) for x in (q, k, v))
        out = dense_attention(q, k, v, softcap=30.0)
        return out, *torch.autograd.grad(out.float().sum(), (q, k, v))

    parts = [x.transpose(1, 2) for x in wide.split((hq, hkv, hkv), 2)]
    print(f"dense layouts {d}", flush=True)
    want = run(*(x.contiguous() for x in parts))
    assert all(torch.equal(x, y) for x, y in zip(run(*parts), want))
    odd = [torch.empty(x.numel() + 1, dtype=BF, device=dev)[1:].view(x.shape).copy_(x) for x in parts]
    assert all(torch.equal(x, y) for x, y in zip(run(*odd), want))
    strided = [torch.empty((*x.shape[:-1], 2 * d), dtype=BF, device=dev)[..., ::2].copy_(x) for x in parts]
    assert all(torch.equal(x, y) for x, y in zip(run(*strided), want))
    one = parts[1][:, :1]
    want = run(parts[0], one.expand(-1, 2, -1, -1).contiguous(), one.expand(-1, 2, -1, -1).contiguous())
    assert all(torch.equal(x, y) for x, y in zip(run(parts[0], one.expand(-1, 2, -1, -1), one.expand(-1, 2, -1, -1)), want))
    row = parts[1][:, :, :1]  # one key and value repeated along the sequence
    whole = [row.expand(-1, -1, s, -1)] * 2
    assert all(torch.equal(x, y) for x, y in zip(run(parts[0], *whole), run(parts[0], *(x.contiguous() for x in whole))))


@pytest.mark.parametrize("cap", [0, 20.0])
def test_large_scores(cap):
    """Scores whose running maximum moves far, some weights 0."""
    dev = require_gpu()
    case = ([250], 4, 2, 128, BF, True, cap, False, None)
    rows = ref.inputs([250], 4, 2, 128, BF, seed=4, scale=3.0)
    rows[0][1] = (rows[0][1].float() * torch.linspace(0.1, 3.0, 250)[:, None, None]).to(BF)
    want = want_of(case, rows)
    q, k, v, go, gl = (x.to(dev) for x in rows[0])
    for x in (q, k, v):
        x.requires_grad_(True)
    print(f"dense large scores {cap}", flush=True)
    out, lse = dense_attention(q, k, v, cu_seqlens=torch.tensor([0, 250]), return_lse=True, softcap=cap or None)
    grads = torch.autograd.grad((out, lse), (q, k, v), (go, gl))
    check_all(out, lse, grads, want, [250], lambda x, n: x)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("cap", [0, 30.0])
@pytest.mark.parametrize("prefix", [0, 70])
def test_what_a_row_does_not_see_does_not_reach_it(cap, prefix, dtype):
    """NaN and infinities of a token change the rows and gradients of the tokens that have to do with it,
    and no others."""
    dev = require_gpu()
    n, hq, hkv, d = 200, 4, 2, 128
    rows = ref.inputs([n], hq, hkv, d, dtype, seed=9)[0]
    cu = torch.tensor([0, n])
    pre = torch.tensor([prefix], dtype=torch.int32)

    def run(q, k, v, go):
        q, k, v = (x.to(dev).requires_grad_(True) for x in (q, k, v))
        out = dense_attention(q, k, v, cu_seqlens=cu, prefix_lens=pre, softcap=cap or None)
        return [x.detach().cpu() for x in (out, *torch.autograd.grad(out, (q, k, v), go.to(dev)))]

    print(f"dense unseen values cap={cap} prefix={prefix} {dtype}", flush=True)
    clean = run(*rows[:4])
    at, bad = 120, (3, float("inf"))
    see = ref.seen(n, True, prefix)
    # A value: rows that see it get the infinity in that dim (and its gradients NaN); others nothing.
    v = rows[2].clone()
    v[at, :, bad[0]] = bad[1]
    out, gq, gk, gv = run(rows[0], rows[1], v, rows[3])
    sees, not_seen = see[:, at], ~see[:, at]
    assert torch.equal(out[not_seen], clean[0][not_seen]) and torch.equal(gq[not_seen], clean[1][not_seen])
    assert bool((out[sees][:, :, bad[0]] == math.inf).all())
    rest = [x for x in range(d) if x != bad[0]]
    assert torch.equal(out[:, :, rest], clean[0][:, :, rest])
    assert bool(torch.isnan(gq[sees]).any(-1).all())
    # dv_j does not read v (only out's own rows do).
    assert torch.equal(gv, clean[3])
    # A key: its row of scores is NaN or infinite for those that see it.
    k = rows[1].clone()
    k[at, :, 5] = float("nan")
    out, gq, gk, gv = run(rows[0], k, rows[2], rows[3])
    assert torch.equal(out[not_seen], clean[0][not_seen]) and torch.equal(gq[not_seen], clean[1][not_seen])
    assert bool(torch.isnan(out[sees]).all()) and bool(torch.isnan(gq[sees]).all())
    # A row's output gradient and its query: the keys that it sees, and no others.
    unseen_by = ~see[at]
    assert unseen_by.any()
    go = rows[3].clone()
    go[at, :, 7] = -float("inf")
    out, gq, gk, gv = run(rows[0], rows[1], rows[2], go)
    assert torch.equal(out, clean[0])
    others = torch.arange(n) != at
    assert torch.equal(gq[others], clean[1][others])
    assert torch.equal(gk[unseen_by], clean[2][unseen_by]) and torch.equal(gv[unseen_by], clean[3][unseen_by])
    assert bool((gv[see[at]][:, :, 7] == -math.inf).all()) or dtype == HF
    rest = [x for x in range(d) if x != 7]
    assert torch.equal(gv[:, :, rest], clean[3][:, :, rest])
    q = rows[0].clone()
    q[at, :, 9] = float("nan")
    out, gq, gk, gv = run(q, rows[1], rows[2], rows[3])
    assert torch.equal(out[others], clean[0][others]) and torch.equal(gq[others], clean[1][others])
    assert bool(torch.isnan(out[at]).all()) and bool(torch.isnan(gq[at]).all())
    assert torch.equal(gk[unseen_by], clean[2][unseen_by]) and torch.equal(gv[unseen_by], clean[3][unseen_by])
    assert bool(torch.isnan(gk[see[at]]).all()) and bool(torch.isnan(gv[see[at]]).all())


@pytest.mark.parametrize(("d", "dtype", "cap"), [(64, HF, 0), (128, BF, 0), (128, HF, 25.0), (64, BF, 25.0)])
def test_slopes_that_favour_distance(d, dtype, cap):
    """Negative slopes, whose bias alone is far above every score, at lengths that end inside a tile."""
    dev = require_gpu()
    lens, hq, hkv = [37, 211, 1], 4, 2
    slopes = torch.tensor([-1.0, -0.25, 0.5, -0.0625])
    rows = ref.inputs(lens, hq, hkv, d, dtype, seed=d)
    want = [ref.reference(*r, causal=True, scale=1 / math.sqrt(d), cap=cap, slopes=slopes, prefix=0, dtype=dtype)
            for r in rows]
    q, k, v, go, gl = (ref.packed(r[i] for r in rows).to(dev) for i in range(5))
    for x in (q, k, v):
        x.requires_grad_(True)
    offs = torch.tensor([0] + lens).cumsum(0).to(torch.int32)
    print(f"dense negative slopes {d} {dtype} {cap}", flush=True)
    out, lse = dense_attention(q, k, v, cu_seqlens=offs, return_lse=True, softcap=cap or None,
                               alibi_slopes=slopes.to(dev))
    grads = torch.autograd.grad((out, lse), (q, k, v), (go, gl))
    check_all(out, lse, grads, want, lens, lambda x, n: x[offs[n]:offs[n + 1]])


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_a_key_of_no_weight(d, causal):
    """A key of -inf where every query is positive: its scores are -inf, its weight and gradients 0."""
    dev = require_gpu()
    n, at = 71, 40
    q, k, v, go, _ = ref.inputs([n], 2, 1, d, BF, seed=6)[0]
    q[..., 3] = q[..., 3].abs() + 1.0
    k[at, 0, 3] = -math.inf
    q, k, v = (x.to(dev).requires_grad_(True) for x in (q, k, v))
    print(f"dense key of no weight {d} {causal}", flush=True)
    out = dense_attention(q, k, v, cu_seqlens=torch.tensor([0, n]), causal=causal)
    _, gk, gv = torch.autograd.grad(out, (q, k, v), go.to(dev))
    assert bool(torch.isfinite(out).all()) and bool(torch.isfinite(gk).all()) and bool(torch.isfinite(gv).all())
    assert not gk[at].any() and not gv[at].any() and bool(gv[at - 1].any())


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("less", [14.5, 16.0, 17.5])
def test_many_small_weights(less, dtype):
    """One key far above 4000 others, whose weights (2^-less of its own) fp16 holds with few bits."""
    dev = require_gpu()
    n, d = 4001, 64
    q = torch.zeros((n, 1, d), dtype=dtype)
    q[..., 0] = 8.0
    k = torch.zeros((n, 1, d), dtype=dtype)
    k[0, 0, 0] = less * math.log(2.0)
    v = torch.ones((n, 1, d), dtype=dtype)
    v[0] = 0.0
    print(f"dense small weights {less} {dtype}", flush=True)
    out = dense_attention(*(x.to(dev) for x in (q, k, v)), cu_seqlens=torch.tensor([0, n]), causal=False)
    small = math.exp(-float(k[0, 0, 0]))
    want = 4000 * small / (1 + 4000 * small)
    # P's rounding (fp16 below 2^-14: 2^-25 of a weight of 1), in the sum and in the divisor, and out's own.
    u = ref.half_step(dtype)
    bound = 3 * u * want + (2 * 4000 * 2.0 ** -25 if dtype == HF else 0.0) + 2.0 ** -12 * want
    assert float((out.cpu().double() - want).abs().max()) <= bound


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("lens", [[2, 3, 2, 3], [5, 8, 11, 4], [60, 90], [400]])
def test_few_rows_lose_little_to_the_rounding_of_ds(lens, dtype):
    """The errors of dq and dk together against those of rounding the exact result alone: a second rounding of
    the same relative size, of dS, would make it the square root of 2 in the mean, and by chance more."""
    dev = require_gpu()
    hq, hkv, d = 8, 2, 128
    rows = ref.inputs(lens, hq, hkv, d, dtype, seed=sum(lens))
    want = want_of((lens, hq, hkv, d, dtype, True, 0, False, None), rows, use_glse=False)
    q, k, v, go = (ref.packed(r[i] for r in rows).to(dev) for i in range(4))
    for x in (q, k, v):
        x.requires_grad_(True)
    print(f"dense few rows {lens} {dtype}", flush=True)
    out = dense_attention(q, k, v, cu_seqlens=torch.tensor([0] + lens).cumsum(0))
    for name, got in zip(("gq", "gk"), torch.autograd.grad(out, (q, k), go)):
        exact = torch.cat([w[name] for w in want])
        least = (exact.to(dtype).double() - exact).norm()
        assert float((got.cpu().double() - exact).norm() / least) < math.sqrt(2), name


def test_max_seqlen_cuts():
    """Tokens behind a document's first max_seqlen are not there: their rows and gradients are 0."""
    dev = require_gpu()
    lens, cut, hq, hkv, d = [150, 20, 90], 70, 4, 2, 64
    case = ([min(x, cut) for x in lens], hq, hkv, d, BF, True, 0, False, None)
    rows = ref.inputs(lens, hq, hkv, d, BF, seed=3)
    want = want_of(case, [[x[:cut] for x in r] for r in rows])
    q, k, v, go, gl = (ref.packed(r[i] for r in rows).to(dev) for i in range(5))
    for x in (q, k, v):
        x.requires_grad_(True)
    offs = torch.tensor([0] + lens).cumsum(0).to(torch.int32)
    print("dense cut", flush=True)
    out, lse = dense_attention(q, k, v, cu_seqlens=offs.to(dev), max_seqlen=cut, return_lse=True)
    grads = torch.autograd.grad((out, lse), (q, k, v), (go, gl))
    check_all(out, lse, grads, want, lens, lambda x, n: x[offs[n]:offs[n] + min(lens[n], cut)])
    for n, m in enumerate(lens):
        for x in (out, *grads):
            assert not x[offs[n] + min(m, cut):offs[n + 1]].any()


def test_lengths_on_the_device_are_clamped():
    """Offsets, lengths and prefixes past what is there."""
    dev = require_gpu()
    q, k, v = (torch.randn((2, h, 100, 64), device=dev).to(BF) for h in (4, 2, 2))
    print("dense clamped", flush=True)
    whole = dense_attention(q, k, v)
    assert torch.equal(dense_attention(q, k, v, seq_lens=torch.tensor([1000, 100], device=dev)), whole)
    none = dense_attention(q, k, v, seq_lens=torch.tensor([-5, 0], device=dev))
    assert not none.any()
    both = dense_attention(q, k, v, causal=False)
    assert torch.equal(dense_attention(q, k, v, prefix_lens=torch.tensor([100, 5000], device=dev)), both)
    assert torch.equal(dense_attention(q, k, v, prefix_lens=torch.tensor([-3, 0], device=dev)), whole)
    flat = [x.transpose(1, 2).flatten(0, 1) for x in (q, k, v)]
    out = dense_attention(*flat, cu_seqlens=torch.tensor([0, 100, 5000], device=dev), max_seqlen=100)
    assert torch.equal(out, whole.transpose(1, 2).flatten(0, 1))


@pytest.mark.parametrize("what", ["none", "out", "lse"])
def test_partial_gradients(what):
    """Gradients of one result, of some of the inputs."""
    dev = require_gpu()
    q, k, v = (torch.randn((1, h, 70, 64), device=dev).to(BF).requires_grad_(True) for h in (4, 2, 2))
    w, wl = torch.randn((1, 4, 70, 64), device=dev).to(BF), torch.randn((1, 4, 70), device=dev)
    print(f"dense partial {what}", flush=True)
    out, lse = dense_attention(q, k, v, return_lse=True)
    if what == "none":
        with torch.no_grad():
            assert not dense_attention(q, k, v).requires_grad
        part = dense_attention(q, k.detach(), v)
        gq, gv = torch.autograd.grad(part, (q, v), w)
        fq, fk, fv = torch.autograd.grad(out, (q, k, v), w)
        assert torch.equal(gq, fq) and torch.equal(gv, fv)
        return
    got = torch.autograd.grad(out if what == "out" else lse, (q, k, v), w if what == "out" else wl)
    zero = torch.autograd.grad(dense_attention(q, k, v, return_lse=True), (q, k, v),
                               (w if what == "out" else torch.zeros_like(w), wl if what == "lse" else torch.zeros_like(wl)))
    assert all(torch.equal(a, b) for a, b in zip(got, zero))
    if what == "lse":
        assert not got[2].any()


def test_second_derivatives_are_refused():
    dev = require_gpu()
    q, k, v = (torch.randn((1, 2, 40, 64), device=dev).to(BF).requires_grad_(True) for _ in range(3))
    g = torch.autograd.grad(dense_attention(q, k, v).float().square().sum(), q, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.float().sum().backward()


@pytest.mark.parametrize("shape", [(0, 4, 10, 64), (2, 4, 0, 64)])
def test_empty(shape):
    dev = require_gpu()
    q = torch.zeros(shape, dtype=BF, device=dev, requires_grad=True)
    k = torch.zeros((shape[0], 2, *shape[2:]), dtype=BF, device=dev)
    out, lse = dense_attention(q, k, k, return_lse=True)
    assert out.shape == shape and lse.shape == shape[:3]
    assert torch.autograd.grad(out.float().sum(), q)[0].shape == shape


def test_graph_and_streams():
    """Forward and backward captured into a graph, replayed with other inputs and eager work between, and
    two streams at once: as eager calls."""
    dev = require_gpu()
    hq, hkv, d, n = 8, 2, 64, 330
    cu = torch.tensor([0, 130, n], dtype=torch.int32, device=dev)
    slopes = slopes_of(hq).to(dev)

    def fill(seed):
        g = torch.Generator(device=dev).manual_seed(seed)
        return [torch.randn((n, h, d), generator=g, device=dev).to(BF) for h in (hq, hkv, hkv, hq)]

    def run(q, k, v, go):
        q, k, v = (x.detach().requires_grad_(True) for x in (q, k, v))
        out = dense_attention(q, k, v, cu_seqlens=cu, max_seqlen=250, alibi_slopes=slopes, softcap=40.0)
        return [out.detach(), *torch.autograd.grad(out, (q, k, v), go)]

    held = fill(0)
    print("dense graph", flush=True)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        run(*held)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(*held)
    for seed in (1, 2, 3):
        fresh = fill(seed)
        for a, b in zip(held, fresh):
            a.copy_(b)
        graph.replay()
        want = run(*fresh)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), seed
    first, second = fill(5), fill(6)
    want = [run(*first), run(*second)]
    torch.cuda.synchronize()
    both = [None, None]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for i, x in enumerate((first, second)):
            with torch.cuda.stream(streams[i]):
                both[i] = run(*x)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for w, g in zip(want, both) for a, b in zip(w, g))


def test_offsets_past_32_bits():
    """Batch entries 6 GB apart: the same bits as close ones."""
    dev = require_gpu()
    s, hq, d = 150, 2, 64
    g = torch.Generator(device=dev).manual_seed(0)
    close = [torch.randn((2, s, hq, d), generator=g, device=dev).to(BF).transpose(1, 2) for _ in range(4)]
    far = []
    for x in close:
        room = torch.empty((2, 3 << 30), dtype=torch.uint8, device=dev).view(BF)
        y = room[:, :s * hq * d].view(2, s, hq, d).transpose(1, 2)
        far.append(y.copy_(x))

    def run(q, k, v, go):
        q, k, v = (x.detach().requires_grad_(True) for x in (q, k, v))
        out = dense_attention(q, k, v)
        return out.detach(), *torch.autograd.grad(out, (q, k, v), go)

    print("dense far entries", flush=True)
    assert all(torch.equal(a, b) for a, b in zip(run(*close), run(*far)))


@pytest.mark.parametrize("d", [64, 128])
def test_tokens_far_apart(d):
    """Tokens as far apart as the kernels take them (16 MB, less a little): the same bits as close ones."""
    dev = require_gpu()
    s, stride = 130, (1 << 23) - 8
    g = torch.Generator(device=dev).manual_seed(0)
    close = [torch.randn((1, 1, s, d), generator=g, device=dev).to(BF) for _ in range(4)]
    room = torch.empty(s * stride, dtype=BF, device=dev)  # the four side by side
    far = [room.as_strided((1, 1, s, d), (0, 0, stride, 1), i * d).copy_(x) for i, x in enumerate(close)]

    def run(q, k, v, go):
        q, k, v = (x.detach().requires_grad_(True) for x in (q, k, v))
        out = dense_attention(q, k, v)
        return [x.contiguous() for x in (out.detach(), *torch.autograd.grad(out, (q, k, v), go))]

    print(f"dense far tokens {d}", flush=True)
    assert all(torch.equal(a, b) for a, b in zip(run(*close), run(*far)))


def test_a_training_step_with_rotary():
    """Projections, rotation, capped attention and their gradients together, against the same step in
    64 bits."""
    dev = require_gpu()
    b, s, hq, hkv, d = 2, 96, 4, 2, 64
    g = torch.Generator().manual_seed(2)
    x = torch.randn((b, s, hq * d), generator=g)
    w = [torch.randn((hq * d, h * d), generator=g) / math.sqrt(hq * d) for h in (hq, hkv, hkv)]
    inv, factor = rotary_frequencies(d)
    pos = torch.arange(s)

    def step(x, w, rotate, attend):
        q, k, v = ((x @ m).unflatten(-1, (h, d)).transpose(1, 2) for m, h in zip(w, (hq, hkv, hkv)))
        q, k = rotate(q, k)
        return attend(q, k, v).transpose(1, 2).flatten(2)

    def rotate64(q, k):
        angle = pos.double()[:, None] * inv
        c, n = angle.cos(), angle.sin()
        return [torch.cat((t[..., :d // 2] * c - t[..., d // 2:] * n, t[..., d // 2:] * c + t[..., :d // 2] * n), -1)
                for t in (q, k)]

    def attend64(q, k, v):
        k, v = (t.repeat_interleave(hq // hkv, 1) for t in (k, v))
        s_ = 20.0 * torch.tanh(q @ k.transpose(2, 3) / math.sqrt(d) / 20.0)
        return torch.softmax(s_.masked_fill(~ref.seen(s, True, 0), -math.inf), -1) @ v

    x16, w16 = x.to(BF), [m.to(BF) for m in w]
    w64 = [m.double().requires_grad_(True) for m in w16]
    want = step(x16.double(), w64, rotate64, attend64)
    want_g = torch.autograd.grad(want.square().mean(), w64)
    wd = [m.to(dev).requires_grad_(True) for m in w16]
    inv = inv.to(dev)
    print("dense training step", flush=True)
    out = step(x16.to(dev), wd, lambda q, k: apply_rotary(q, k, pos.to(dev), inv, scale=factor),
               lambda q, k, v: dense_attention(q, k, v, softcap=20.0))
    got = torch.autograd.grad(out.float().square().mean(), wd)
    # Some ten roundings of 2^-8 at most on every path, which add up like independent ones over the sums.
    u = 2.0 ** -8
    assert float((out.detach().cpu().double() - want.detach()).norm() / want.detach().norm()) < 4 * u
    for a, b_ in zip(got, want_g):
        assert float((a.cpu().double() - b_).norm() / b_.norm()) < 4 * u
