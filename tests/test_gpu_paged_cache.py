"""Writing into and evicting from a paged cache, and a run of the serving calls together."""
from __future__ import annotations

import math

import pytest
import torch

import paged_ref as ref
from helpers import require_gpu
from tasft_amd.kernels import (
    BlockSparseFlashAttention,
    accumulate_key_weights,
    append_paged,
    apply_rotary,
    evict_paged,
    rotary_frequencies,
)

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def _tokens(t, hq, hkv, d, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn((t, h, d), generator=g).to(dtype) for h in (hq, hkv, hkv)]


@pytest.mark.parametrize(("lens", "kv", "hq", "hkv", "d", "r", "page", "dtype", "inter", "given"), [
    ([1], [1], 1, 1, 128, 128, 16, BF, False, False),
    ([1, 1, 1, 1], [17, 1, 64, 65], 28, 4, 128, 128, 16, BF, False, True),
    ([5, 0, 40, 3], [300, 9, 40, 4], 8, 2, 64, 32, 32, HF, True, True),
    ([7, 130], [8, 500], 6, 3, 80, 20, 1, BF, False, False),
    ([70, 9], [65, 9], 4, 4, 96, 24, 8, HF, False, True),       # five tokens before the cache's start
    ([3000, 2000], [3000, 2500], 2, 1, 128, 64, 64, BF, True, False),
    ([1] * 300, list(range(1, 301)), 4, 2, 64, 64, 16, BF, False, True),
])
def test_append(lens, kv, hq, hkv, d, r, page, dtype, inter, given):
    dev = require_gpu()
    pad = 2
    _, kp, vp, table, kvl, cu = ref.make(lens, kv, hq, hkv, d, page, dtype, seed=len(lens))
    kp, vp = kp.nan_to_num(7.0), vp.nan_to_num(7.0, posinf=7.0)
    t = sum(lens) + pad
    q, k, v = _tokens(t, hq, hkv, d, dtype, 5)
    inv, scale = rotary_frequencies(r, 10000.0, {"rope_type": "linear", "factor": 2.0})
    pos = torch.randint(0, 1 << 20, (t,), generator=torch.Generator().manual_seed(9)) if given else None
    cap = table.shape[1] * page
    slots = torch.full((len(lens), hkv, cap), -5, dtype=torch.int32)
    a = [x.to(dev) for x in (q, k, v, kp, vp, table, kvl, cu, inv)]
    slots_d = slots.to(dev)
    print(f"append lens={lens[:5]} kv={kv[:5]} d={d} r={r} page={page}", flush=True)
    out = append_paged(*a, positions=None if pos is None else pos.to(dev), interleaved=inter, scale=1.5,
                       slot_positions=slots_d)
    torch.cuda.synchronize()
    written = torch.zeros(kp.shape[:2], dtype=torch.bool)
    for n in range(len(lens)):
        s0, s1 = int(cu[n]), int(cu[n + 1])
        if s0 == s1:
            continue
        slot = torch.arange(kv[n] - lens[n], kv[n])
        p = slot if pos is None else pos[s0:s1]
        on = slot >= 0
        for got, x in ((out[s0:s1].cpu(), q[s0:s1]),):
            want = ref.rotate(x, p[:, None], inv, 1.5, inter)
            err = (got.double() - want).abs() - ref.rotate_bound(x, want, inv, 1.5, inter, dtype)
            assert bool((err <= 0).all()), float(err.max())
        pg, row = table[n, slot[on] // page].long(), slot[on] % page
        want = ref.rotate(k[s0:s1][on], p[on][:, None], inv, 1.5, inter)
        err = (a[3].cpu()[pg, row].double() - want).abs() - ref.rotate_bound(k[s0:s1][on], want, inv, 1.5, inter, dtype)
        assert bool((err <= 0).all()), float(err.max())
        assert torch.equal(a[4].cpu()[pg, row], v[s0:s1][on])
        written[pg, row] = True
        slots[n, :, slot[on]] = p[on].to(torch.int32)
    assert torch.equal(slots_d.cpu(), slots)
    assert torch.equal(a[3].cpu()[~written], kp[~written]) and torch.equal(a[4].cpu()[~written], vp[~written])
    assert not out[t - pad:].any()


def test_append_skips_pages_outside_the_pool_and_takes_views():
    dev = require_gpu()
    lens, kv = [4, 20], [30, 50]
    _, kp, vp, table, kvl, cu = ref.make(lens, kv, 4, 2, 64, 16, BF, seed=3)
    kp, vp = kp.nan_to_num(1.0), vp.nan_to_num(1.0, posinf=1.0)
    q, k, v = _tokens(24, 4, 2, 64, BF, 1)
    inv, _ = rotary_frequencies(64)
    wild = table.clone()
    wild[0, 1] = -3
    wild[1, 3] = 1 << 29
    print("append wild table", flush=True)
    d = [x.to(dev) for x in (q, k, v, kp, vp, wild, kvl, cu, inv)]
    out = append_paged(*d)
    good = [x.to(dev) for x in (q, k, v, kp, vp, table, kvl, cu, inv)]
    want = append_paged(*good)
    assert torch.equal(out, want)
    assert torch.equal(d[3][wild[1, 2]], good[3][table[1, 2]])
    changed = (d[3].cpu() != kp).any(-1).any(-1).any(-1).nonzero().flatten().tolist()
    assert set(changed) <= {int(x) for x in wild[1, :3]}
    # Fused projections and head-major pools are used in place.
    qkv = torch.cat((good[0], good[1], good[2]), 1)
    hk, hv = (x.to(dev).permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for x in (kp, vp))
    again = append_paged(qkv[:, :4], qkv[:, 4:6], qkv[:, 6:], hk, hv, *good[5:])
    assert torch.equal(again, want) and torch.equal(hk, good[3]) and torch.equal(hv, good[4])


@pytest.mark.parametrize(("kv", "budget", "recent", "sinks", "hkv", "d", "page", "kind"), [
    ([1], 1, 0, 0, 1, 64, 8, "random"),
    ([5, 1, 0], 3, 1, 1, 2, 64, 8, "random"),
    ([100, 17, 64], 16, 4, 2, 2, 128, 16, "random"),
    ([100, 90], 64, 64, 0, 1, 64, 16, "random"),          # recent alone fills the budget
    ([70, 200], 33, 5, 3, 3, 64, 32, "equal"),            # every weight equal: lowest slots
    ([150], 40, 7, 2, 2, 64, 8, "zeros"),
    ([150, 80], 40, 7, 2, 2, 64, 8, "odd"),               # NaN, infinities, negative weights, -0
    ([1500, 2048, 2049], 1000, 100, 4, 2, 64, 16, "random"),
    ([3000, 9000], 512, 50, 4, 1, 64, 64, "few"),         # few distinct weights
    ([33000], 700, 20, 4, 1, 8, 128, "random"),           # more slots than a workgroup holds
    ([40000, 70001, 100, 0], 20000, 300, 4, 2, 8, 128, "random"),
    ([40000, 24576, 16385], 9000, 0, 0, 2, 8, 64, "equal"),
    ([50000, 49152], 30000, 30000, 0, 1, 8, 64, "odd"),
    ([45000, 33000], 12345, 7, 2, 1, 8, 8, "zeros"),
    ([66000], 66000 - 1, 9, 0, 2, 8, 32, "few"),
    ([530000, 9000], 8200, 1000, 4, 1, 8, 128, "few"),    # parts of two runs
    ([500], 1000, 10, 4, 2, 64, 16, "random"),            # within the budget
])
def test_evict(kv, budget, recent, sinks, hkv, d, page, kind):
    dev = require_gpu()
    n = len(kv)
    _, kp, vp, table, kvl, _ = ref.make([0] * n, kv, hkv, hkv, d, page, BF, seed=budget)
    kp, vp = kp.nan_to_num(3.0), vp.nan_to_num(3.0, posinf=3.0)
    cap = table.shape[1] * page
    g = torch.Generator().manual_seed(budget + d)
    scores = torch.rand((n, hkv, cap), generator=g) ** 6
    if kind == "equal":
        scores.fill_(0.25)
    elif kind == "zeros":
        scores.zero_()
        scores[..., ::7] = 1e-30
    elif kind == "odd":
        scores = torch.randn((n, hkv, cap), generator=g)
        scores[..., 3::11] = float("nan")
        scores[..., 4::13] = float("inf")
        scores[..., 5::9] = -float("inf")
        scores[..., 6::10] = 0.0
        scores[..., 1::10] = -0.0
    elif kind == "few":
        scores = (scores * 4).round()
    pos = torch.rand((n, hkv, cap), generator=g).argsort(-1).to(torch.int32)
    want = ref.evict(kp, vp, table, kvl, scores, pos, budget, recent, sinks)
    d_ = [x.to(dev) for x in (kp, vp, table, kvl, scores, pos)]
    print(f"evict kv={kv} budget={budget} {kind}", flush=True)
    lens, s, p = evict_paged(*d_, budget, recent=recent, sinks=sinks)
    torch.cuda.synchronize()
    assert torch.equal(lens.cpu(), want[2]) and torch.equal(p.cpu(), want[4])
    assert torch.equal(s.cpu().view(torch.int32), want[3].view(torch.int32))
    assert torch.equal(d_[0].cpu(), want[0]) and torch.equal(d_[1].cpu(), want[1])
    assert torch.equal(d_[4].cpu().view(torch.int32), scores.view(torch.int32)) and torch.equal(d_[5].cpu(), pos)
    # Once more on the smaller cache: nothing to evict, nothing changes.
    again = evict_paged(d_[0], d_[1], d_[2], lens, s, p, budget, recent=recent, sinks=sinks)
    assert torch.equal(again[0], lens) and torch.equal(again[2], p)
    assert torch.equal(again[1].view(torch.int32), s.view(torch.int32))
    assert torch.equal(d_[0].cpu(), want[0]) and torch.equal(d_[1].cpu(), want[1])


def test_evict_views():
    dev = require_gpu()
    _, kp, vp, table, kvl, _ = ref.make([0, 0], [90, 60], 2, 2, 64, 16, HF, seed=8)
    kp, vp = kp.nan_to_num(1.0).to(dev), vp.nan_to_num(1.0, posinf=1.0).to(dev)
    table, kvl = table.to(dev), kvl.to(dev)
    cap = table.shape[1] * 16
    scores = torch.rand(2, 2, cap, device=dev)
    pos = torch.rand(2, 2, cap, device=dev).argsort(-1).to(torch.int32)
    k1, v1, k2, v2 = kp.clone(), vp.clone(), *(x.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for x in (kp, vp))
    print("evict views", flush=True)
    a = evict_paged(k1, v1, table, kvl, scores, pos, 30, recent=5, sinks=1)
    b = evict_paged(k2, v2, table, kvl.long(), scores.transpose(0, 1).contiguous().transpose(0, 1),
                    torch.stack((pos, pos), -1)[..., 0], 30, recent=5, sinks=1)
    assert all(torch.equal(x, y) for x, y in zip(a, b)) and torch.equal(k1, k2) and torch.equal(v1, v2)


def test_evict_budget_of_more_than_the_table():
    """What is always kept may be more than a small table holds, as long as it fits the budget."""
    dev = require_gpu()
    _, kp, vp, table, kvl, _ = ref.make([0, 0], [90, 60], 2, 2, 64, 16, HF, seed=8)
    kp, vp = kp.nan_to_num(1.0), vp.nan_to_num(1.0, posinf=1.0)
    cap = table.shape[1] * 16
    scores, pos = torch.rand(2, 2, cap), torch.arange(cap, dtype=torch.int32).expand(2, 2, cap).contiguous()
    for budget, recent, sinks in ((cap, cap - 1, 1), (cap + 1, cap, 1), (4096, 2000, 2000), (1 << 40, 1 << 39, 5)):
        print(f"evict budget {budget} of {cap} slots", flush=True)
        d = [x.to(dev) for x in (kp, vp, table, kvl, scores, pos)]
        lens, s, p = evict_paged(*d, budget, recent=recent, sinks=sinks)
        assert torch.equal(lens.cpu(), kvl) and torch.equal(d[0].cpu(), kp) and torch.equal(d[1].cpu(), vp)
        for n in range(2):
            x = int(kvl[n])
            assert torch.equal(s[n, :, :x].cpu(), scores[n, :, :x]) and torch.equal(p[n, :, :x].cpu(), pos[n, :, :x])
            assert not s[n, :, x:].any() and bool((p[n, :, x:] == -1).all())


def test_cache_offsets_past_32_bits():
    """Appending to and evicting from pools whose pages lie 128 MB apart."""
    dev = require_gpu()
    lens, kv, page = [3, 40], [300, 700], 32
    _, kp, vp, table, kvl, cu = ref.make(lens, kv, 4, 2, 128, page, BF, seed=4)
    kp, vp = kp.nan_to_num(2.0).to(dev), vp.nan_to_num(2.0, posinf=2.0).to(dev)
    far = [torch.empty((kp.shape[0], 1 << 26), dtype=BF, device=dev)[:, :kp[0].numel()].view(kp.shape).copy_(x)
           for x in (kp, vp)]
    assert (kp.shape[0] - 1) << 26 > 1 << 31
    cap = table.shape[1] * page
    table, kvl, cu = table.to(dev), kvl.to(dev), cu.to(dev)
    q, k, v = (x.to(dev) for x in _tokens(sum(lens), 4, 2, 128, BF, 1))
    inv = rotary_frequencies(128, device=dev)[0]
    scores = torch.rand((2, 2, cap), device=dev)
    results = []
    print("append and evict, far pages", flush=True)
    for a, b in ((kp, vp), far):
        pos = torch.arange(cap, dtype=torch.int32, device=dev).expand(2, 2, cap).contiguous()
        out = append_paged(q, k, v, a, b, table, kvl, cu, inv, slot_positions=pos)
        results.append((out, *evict_paged(a, b, table, kvl, scores, pos, 200, recent=20, sinks=2), a, b))
    assert all(torch.equal(x, y) for x, y in zip(*results))


@pytest.mark.parametrize(("dtype", "page", "hq", "hkv", "d"), [(BF, 16, 8, 2, 128), (HF, 8, 4, 4, 64)])
def test_serving_steps(dtype, page, hq, hkv, d):
    """Two requests served in chunks and then token by token on a bounded cache: every step's
    append, attention, weights and eviction against the 64-bit forms on the same state."""
    dev = require_gpu()
    n, budget, recent, sinks = 2, 96, 16, 4
    max_pages = 200 // page
    cap = max_pages * page
    table = torch.randperm(n * max_pages, generator=torch.Generator().manual_seed(1)).view(n, max_pages).to(torch.int32)
    kp = torch.zeros((n * max_pages, page, hkv, d), dtype=dtype, device=dev)
    vp = torch.zeros_like(kp)
    inv, scale = rotary_frequencies(d, 10000.0)
    attn = BlockSparseFlashAttention(min_sparsity_for_speedup=0.0)
    kvl = torch.zeros(n, dtype=torch.int32, device=dev)
    seen = torch.zeros(n, dtype=torch.int64)
    scores = torch.zeros((n, hkv, cap), device=dev)
    pos_state = torch.full((n, hkv, cap), -1, dtype=torch.int32, device=dev)
    table_d, inv_d = table.to(dev), inv.to(dev)
    for step, lens in enumerate(([70, 40], [64, 90], [1, 1], [3, 1], [1, 1])):
        t = sum(lens)
        q, k, v = (x.to(dev) for x in _tokens(t, hq, hkv, d, dtype, 20 + step))
        cu = torch.tensor([0, lens[0], t], dtype=torch.int32)
        pos = torch.cat([seen[i] + torch.arange(lens[i]) for i in range(n)])
        seen += torch.tensor(lens)
        kvl = kvl + torch.tensor(lens, dtype=torch.int32, device=dev)
        print(f"serving step {step} lens={lens}", flush=True)
        qr = append_paged(q, k, v, kp, vp, table_d, kvl, cu.to(dev), inv_d, positions=pos.to(dev),
                          slot_positions=pos_state)
        want_q, _ = apply_rotary(q, None, pos.to(dev), inv_d)
        assert torch.equal(qr, want_q)
        out, lse = attn.forward_chunk_paged(qr, kp, vp, table_d, kvl, cu.to(dev), max_seqlen=max(lens), return_lse=True)
        cpu = [x.cpu() for x in (qr, kp, vp, table_d, kvl)]
        want = ref.attention(*cpu, cu)
        o, e = ref.attention_bounds(*want, dtype, d, cap)
        assert bool(((out.cpu().double() - want[0]).abs() <= o).all())
        assert bool(((lse.cpu().double() - want[1]).abs() <= e).all())
        new = accumulate_key_weights(qr, kp, table_d, kvl, cu.to(dev), lse, scores, max_seqlen=max(lens))
        total, dot = ref.key_weights(cpu[0], cpu[1], cpu[3], cpu[4], cu, lse.cpu(), scores.cpu())
        rel = 2 * ((d + 3) * dot + 8 * (1 + dot)) * 2.0 ** -24 + (max(lens) * hq // hkv + 2) * 2.0 ** -24
        assert bool(((new.cpu().double() - total).abs() <= rel * total + 1e-30).all())
        want_e = ref.evict(cpu[1], cpu[2], table, cpu[4], new.cpu(), pos_state.cpu(), budget, recent, sinks)
        kvl, scores, pos_state = evict_paged(kp, vp, table_d, kvl, new, pos_state, budget, recent=recent, sinks=sinks)
        got = [x.cpu() for x in (kp, vp, kvl, scores, pos_state)]
        assert all(torch.equal(a, b) for a, b in zip(got, want_e))
        for i in range(n):  # the newest tokens and the sinks are there, no position twice
            kept = pos_state[i, 0, :int(kvl[i])].tolist()
            assert len(set(kept)) == len(kept) and set(range(sinks)) <= set(kept)
            assert set(range(int(seen[i]) - min(recent, len(kept)), int(seen[i]))) <= set(kept)
    assert math.prod(kp.shape) > 0


def test_serving_step_in_a_graph():
    """Append, attention, weights and eviction captured once and replayed over new tokens, each
    replay against the eager calls on a copy of its state."""
    dev = require_gpu()
    n, hq, hkv, d, page, max_pages, budget = 3, 8, 2, 64, 16, 12, 128
    cap = max_pages * page
    g = torch.Generator().manual_seed(4)
    table = torch.randperm(n * max_pages, generator=g).view(n, max_pages).to(torch.int32).to(dev)
    kp = torch.randn((n * max_pages, page, hkv, d), generator=g).to(BF).to(dev)
    vp = torch.randn((n * max_pages, page, hkv, d), generator=g).to(BF).to(dev)
    kvl = torch.tensor([130, 129, 60], dtype=torch.int32, device=dev)
    cu = torch.tensor([0, 2, 3, 5], dtype=torch.int32, device=dev)
    scores = torch.rand((n, hkv, cap), generator=g).to(dev)
    slots = torch.arange(cap, dtype=torch.int32).expand(n, hkv, cap).contiguous().to(dev)
    q, k, v = (x.to(dev) for x in _tokens(5, hq, hkv, d, BF, 2))
    pos = torch.tensor([128, 129, 128, 58, 59], device=dev)
    inv, _ = rotary_frequencies(d, device=dev)
    attn = BlockSparseFlashAttention(min_sparsity_for_speedup=0.0)

    def step(kp, vp, slots):
        qr = append_paged(q, k, v, kp, vp, table, kvl, cu, inv, positions=pos, slot_positions=slots)
        out, lse = attn.forward_chunk_paged(qr, kp, vp, table, kvl, cu, max_seqlen=2, return_lse=True)
        w = accumulate_key_weights(qr, kp, table, kvl, cu, lse, scores, max_seqlen=2)
        return (qr, out, lse, w, *evict_paged(kp, vp, table, kvl, w, slots, budget, recent=8, sinks=2))

    print("serving step in a graph", flush=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(kp.clone(), vp.clone(), slots.clone())
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(kp, vp, slots)
    for r in range(3):
        q.normal_()
        k.normal_()
        kp.normal_()
        scores.uniform_()
        copies = kp.clone(), vp.clone(), slots.clone()
        want = step(*copies)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert all(torch.equal(a, b) for a, b in zip((kp, vp, slots), copies))


def test_calls_on_two_streams_at_once():
    """Splits, weights and evictions (one head in parts) of two requests on streams of their own, queued
    together: what each gives alone."""
    dev = require_gpu()
    attn = BlockSparseFlashAttention(min_sparsity_for_speedup=0.0)
    work = []
    for i, (lens, kv) in enumerate((([3, 1], [900, 2500]), ([2], [40000]))):
        q, kp, vp, table, kvl, cu = (x.to(dev) for x in ref.make(lens, kv, 8, 2, 64, 16, BF, seed=30 + i))
        cap = table.shape[1] * 16
        scores = torch.rand((len(lens), 2, cap), generator=torch.Generator().manual_seed(i)).to(dev)
        pos = torch.arange(cap, dtype=torch.int32, device=dev).expand(len(lens), 2, cap).contiguous()
        work.append((q, kp.nan_to_num(1.0), vp.nan_to_num(1.0, posinf=1.0), table, kvl, cu, scores, pos, max(lens)))

    def step(q, kp, vp, table, kvl, cu, scores, pos, longest):
        kp, vp = kp.clone(), vp.clone()
        out, lse = attn.forward_chunk_paged(q, kp, vp, table, kvl, cu, max_seqlen=longest, return_lse=True, num_splits=12)
        w = accumulate_key_weights(q, kp, table, kvl, cu, lse, scores, max_seqlen=longest)
        return (out, lse, w, *evict_paged(kp, vp, table, kvl, w, pos, 500, recent=20, sinks=2), kp, vp)

    alone = [step(*x) for x in work]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in work]
    print("two streams", flush=True)
    for _ in range(4):
        got = []
        for x, s in zip(work, streams):
            with torch.cuda.stream(s):
                got.append(step(*x))
        torch.cuda.synchronize()
        for a, b in zip(alone, got):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize(("lens", "over"), [([1], [1]), ([4, 1, 6], [2, 1, 6]), ([40, 300, 2], [9, 0, 2 ** 31 - 1 - 80])])
def test_append_past_the_table(lens, over, given):
    """Lengths (on the device) that pass the table: a token whose slot lies behind it is rotated at its
    own position and written nowhere, and no live key of the table changes."""
    dev = require_gpu()
    page, cap, hq, hkv, d = 16, 80, 4, 2, 64
    _, kp, vp, table, _, cu = ref.make(lens, [cap] * len(lens), hq, hkv, d, page, BF, seed=6, max_pages=cap // page)
    kvl = torch.tensor([cap + x for x in over], dtype=torch.int32)
    t = sum(lens)
    q, k, v = _tokens(t, hq, hkv, d, BF, 5)
    inv, _ = rotary_frequencies(d)
    pos = torch.randint(0, 1 << 20, (t,), generator=torch.Generator().manual_seed(9)) if given else None
    slots = torch.full((len(lens), hkv, cap), -5, dtype=torch.int32)
    a = [x.to(dev) for x in (q, k, v, kp, vp, table, kvl, cu, inv)]
    slots_d = slots.to(dev)
    print(f"append past the table lens={lens} over={over}", flush=True)
    out = append_paged(*a, positions=None if pos is None else pos.to(dev), slot_positions=slots_d)
    torch.cuda.synchronize()
    want_k, want_v = kp.clone(), vp.clone()
    for n, length in enumerate(lens):
        rows = slice(int(cu[n]), int(cu[n + 1]))
        slot = int(kvl[n]) - length + torch.arange(length)
        p = slot if pos is None else pos[rows]
        turned = []
        for got, x in ((out, q), (None, k)):
            want = ref.rotate(x[rows], p[:, None], inv)
            bound = ref.rotate_bound(x[rows], want, inv, 1.0, False, BF)
            turned.append((want, bound))
            if got is not None:
                assert bool(((got[rows].cpu().double() - want).abs() <= bound).all())
        on = (slot >= 0) & (slot < cap)
        pg, row = table[n, slot[on] // page].long(), slot[on] % page
        got = a[3].cpu()[pg, row]
        assert bool(((got.double() - turned[1][0][on]).abs() <= turned[1][1][on]).all())
        want_k[pg, row], want_v[pg, row] = got, v[rows][on]
        slots[n, :, slot[on]] = p[on].to(torch.int32)
    assert torch.equal(slots_d.cpu(), slots)
    assert torch.equal(a[3].cpu().view(torch.int16), want_k.view(torch.int16))  # bits: spare pages hold NaN
    assert torch.equal(a[4].cpu().view(torch.int16), want_v.view(torch.int16))


@pytest.mark.parametrize("masked", [False, True])
def test_no_new_tokens(masked):
    """A step without new tokens: empty results, scores as they were, pages untouched."""
    dev = require_gpu()
    _, kp, vp, table, kvl, cu = ref.make([0, 0], [70, 33], 8, 2, 64, 16, BF, seed=2)
    q, k, v = (torch.empty((0, h, 64), dtype=BF, device=dev) for h in (8, 2, 2))
    a = [x.to(dev) for x in (kp, vp, table, kvl, cu)]
    cap = table.shape[1] * 16
    scores = torch.rand((2, 2, cap), device=dev)
    inv = rotary_frequencies(64, device=dev)[0]
    mask = torch.ones((2, 8, 1, -(-cap // 64)), dtype=torch.bool, device=dev) if masked else None
    print(f"no new tokens, masked={masked}", flush=True)
    qr = append_paged(q, k, v, *a, inv)
    attn = BlockSparseFlashAttention(min_sparsity_for_speedup=0.0)
    for splits in (None, 1, 4):
        out, lse = attn.forward_chunk_paged(qr, *a, mask, max_seqlen=1, return_lse=True, num_splits=splits)
        assert out.shape == (0, 8, 64) and out.dtype == BF and lse.shape == (0, 8) and lse.dtype == torch.float32
    w = accumulate_key_weights(qr, a[0], *a[2:], lse, scores, block_mask=mask, max_seqlen=1)
    assert torch.equal(w, scores)
    assert not accumulate_key_weights(qr, a[0], *a[2:], lse, block_mask=mask, max_seqlen=1).any()
    assert torch.equal(a[0].cpu().view(torch.int16), kp.view(torch.int16))
