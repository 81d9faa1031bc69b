"""Trees of drafted tokens: plans, what is kept, and the move of the kept tokens' keys and values."""
from __future__ import annotations

import pytest
import torch

import paged_ref
import scored_ref as ref
from helpers import require_gpu
from tasft_amd.kernels import (
    BlockSparseFlashAttention,
    accept_draft,
    append_paged,
    commit_draft_paged,
    draft_tree,
    rotary_frequencies,
)

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
SIZES = [[1], [2, 1, 3], [25], [64, 63, 0, 33], [65, 64], [130, 7, 200], [700], [0, 0, 5], [17] * 70, [4096, 9]]


def offsets(sizes):
    return torch.tensor([0] + sizes).cumsum(0).to(torch.int32)


@pytest.mark.parametrize("index", range(len(SIZES)))
@pytest.mark.parametrize("deep", [0.3, 0.95])
def test_plans(index, deep):
    sizes, pad = SIZES[index], 3
    dev = require_gpu()
    parents = ref.random_parents(sizes, index, deep=deep)
    cu = offsets(sizes)
    rows = ref.chains(parents, cu.tolist())
    most = max(sizes) + (index % 3)
    most = min(most, 4096)
    words = -(-most // 64)
    lens = torch.tensor([n + 100 * i for i, n in enumerate(sizes)], dtype=torch.int32)
    p = torch.tensor(parents + [7] * pad)
    print(f"plan {sizes[:6]} deep={deep}", flush=True)
    tree = draft_tree(p.to(dev), cu.to(dev), lens.to(dev), max_nodes=most)
    assert tree.ancestors.shape == (len(p), words)
    assert torch.equal(tree.ancestors[:len(rows)].cpu(), ref.bits(rows, words))
    start = torch.cat([torch.full((n,), 100 * i) for i, n in enumerate(sizes)])
    want = start + torch.tensor([len(r) - 1 for r in rows], dtype=torch.int64)
    assert torch.equal(tree.positions[:len(rows)].cpu().long(), want)
    assert not tree.ancestors[len(rows):].any() and not tree.positions[len(rows):].any()
    # From host tensors the same.
    if most == max(sizes):
        host = draft_tree(torch.tensor(parents, dtype=torch.int32), cu, lens.to(dev))
        assert torch.equal(host.ancestors, tree.ancestors[:len(rows)])


def test_plans_of_odd_parents_and_cut_trees():
    """On the device anything that is no earlier node is a root; nodes behind max_nodes have no bits."""
    dev = require_gpu()
    parents = torch.tensor([-1, 0, 5, -7, 3, 4, 6, 1 << 30, -(1 << 31), 8], dtype=torch.int32)
    cu = torch.tensor([0, 10], dtype=torch.int32)
    clean = [p if 0 <= p < i else -1 for i, p in enumerate(parents.tolist())]
    rows = ref.chains(clean, [0, 10])
    print("plan odd", flush=True)
    tree = draft_tree(parents.to(dev), cu.to(dev), torch.tensor([10], device=dev), max_nodes=64)
    assert torch.equal(tree.ancestors.cpu(), ref.bits(rows, 1))
    wide = parents.long()
    wide[7], wide[8] = 1 << 32, -(1 << 32) + 2  # of which 32 bits would be earlier nodes
    assert torch.equal(draft_tree(wide.to(dev), cu.to(dev), torch.tensor([10], device=dev), max_nodes=64).ancestors,
                       tree.ancestors)
    tree = draft_tree(parents.to(dev), cu.to(dev), torch.tensor([30], device=dev), max_nodes=6)
    assert torch.equal(tree.ancestors[:6].cpu(), ref.bits(rows, 1)[:6]) and not tree.ancestors[6:].any()
    assert tree.positions[:6].tolist() == [20 + len(r) - 1 for r in rows[:6]]


@pytest.mark.parametrize("dtype", [torch.int64, torch.int32])
@pytest.mark.parametrize("first", [False, True])
@pytest.mark.parametrize("index", range(len(SIZES)))
def test_accept(index, first, dtype):
    sizes = SIZES[index]
    dev = require_gpu()
    parents = ref.random_parents(sizes, 50 + index, deep=0.6)
    cu = offsets(sizes)
    g = torch.Generator().manual_seed(index)
    # Few tokens, so that paths agree for a while and several agree equally far.
    t = len(parents)
    vocab = 1 << 40 if dtype == torch.int64 else 1 << 20
    tokens = torch.randint(0, 2, (t + 2,), generator=g).to(dtype) * (vocab - 1)
    targets = torch.randint(0, 2, (t + 2,), generator=g).to(dtype) * (vocab - 1)
    start = torch.randint(0, 2, (len(sizes),), generator=g).to(dtype) * (vocab - 1) if first else None
    most = max(sizes)
    want = ref.accept(parents, tokens.tolist(), targets.tolist(), cu.tolist(), None if start is None else start.tolist(),
                      most)
    p = torch.tensor(parents + [0, 0], dtype=torch.int32)
    print(f"accept {sizes[:6]} first={first} {dtype}", flush=True)
    got = accept_draft(p.to(dev), tokens.to(dev), targets.to(dev), cu.to(dev), max_nodes=most,
                       first_targets=None if start is None else start.to(dev))
    assert got.path.tolist() == want[0] and got.counts.tolist() == want[1]
    assert got.next_tokens.dtype == dtype and got.next_tokens.tolist() == want[2]


@pytest.mark.parametrize("stop", [1, 63, 64, 1000, 4096])
def test_accept_chains(stop):
    """The deepest trees there are: chains that agree up to a node, beside one that agrees to its end."""
    dev = require_gpu()
    sizes = [4096, 300, 1]
    parents = [i - 1 for n in sizes for i in range(n)]
    tokens = torch.ones(sum(sizes), dtype=torch.int64)
    targets = tokens.clone()
    if 0 < stop < 4096:
        tokens[stop] = 7
    cu = offsets(sizes)
    want = ref.accept(parents, tokens.tolist(), targets.tolist(), cu.tolist(), None, 4096)
    assert want[1] == [stop, 300, 1]
    p = torch.tensor(parents, dtype=torch.int32, device=dev)
    print(f"accept chain {stop}", flush=True)
    got = accept_draft(p, tokens.to(dev), targets.to(dev), cu.to(dev), max_nodes=4096)
    assert got.path.tolist() == want[0] and got.counts.tolist() == want[1] and got.next_tokens.tolist() == want[2]
    tree = draft_tree(p, cu.to(dev), torch.tensor(sizes, device=dev), max_nodes=4096)
    assert torch.equal(tree.ancestors.cpu(), ref.bits(ref.chains(parents, cu.tolist()), 64))


def _pools(kv, sizes, hkv, d, page, dtype, seed, spare=2):
    _, k, v, table, lens, cu = paged_ref.make(sizes, kv, hkv, hkv, d, page, dtype, seed=seed, spare_pages=spare)
    return k.nan_to_num(3.0), v.nan_to_num(4.0, posinf=5.0), table, lens, cu


def _paths(sizes, seed):
    g = torch.Generator().manual_seed(seed)
    width = max(max(sizes), 1)
    path, counts = torch.full((len(sizes), width), -1, dtype=torch.int32), []
    for n, size in enumerate(sizes):
        c = int(torch.randint(0, min(size, 40) + 1, (1,), generator=g))
        path[n, :c] = torch.randperm(size, generator=g)[:c].sort().values.to(torch.int32)
        counts.append(c)
    return path, torch.tensor(counts, dtype=torch.int32)


@pytest.mark.parametrize("positions", [False, True])
@pytest.mark.parametrize(("sizes", "kv", "hkv", "d", "page", "dtype"), [
    ([1], [1], 1, 8, 1, BF),
    ([5, 0, 9], [20, 7, 9], 2, 64, 8, HF),
    ([64, 33, 17, 64], [64, 1000, 100, 333], 8, 128, 16, BF),
    ([300], [511], 3, 256, 64, BF),
    ([25] * 70, [300] * 70, 4, 128, 4, HF),
])
def test_commit(sizes, kv, hkv, d, page, dtype, positions):
    dev = require_gpu()
    k, v, table, lens, cu = _pools(kv, sizes, hkv, d, page, dtype, seed=len(sizes))
    path, counts = _paths(sizes, d)
    cap = table.shape[1] * page
    pos = torch.arange(len(sizes) * hkv * cap, dtype=torch.int32).view(len(sizes), hkv, cap) if positions else None
    want = ref.commit(k, v, table, lens, cu, path, counts, pos)
    kd, vd = k.to(dev), v.to(dev)
    pd = None if pos is None else pos.to(dev)
    print(f"commit {sizes[:6]} {hkv} x {d} page {page}", flush=True)
    got = commit_draft_paged(kd, vd, table.to(dev), lens.to(dev), cu.to(dev), path.to(dev), counts.to(dev),
                             slot_positions=pd)
    assert got.dtype == torch.int32 and torch.equal(got.cpu(), want[2])
    assert torch.equal(kd.cpu(), want[0]) and torch.equal(vd.cpu(), want[1])
    if positions:
        assert torch.equal(pd.cpu(), want[3])


def test_commit_leaves_alone_what_is_not_there():
    """Counts and nodes past what there is, pages outside the pool and slots outside the table."""
    dev = require_gpu()
    sizes, kv = [6, 6], [40, 20]
    k, v, table, lens, cu = _pools(kv, sizes, 2, 64, 8, BF, seed=3)
    path = torch.tensor([[0, 99, -5, 4], [3, 1, 2, 5]], dtype=torch.int32)
    counts = torch.tensor([9, 4], dtype=torch.int32)
    kd, vd = k.to(dev), v.to(dev)
    print("commit odd", flush=True)
    got = commit_draft_paged(kd, vd, table.to(dev), lens.to(dev), cu.to(dev), path.to(dev), counts.to(dev))
    assert got.tolist() == [34 + 4, 14 + 4]
    where = lambda n, s: (int(table[n, s // 8]), s % 8)  # noqa: E731
    for pool, was in ((kd.cpu(), k), (vd.cpu(), v)):
        moved = was.clone()
        moved[where(0, 37)] = was[where(0, 38)]  # node 4 to place 3
        moved[where(1, 14)] = was[where(1, 17)]  # node 3 to place 0; 1 and 2 stay, 5 to place 3
        moved[where(1, 17)] = was[where(1, 19)]
        assert torch.equal(pool, moved)
    # Every slot outside the table, or every page outside the pool: nothing moves.
    before = kd.clone()
    far = (lens + 10000).to(dev)
    commit_draft_paged(kd, vd, table.to(dev), far, cu.to(dev), path.to(dev), counts.to(dev))
    commit_draft_paged(kd, vd, table.to(dev), (lens - 10000).to(dev), cu.to(dev), path.to(dev), counts.to(dev))
    commit_draft_paged(kd, vd, torch.full_like(table, 1 << 20).to(dev), lens.to(dev), cu.to(dev), path.to(dev),
                       counts.to(dev))
    commit_draft_paged(kd, vd, torch.full_like(table, -3).to(dev), lens.to(dev), cu.to(dev), path.to(dev),
                       counts.to(dev))
    assert torch.equal(kd, before)


def test_commit_layouts_and_far_pages():
    """Head-major pools, and pages 128 MB apart."""
    dev = require_gpu()
    sizes, kv = [20, 33], [300, 64]
    k, v, table, lens, cu = _pools(kv, sizes, 4, 128, 32, BF, seed=5)
    path, counts = _paths(sizes, 5)
    want = ref.commit(k, v, table, lens, cu, path, counts)
    rest = [x.to(dev) for x in (table, lens, cu, path, counts)]
    print("commit layouts", flush=True)
    for lay in range(2):
        pools = []
        for x in (k, v):
            if lay == 0:
                y = x.to(dev).permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
            else:
                y = torch.empty((x.shape[0], 1 << 26), dtype=BF, device=dev)[:, :x[0].numel()].view(x.shape)
                y.copy_(x)
            pools.append(y)
        wide = torch.full((2, table.shape[1] + 3), 99, dtype=torch.int32, device=dev)
        wide[:, :table.shape[1]] = rest[0]
        commit_draft_paged(*pools, wide[:, :table.shape[1]], *rest[1:])
        assert torch.equal(pools[0].cpu(), want[0]) and torch.equal(pools[1].cpu(), want[1])


def test_empty():
    dev = require_gpu()
    none = torch.zeros(0, dtype=torch.int32, device=dev)
    cu = torch.zeros(3, dtype=torch.int32, device=dev)
    lens = torch.tensor([5, 0], dtype=torch.int32, device=dev)
    tree = draft_tree(none, cu, lens, max_nodes=10)
    assert tree.ancestors.shape == (0, 1) and tree.positions.shape == (0,)
    kept = accept_draft(none, none, none, cu, max_nodes=4)
    assert kept.counts.tolist() == [0, 0] and kept.next_tokens.tolist() == [-1, -1] and bool((kept.path == -1).all())
    first = torch.tensor([7, 8], dtype=torch.int32, device=dev)
    assert accept_draft(none, none, none, cu, max_nodes=4, first_targets=first).next_tokens.tolist() == [7, 8]
    k = torch.zeros((4, 8, 2, 64), dtype=BF, device=dev)
    table = torch.arange(4, dtype=torch.int32, device=dev).view(2, 2)
    got = commit_draft_paged(k, k.clone(), table, lens, cu, kept.path[:, :0], kept.counts)
    assert got.tolist() == [5, 0]


@pytest.mark.parametrize("graph", [False, True])
def test_a_drafting_step(graph):
    """Plan, append, attention, acceptance and commit, as a server runs them, eager and captured: the cache
    ends as if the kept tokens alone had been appended, and the attention is that of the 64-bit form."""
    dev = require_gpu()
    sizes, past, hq, hkv, d, page, most = [13, 20, 1, 7], [50, 3, 0, 97], 8, 2, 64, 16, 20
    cu = offsets(sizes)
    t, n = sum(sizes), len(sizes)
    inv, factor = rotary_frequencies(d, device=dev)
    table = torch.randperm(40, generator=torch.Generator().manual_seed(1))[:4 * 9].view(4, 9).to(torch.int32)
    lens = torch.tensor([a + b for a, b in zip(past, sizes)], dtype=torch.int32)
    attn = BlockSparseFlashAttention(min_sparsity_for_speedup=0.0)
    held = None
    captured = None
    cu_d, table_d, lens_d = cu.to(dev), table.to(dev), lens.to(dev)

    def step(parents, tokens, targets, q, k, v, kp, vp):
        tree = draft_tree(parents, cu_d, lens_d, max_nodes=most)
        turned = append_paged(q, k, v, kp, vp, table_d, lens_d, cu_d, inv, scale=factor, positions=tree.positions)
        out, lse = attn.forward_chunk_paged(turned, kp, vp, table_d, lens_d, cu_d, max_seqlen=most,
                                            ancestors=tree.ancestors, return_lse=True)
        before = kp.clone(), vp.clone()
        kept = accept_draft(parents, tokens, targets, cu_d, max_nodes=most)
        return turned, out, lse, *before, commit_draft_paged(kp, vp, table_d, lens_d, cu_d, kept.path, kept.counts), *kept

    for seed in range(4):
        g = torch.Generator().manual_seed(seed)
        parents = ref.random_parents(sizes, seed, roots=0.0)
        tokens, targets = torch.randint(0, 2, (2, t), generator=g)
        q, k, v = (torch.randn((t, h, d), generator=g).to(BF) for h in (hq, hkv, hkv))
        pools = [torch.randn((40, page, hkv, d), generator=g).to(BF) for _ in range(2)]
        fresh = [x.to(dev) for x in (torch.tensor(parents, dtype=torch.int32), tokens, targets, q, k, v, *pools)]
        print(f"draft step graph={graph} seed={seed}", flush=True)
        if not graph:
            got = step(*fresh)
        else:
            if held is None:
                held = [x.clone() for x in fresh]
                side = torch.cuda.Stream()
                with torch.cuda.stream(side):
                    step(*held)
                torch.cuda.synchronize()
                captured = torch.cuda.CUDAGraph()
                with torch.cuda.graph(captured):
                    result = step(*held)
            for a, b in zip(held, fresh):
                a.copy_(b)
            captured.replay()
            got, fresh = result, held
        torch.cuda.synchronize()
        turned, out, lse, kb, vb, new_lens, path, counts, following = (x.cpu() for x in got)
        rows = ref.chains(parents, cu.tolist())
        o, l, e_o, e_l = ref.attention(turned, kb, vb, table, lens, cu, rows=rows)
        assert bool(((out.double() - o).abs() <= e_o).all()) and bool(((lse.double() - l).abs() <= e_l).all())
        want = ref.accept(parents, tokens.tolist(), targets.tolist(), cu.tolist(), None, most)
        assert path.tolist() == want[0] and counts.tolist() == want[1] and following.tolist() == want[2]
        assert new_lens.tolist() == [a + c for a, c in zip(past, want[1])]
        # The kept tokens alone, appended as a chain.
        index = torch.cat([int(cu[i]) + path[i, :counts[i]] for i in range(n)]).long()
        plain = [x.to(dev) for x in pools]
        append_paged(q[index].to(dev), k[index].to(dev), v[index].to(dev), *plain, table_d, new_lens.to(dev),
                     offsets(counts.tolist()).to(dev), inv, scale=factor)
        for a, b in zip(fresh[6:], plain):
            for i in range(n):
                s = torch.arange(int(new_lens[i]), device=dev)
                at = table_d[i, s // page].long(), s % page
                assert torch.equal(a[at], b[at])


def test_two_streams():
    """Plans and commits of two streams at once."""
    dev = require_gpu()
    sizes, kv = [64, 40], [300, 100]
    made = []
    for seed in (1, 2):
        k, v, table, lens, cu = _pools(kv, sizes, 4, 128, 16, BF, seed=seed)
        path, counts = _paths(sizes, seed)
        parents = torch.tensor(ref.random_parents(sizes, seed), dtype=torch.int32)
        made.append(([x.to(dev) for x in (k, v, table, lens, cu, path, counts)], parents.to(dev),
                     ref.commit(k, v, table, lens, cu, path, counts), ref.chains(parents.tolist(), cu.tolist())))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    print("draft two streams", flush=True)
    for s, (a, parents, _, _) in zip(streams, made):
        with torch.cuda.stream(s):
            tree = draft_tree(parents, a[4], a[3], max_nodes=64)
            got.append((commit_draft_paged(*a), tree))
    torch.cuda.synchronize()
    for (lens, tree), (a, _, want, rows) in zip(got, made):
        assert torch.equal(a[0].cpu(), want[0]) and torch.equal(a[1].cpu(), want[1]) and torch.equal(lens.cpu(), want[2])
        assert torch.equal(tree.ancestors.cpu(), ref.bits(rows, 1)) and tree.positions.numel() == sum(sizes)
