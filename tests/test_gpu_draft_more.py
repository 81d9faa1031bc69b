"""Trees of drafted tokens, continued: indices that 32 bits do not hold, positions of two streams at once."""
from __future__ import annotations

import pytest
import torch

import scored_ref as ref
from helpers import require_gpu
from tasft_amd.kernels import accept_draft, commit_draft_paged, draft_tree

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
WIDE = (1 << 32, (1 << 32) + 2, -(1 << 32) + 2, (1 << 63) - 1, -(1 << 63))  # 0, 2, 2, -1 and 0 in 32 bits


@pytest.mark.parametrize("where", ["cpu", "cuda"])
def test_wide_parents_beside_offsets_on_the_device(where):
    """What is no earlier node is a root, also where its low bits would be one."""
    dev = require_gpu()
    parents = [-1, 0, 1, *WIDE, 2]
    n = len(parents)
    clean = [p if 0 <= p < i else -1 for i, p in enumerate(parents)]
    rows = ref.chains(clean, [0, n])
    p = torch.tensor(parents).to(dev if where == "cuda" else "cpu")
    cu, lens = torch.tensor([0, n], device=dev), torch.tensor([n + 20], device=dev)
    print(f"wide parents {where}", flush=True)
    tree = draft_tree(p, cu, lens, max_nodes=n)
    assert torch.equal(tree.ancestors.cpu(), ref.bits(rows, 1))
    assert tree.positions.tolist() == [20 + len(r) - 1 for r in rows]
    tokens, targets = torch.ones(n, dtype=torch.int64), torch.ones(n, dtype=torch.int64)
    got = accept_draft(p, tokens.to(dev), targets.to(dev), cu, max_nodes=n)
    want = ref.accept(clean, tokens.tolist(), targets.tolist(), [0, n], None, n)
    assert got.path.tolist() == want[0] and got.counts.tolist() == want[1]


@pytest.mark.parametrize("where", ["cpu", "cuda"])
def test_wide_paths(where):
    """An index that is no node is not moved, also where its low bits would be one; counts alike."""
    dev = require_gpu()
    g = torch.Generator().manual_seed(0)
    k, v = (torch.randn((4, 8, 2, 64), generator=g).to(BF) for _ in range(2))
    table, lens, cu = torch.arange(4, dtype=torch.int32).view(1, 4), torch.tensor([30]), torch.tensor([0, 10])
    path = torch.tensor([[(1 << 32) + 5, 3, (1 << 32) + 7, 8]])
    print(f"wide path {where}", flush=True)
    for count, moved in ((4, {1: 3, 3: 8}), ((1 << 32) + 1, {1: 3, 3: 8}), (-(1 << 32) + 1, {})):
        kd, vd = k.to(dev), v.to(dev)
        at = dev if where == "cuda" else "cpu"
        out = commit_draft_paged(kd, vd, table.to(dev), lens.to(dev), cu.to(dev), path.to(at), torch.tensor([count]).to(at))
        assert out.tolist() == [20 + (4 if count > 0 else 0)]
        for pool, was in ((kd, k), (vd, v)):
            want = was.flatten(0, 1).clone()
            for to, node in moved.items():
                want[20 + to] = was.flatten(0, 1)[20 + node]
            assert torch.equal(pool.cpu().flatten(0, 1), want)


def test_positions_of_two_streams():
    dev = require_gpu()
    sizes, past = [64, 40], [236, 60]
    cu = torch.tensor([0, 64, 104], dtype=torch.int32, device=dev)
    lens = torch.tensor([a + b for a, b in zip(sizes, past)], dtype=torch.int32, device=dev)
    made = [ref.random_parents(sizes, seed) for seed in (1, 2)]
    given = [torch.tensor(p, dtype=torch.int32, device=dev) for p in made]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [None, None]
    print("positions of two streams", flush=True)
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = draft_tree(given[i], cu, lens, max_nodes=64)
        torch.cuda.synchronize()
        for parents, tree in zip(made, got):
            rows = ref.chains(parents, [0, 64, 104])
            start = [past[0]] * 64 + [past[1]] * 40
            assert tree.positions.tolist() == [a + len(r) - 1 for a, r in zip(start, rows)]
            assert torch.equal(tree.ancestors.cpu(), ref.bits(rows, 1))
