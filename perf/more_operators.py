"""Attention with capped and biased scores, and drafted token trees, as cases for timing and comparison.

Operators: dense attention of a training step with its gradients (scores capped by a tanh, a bias
that falls with distance, packed documents, prefixes that see both ways); the same scores in
attention over a paged cache, down to single tokens; attention of a tree of drafted tokens over a
paged cache; the plan of such a tree and which of its tokens are kept; and the move of the kept
tokens' keys and values to the end of the cache. Head counts and lengths are those of
``perf/cases.py`` and ``tasft_amd.workloads`` (Llama-3-8B and Qwen-2.5-7B heads) and generic ones
beside them.

With ``own`` false ``run`` computes each operator in plain torch, in 32 bits; with ``own`` true it
calls ``tasft_amd``. ``exact`` is the definition in 64 bits.
"""
from __future__ import annotations

import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed() -> list[dict]:
    return [
        # A training step over one long sequence, scores capped at 50 (Llama-3-8B heads).
        _case("attend", "attend_capped", batch=1, seq=8192, softcap=50.0, grad=True),
        # A packed batch of documents of different lengths, each with a prefix that sees both ways
        # (Qwen-2.5-7B heads).
        _case("attend", "attend_documents", batch=10, seq=3500, ragged=True, packed=True, prefix=True, q_heads=28,
              kv_heads=4, grad=True),
        # A padded batch with a bias by distance, heads of 64 in fp16.
        _case("attend", "attend_biased", batch=3, seq=1000, ragged=True, alibi=True, q_heads=16, kv_heads=16,
              head_dim=64, dtype="fp16", grad=True),
        # A few short sequences: launches and host time count.
        _case("attend", "attend_short", batch=4, seq=77, softcap=30.0, prefix=True, q_heads=8, kv_heads=2, grad=True),
        # One new token of each of 64 requests over their caches, scores capped.
        _case("chunk", "chunk_capped", batch=64, chunk=1, kv=8192, ragged=True, softcap=50.0),
        # Chunked prefill of one prompt with a bias by distance.
        _case("chunk", "chunk_biased", batch=1, chunk=1024, kv=16384, page=64, alibi=True, q_heads=28, kv_heads=4),
        # Trees of 64 drafted tokens of each of 16 requests, checked at once.
        _case("tree", "tree_batch", batch=16, nodes=64, depth=8, kv=8192, ragged=True),
        # A small tree of one request, biased and capped, heads of 64 in fp16.
        _case("tree", "tree_single", batch=1, nodes=25, depth=6, kv=1000, page=32, alibi=True, softcap=30.0,
              q_heads=16, kv_heads=16, head_dim=64, dtype="fp16"),
        # The plan of a step's trees and which tokens of them are kept, of 64 requests.
        _case("draft", "draft_batch", batch=64, nodes=64, depth=8, ragged=True),
        # The same of a few wide trees.
        _case("draft", "draft_wide", batch=4, nodes=500, depth=20, ragged=True),
        # The kept tokens' keys and values of 64 requests moved to the ends of their caches.
        _case("commit", "commit_batch", batch=64, nodes=64, depth=8, kv=1040, ragged=True),
        # The same of one request.
        _case("commit", "commit_single", batch=1, nodes=25, depth=6, kv=1000, page=32, q_heads=16, kv_heads=16,
              head_dim=64, dtype="fp16"),
    ]


def draw(rng) -> dict:
    heads, kv_heads = rng.choice([(32, 8), (28, 4), (16, 16), (8, 2), (12, 4)])
    f = {"q_heads": heads, "kv_heads": kv_heads, "head_dim": rng.choice([128, 128, 64]),
         "dtype": rng.choice(["bf16", "bf16", "fp16"])}
    score = {"softcap": rng.choice([0.0, 0.0, 20.0, 50.0]), "alibi": rng.random() < 0.4}
    page = {"page": rng.choice([8, 16, 16, 32, 64, 128])}

    def length(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["attend", "attend", "attend", "chunk", "tree", "tree", "draft", "commit"])
    if kind == "attend":
        seq = length(1, 8192)
        most = max(1, min(16, 16384 // seq, (1 << 26) // (seq * seq)))
        causal = rng.random() < 0.8
        return _case(kind, None, batch=rng.randint(1, most), seq=seq, ragged=rng.random() < 0.6,
                     packed=rng.random() < 0.5, causal=causal, prefix=causal and rng.random() < 0.4,
                     grad=rng.random() < 0.75, **f, **score)
    if kind == "chunk":
        kv = length(50, 32768)
        chunk = min(kv, rng.choice([1, length(2, 16), length(16, 1024)]))
        most = min(64, 500000 // kv, (1 << 24) // (chunk * kv))
        return _case(kind, None, batch=rng.randint(1, max(1, most)), chunk=chunk, kv=kv, ragged=rng.random() < 0.7,
                     **f, **page, **score)
    nodes = length(2, 300)
    depth = rng.randint(1, min(24, nodes - 1))
    if kind == "draft":
        return _case(kind, None, batch=rng.randint(1, max(1, 4096 // nodes)), nodes=nodes, depth=depth,
                     ragged=rng.random() < 0.7)
    kv = max(2 * nodes, length(100, 16384 if kind == "tree" else 2048))
    most = max(1, min(64, 200000 // kv, (1 << 23) // (nodes * kv)))
    return _case(kind, None, batch=rng.randint(1, most), nodes=nodes, depth=depth, kv=kv, ragged=rng.random() < 0.7,
                 **f, **page, **(score if kind == "tree" else {}))


def _case(kind, name, **fields):
    case = {"kind": kind, "ragged": False}
    if kind != "draft":
        case.update(q_heads=32, kv_heads=8, head_dim=128, dtype="bf16")
    if kind in ("attend", "chunk", "tree"):
        case.update(softcap=0.0, alibi=False)
    if kind == "attend":
        case.update(packed=False, causal=True, prefix=False, grad=False)
    elif kind != "draft":
        case.update(page=16)
    case.update(fields)
    if name is not None:
        case["name"] = name
    return case


# ------------------------------------------------------------------------------- inputs
def _randn(g, shape, dtype):
    return torch.randn(shape, generator=g, device="cuda", dtype=dtype)


def _sizes(case, n, longest, least):
    """New tokens of each sequence. They go by the case alone, so that outputs of every seed have one
    shape."""
    if not case["ragged"]:
        return [longest] * n
    rng = random.Random(longest * 1000003 + n)
    return [longest] + [rng.randint(least, longest) for _ in range(n - 1)]


def _offsets(sizes):
    return torch.tensor([0] + sizes, dtype=torch.int32).cumsum(0).to(torch.int32).to("cuda")


def _slopes(case):
    """A head's bias per position: a geometric series over the heads."""
    if not case["alibi"]:
        return None
    h = case["q_heads"]
    return torch.tensor([2.0 ** (-8.0 * (i + 1) / h) for i in range(h)], dtype=torch.float32, device="cuda")


def _trees(rng, sizes, depth):
    """Parents of trees of drafted tokens: node 0 is the last token, later nodes hang below it, at
    most ``depth`` deep, earlier ones (the likelier) more often chosen."""
    parents = []
    for size in sizes:
        at, level = [-1], [0]
        for i in range(1, size):
            p = min(int(i * rng.random() ** 1.5), i - 1)
            while level[p] >= depth:
                p = at[p]
            at.append(p)
            level.append(level[p] + 1)
        parents += at
    return parents


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind, n = case["kind"], case["batch"]
    st = {"case": case}
    if kind == "draft":
        rng = random.Random(seed)
        sizes = _sizes(case, n, case["nodes"], max(1, case["nodes"] // 2))
        parents = _trees(rng, sizes, case["depth"])
        tokens = [rng.randrange(32000) for _ in parents]
        targets, first = [rng.randrange(32000) for _ in parents], 0
        for size in sizes:  # four of five nodes with drafted successors are followed by one of them
            for i in range(size - 1, 0, -1):
                if rng.random() < 0.8:
                    targets[first + parents[first + i]] = tokens[first + i]
            first += size
        st["parents"] = torch.tensor(parents, dtype=torch.int32, device="cuda")
        st["tokens"] = torch.tensor(tokens, dtype=torch.int64, device="cuda")
        st["targets"] = torch.tensor(targets, dtype=torch.int64, device="cuda")
        st["cu"] = _offsets(sizes)
        lens = torch.randint(0, 8192, (n,), generator=g, device="cuda", dtype=torch.int32)
        st["kv_lens"] = lens + torch.tensor(sizes, dtype=torch.int32, device="cuda")
        return st
    dt, hq, hkv, d = _DTYPES[case["dtype"]], case["q_heads"], case["kv_heads"], case["head_dim"]
    if kind == "attend":
        s = case["seq"]
        sizes = _sizes(case, n, s, max(1, s // 8))
        st["sizes"], st["slopes"] = sizes, _slopes(case)
        st["cu"] = _offsets(sizes)
        st["lens"] = st["cu"][1:] - st["cu"][:-1]
        if case["packed"]:
            shape = (sum(sizes), hq, d)
            st["q"], st["k"], st["v"], st["gout"] = (_randn(g, (sum(sizes), h, d), dt) for h in (hq, hkv, hkv, hq))
        else:
            # Projections give [B, S, H, D]; attention takes the transposed view.
            st["q"], st["k"], st["v"], st["gout"] = (_randn(g, (n, s, h, d), dt).transpose(1, 2)
                                                     for h in (hq, hkv, hkv, hq))
        st["prefix"] = None
        if case["prefix"]:
            part = torch.rand((n,), generator=g, device="cuda")
            st["prefix"] = (part * (st["lens"] + 1)).to(torch.int32).minimum(st["lens"])
        if case["grad"]:
            for x in ("q", "k", "v"):
                st[x].requires_grad_(True)
        return st
    ps, kv = case["page"], case["kv"]
    pages = -(-kv // ps)
    st["table"] = torch.randperm(n * pages, generator=g, device="cuda").view(n, pages).to(torch.int32)
    st["k_pages"] = _randn(g, (n * pages, ps, hkv, d), dt)
    st["v_pages"] = _randn(g, (n * pages, ps, hkv, d), dt)
    lens = torch.full((n,), kv, dtype=torch.int32, device="cuda")
    if case["ragged"]:
        lens = torch.randint(kv // 2 + 1, kv + 1, (n,), generator=g, device="cuda", dtype=torch.int32)
        lens[0] = kv
    st["kv_lens"] = lens
    new = case["chunk"] if kind == "chunk" else case["nodes"]
    most = kv // 2 + 1
    sizes = [new] + [min(x, most) for x in _sizes(case, n, new, new // 2 + 1)[1:]]
    st["tokens"], st["max_seqlen"] = sum(sizes), new
    st["cu"] = _offsets(sizes)
    if kind == "commit":
        # Of each tree, a path of rising nodes from node 0 on.
        rng = random.Random(seed)
        rows, counts = [], []
        for size in sizes:
            deep = rng.randint(1, min(size, case["depth"] + 1))
            rows.append([0] + sorted(rng.sample(range(1, size), deep - 1)) + [-1] * (new - deep))
            counts.append(deep)
        st["path"] = torch.tensor(rows, dtype=torch.int32, device="cuda")
        st["counts"] = torch.tensor(counts, dtype=torch.int32, device="cuda")
        return st
    st["slopes"] = _slopes(case)
    st["q"] = _randn(g, (st["tokens"], hq, d), dt)
    if kind == "tree":
        parents = _trees(random.Random(seed), sizes, case["depth"])
        parents = torch.tensor(parents, dtype=torch.int32, device="cuda")
        st["ancestors"] = _pack(_reach(parents, st["cu"], new))[_of_token(st["cu"], st["tokens"])]
    return st


# ----------------------------------------------------------------------- the plain forms
def _of_token(cu, tokens):
    """Each packed token's sequence, and its place in it."""
    at = torch.arange(tokens, device=cu.device)
    seq = torch.searchsorted(cu[1:].long(), at, right=True)
    return seq, at - cu[seq]


def _reach(parents, cu, longest):
    """[N, L, L] bool: node j is node i or one of its ancestors, by doubling the steps taken."""
    seq, place = _of_token(cu, parents.numel())
    step = torch.zeros((cu.numel() - 1, longest, longest), device="cuda")
    step[seq, place, place] = 1.0
    step[seq, place, torch.where(parents >= 0, parents, place).long()] = 1.0
    for _ in range(max(1, (longest - 1).bit_length())):
        step = (torch.matmul(step, step) > 0).float()
    return step > 0


def _pack(bits):
    """Bools [..., L] as words of 64 bits [..., ceil(L / 64)]."""
    words = -(-bits.shape[-1] // 64)
    padded = torch.nn.functional.pad(bits, (0, 64 * words - bits.shape[-1])).unflatten(-1, (words, 64))
    return (padded.long() << torch.arange(64, device=bits.device)).sum(-1)


def _modified(s, case, slopes, distance):
    """Scores [N, Hq, L, C] with the cap and the bias, and the cap's derivative (None without one)."""
    slope = None
    if case["softcap"]:
        t = torch.tanh(s / case["softcap"])
        s, slope = t * case["softcap"], 1.0 - t * t
    if slopes is not None:
        s = s - slopes.view(1, -1, 1, 1) * distance
    return s, slope


def _padded(x, st):
    """Packed [T, H, D] or batched [B, H, S, D] as [N, H, L, D] in 32 bits."""
    if not st["case"]["packed"]:
        return x.detach().float()
    seq, place = _of_token(st["cu"], x.shape[0])
    out = torch.zeros((len(st["sizes"]), st["case"]["seq"], *x.shape[1:]), device="cuda")
    out[seq, place] = x.detach().float()
    return out.transpose(1, 2)


def _as_given(x, st):
    """[N, H, L, D] in the inputs' layout and type, 0 where no token is."""
    dt = _DTYPES[st["case"]["dtype"]]
    if st["case"]["packed"]:
        seq, place = _of_token(st["cu"], sum(st["sizes"]))
        return x[seq, :, place].to(dt)
    live = torch.arange(x.shape[2], device="cuda") < st["lens"].view(-1, 1)
    return torch.where(live[:, None, :, None], x, 0.0).to(dt)


def _attend(st):
    case = st["case"]
    hq, hkv, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    n, L, grp, scale = case["batch"], case["seq"], hq // hkv, 1.0 / math.sqrt(d)
    q, k, v = (_padded(st[x], st) for x in "qkv")
    rows = lambda x: x.reshape(n, hkv, grp * L, x.shape[-1])  # noqa: E731  the rows that share a KV head
    i, j = torch.arange(L, device="cuda").view(L, 1), torch.arange(L, device="cuda")
    s = torch.matmul(rows(q), k.transpose(2, 3)).view(n, hq, L, L).mul_(scale)
    s, slope = _modified(s, case, st["slopes"], (i - j).abs().float())
    lens = st["lens"].view(n, 1, 1, 1)
    dead = (j >= lens) | (i >= lens)
    if case["causal"]:
        behind = j > i
        if st["prefix"] is not None:
            behind = behind & (j >= st["prefix"].view(n, 1, 1, 1))
        dead = dead | behind
    s = s.masked_fill_(dead, -math.inf)
    top = s.amax(-1, keepdim=True).nan_to_num_(neginf=0.0)
    p = s.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    lse = (top + total.log()).squeeze(-1)
    p = p.div_(torch.where(total > 0, total, 1.0))
    o = torch.matmul(rows(p), v).view(n, hq, L, d)
    if not case["grad"]:
        if case["packed"]:
            seq, place = _of_token(st["cu"], sum(st["sizes"]))
            lse = lse[seq, :, place]
        return [_as_given(o, st), lse]
    go = _padded(st["gout"], st)
    ds = torch.matmul(rows(go), v.transpose(2, 3)).view(n, hq, L, L)
    ds = ds.sub_((go * o).sum(-1, keepdim=True)).mul_(p).masked_fill_(dead, 0.0)
    if slope is not None:
        ds = ds.mul_(slope)
    gq = torch.matmul(rows(ds), k).view(n, hq, L, d) * scale
    gk = torch.matmul(rows(ds).transpose(2, 3), rows(q)) * scale
    gv = torch.matmul(rows(p).transpose(2, 3), rows(go))
    return [_as_given(x, st) for x in (o, gq, gk, gv)]


def _over_cache(st):
    """A chunk's or a tree's tokens over the pages of their sequences."""
    case, cu, lens = st["case"], st["cu"], st["kv_lens"]
    n, ps, L = case["batch"], case["page"], st["max_seqlen"]
    hq, hkv, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    seq, place = _of_token(cu, st["tokens"])
    q = torch.zeros((n, L, hq, d), device="cuda")
    q[seq, place] = st["q"].float()
    k = st["k_pages"][st["table"].long()].flatten(1, 2).float().permute(0, 2, 3, 1)  # [N, Hkv, D, C]
    v = st["v_pages"][st["table"].long()].flatten(1, 2).float().permute(0, 2, 1, 3)
    c = k.shape[-1]
    s = torch.matmul(q.permute(0, 2, 1, 3).reshape(n, hkv, hq // hkv * L, d), k)
    s = s.view(n, hq, L, c).mul_(1.0 / math.sqrt(d))
    start = (lens - (cu[1:] - cu[:-1])).view(n, 1, 1).long()
    key = torch.arange(c, device="cuda").view(1, 1, c)
    if case["kind"] == "tree":
        words = torch.zeros((n, L, st["ancestors"].shape[1]), dtype=torch.int64, device="cuda")
        words[seq, place] = st["ancestors"]
        node = (key - start).expand(n, L, c)
        at = node.clamp(0, L - 1)
        bit = (words.gather(2, at // 64) >> (at % 64)) & 1
        dead = ((node >= 0) & ((bit == 0) | (node >= L))) | (key >= lens.view(n, 1, 1))
        # A node's position: behind the cache by the number of its ancestors.
        bits = (words.unsqueeze(-1) >> torch.arange(64, device="cuda")) & 1
        deep = bits.sum((2, 3)) - 1  # [N, L]
        pos = start.squeeze(-1) + deep
        key_pos = torch.where(node >= 0, start + deep.unsqueeze(1).expand(n, L, L).gather(2, at), key)
    else:
        pos = start.squeeze(-1) + torch.arange(L, device="cuda")
        key_pos = key
        dead = (key > pos.unsqueeze(-1)) | (key >= lens.view(n, 1, 1))
    s, _ = _modified(s, case, st["slopes"], (pos.unsqueeze(-1) - key_pos).abs().float().unsqueeze(1))
    s = s.masked_fill_(dead.unsqueeze(1), -math.inf)
    top = s.amax(-1, keepdim=True).nan_to_num_(neginf=0.0)
    p = s.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(n, hkv, -1, c), v).view(n, hq, L, d) / torch.where(total > 0, total, 1.0)
    lse = (top + total.log()).squeeze(-1)
    return [o[seq, :, place].to(st["q"].dtype), lse[seq, :, place]]


def _draft(st):
    """The trees' ancestors and positions; the longest kept path of each, its length, and the target's
    token behind it."""
    cu, parents, longest = st["cu"], st["parents"], st["case"]["nodes"]
    n = cu.numel() - 1
    seq, place = _of_token(cu, parents.numel())
    reach = _reach(parents, cu, longest)
    deep = reach.sum(-1) - 1
    new = cu[1:] - cu[:-1]
    ancestors = _pack(reach)[seq, place]
    positions = ((st["kv_lens"] - new)[seq] + deep[seq, place]).to(torch.int32)
    above = cu[seq].long() + parents.clamp(min=0)
    fits = torch.zeros((n, longest), dtype=torch.bool, device="cuda")
    fits[seq, place] = (parents < 0) | (st["tokens"] == st["targets"][above])
    kept = (reach & ~fits.unsqueeze(1)).sum(-1) == 0
    kept &= torch.arange(longest, device="cuda") < new.view(n, 1)
    at = torch.arange(longest, device="cuda")
    best = torch.where(kept, deep * longest - at, -1 - longest).argmax(-1)
    chain = reach[torch.arange(n, device="cuda"), best]
    path = torch.where(chain, at, longest).sort(-1).values
    counts = chain.sum(-1).to(torch.int32)
    path = torch.where(path < longest, path, -1).to(torch.int32)
    return [ancestors, positions, path, counts, st["targets"][cu[:-1].long() + best]]


def _commit(st):
    ps, lens, table, path = st["case"]["page"], st["kv_lens"], st["table"].long(), st["path"].long()
    n, width = path.shape
    start = (lens - (st["cu"][1:] - st["cu"][:-1])).view(n, 1).long()
    at = torch.arange(width, device="cuda").view(1, width)
    live = at < st["counts"].view(n, 1)
    seq = torch.arange(n, device="cuda").view(n, 1).expand(n, width)
    # Where there is nothing to move, the sequence's first new slot moves to itself (as the first kept
    # node, the root, does).
    src, to = start + torch.where(live, path, 0), start + torch.where(live, at, 0)
    for pool in (st["k_pages"], st["v_pages"]):
        pool[table[seq, to // ps], to % ps] = pool[table[seq, src // ps], src % ps]
    return [(start.view(n) + st["counts"]).to(torch.int32), st["k_pages"], st["v_pages"]]


def run(st: dict):
    case, kind = st["case"], st["case"]["kind"]
    if not own:
        with torch.no_grad():
            if kind == "attend":
                return _attend(st)
            return _draft(st) if kind == "draft" else _commit(st) if kind == "commit" else _over_cache(st)
    from tasft_amd import kernels as K

    if kind == "attend":
        where = {"cu_seqlens": st["cu"], "max_seqlen": case["seq"]} if case["packed"] else {}
        if case["ragged"] and not case["packed"]:
            where = {"seq_lens": st["lens"]}
        scores = {"softcap": case["softcap"] or None, "alibi_slopes": st["slopes"], "prefix_lens": st["prefix"],
                  "causal": case["causal"]}
        if not case["grad"]:
            return list(K.dense_attention(st["q"], st["k"], st["v"], return_lse=True, **scores, **where))
        out = K.dense_attention(st["q"], st["k"], st["v"], **scores, **where)
        return [out.detach(), *torch.autograd.grad(out, (st["q"], st["k"], st["v"]), st["gout"])]
    if kind == "draft":
        tree = K.draft_tree(st["parents"], st["cu"], st["kv_lens"], max_nodes=case["nodes"])
        kept = K.accept_draft(st["parents"], st["tokens"], st["targets"], st["cu"], max_nodes=case["nodes"])
        return [tree.ancestors, tree.positions, kept.path, kept.counts, kept.next_tokens]
    if kind == "commit":
        lens = K.commit_draft_paged(st["k_pages"], st["v_pages"], st["table"], st["kv_lens"], st["cu"], st["path"],
                                    st["counts"])
        return [lens, st["k_pages"], st["v_pages"]]
    attn = K.BlockSparseFlashAttention(min_sparsity_for_speedup=0.0)
    out, lse = attn.forward_chunk_paged(st["q"], st["k_pages"], st["v_pages"], st["table"], st["kv_lens"], st["cu"],
                                        max_seqlen=st["max_seqlen"], softcap=case["softcap"] or None,
                                        alibi_slopes=st["slopes"], ancestors=st.get("ancestors"), return_lse=True)
    return [out, lse]


# --------------------------------------------------------------------------------- work
def work(case: dict) -> dict:
    kind, n = case["kind"], case["batch"]
    if kind == "draft":
        t = sum(_sizes(case, n, case["nodes"], max(1, case["nodes"] // 2)))
        words = -(-case["nodes"] // 64)
        # Parents, tokens and targets read; words, positions, paths and tokens written.
        return {"bytes": t * (4 + 8 + 8 + 8 * words + 4) + n * (4 * case["nodes"] + 20), "flops": t * words}
    hq, hkv, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    if kind == "attend":
        s = case["seq"]
        sizes = _sizes(case, n, s, max(1, s // 8))
        t = sum(sizes)
        # A prefix's length is anything up to the whole: a sixth of the square on average.
        pairs = sum(x * (x + 1) / 2 + (x * x / 6 if case["prefix"] else 0) if case["causal"] else x * x
                    for x in sizes)
        x = 2 * t * d * (2 * hq + 2 * hkv)  # q, k, v and the output
        if case["grad"]:
            return {"bytes": 2 * x, "flops": 14 * pairs * hq * d}
        return {"bytes": x + 4 * t * hq, "flops": 4 * pairs * hq * d}
    kv = case["kv"]
    # Ragged lengths spread evenly over the upper half; the first is the full one.
    mean_kv = kv if not case["ragged"] else (kv + (n - 1) * 0.75 * kv) / n
    new = case["chunk"] if kind == "chunk" else case["nodes"]
    mean_new = new if not case["ragged"] or new == 1 else (new + (n - 1) * 0.75 * new) / n
    if kind == "commit":
        return {"bytes": n * (case["depth"] / 2 + 1) * hkv * d * 8, "flops": n}
    t = n * mean_new
    if kind == "chunk":
        pairs = t * (mean_kv - (mean_new - 1) / 2)
    else:
        pairs = t * (mean_kv - mean_new + case["depth"] / 2 + 1)
    return {"bytes": n * mean_kv * hkv * d * 4 + 2 * t * hq * d * 2 + t * hq * 4, "flops": 4 * pairs * hq * d}


# ---------------------------------------------------------------------------- definition
def _scores64(q, k, case, slope, distance):
    s = q @ k.t().contiguous() / math.sqrt(case["head_dim"])
    if case["softcap"]:
        s = case["softcap"] * torch.tanh(s / case["softcap"])
    return s if slope is None else s - slope * distance


def exact(case: dict, seed: int):
    kind = case["kind"]
    if kind in ("draft", "commit"):
        return None  # whole numbers and moves: no computed numbers
    st = prepare(case, seed)
    grp = case["q_heads"] // case["kv_heads"]
    slopes = None if st["slopes"] is None else st["slopes"].double()
    cu = st["cu"].tolist()
    if kind == "attend":
        return _attend64(st, grp, slopes, cu)
    lens, ps = st["kv_lens"].tolist(), case["page"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(st["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    for i in range(case["batch"]):
        a, b, kv = cu[i], cu[i + 1], lens[i]
        p0 = kv - (b - a)
        pages = st["table"][i].long()
        k = st["k_pages"][pages].flatten(0, 1)[:kv].double()
        v = st["v_pages"][pages].flatten(0, 1)[:kv].double()
        key = torch.arange(kv, device="cuda")
        if kind == "tree":
            node = torch.arange(b - a, device="cuda")
            seen = ((st["ancestors"][a:b][:, node // 64] >> (node % 64)) & 1) == 1
            deep = seen.sum(1) - 1
            pos, key_pos = p0 + deep, torch.cat((key[:p0], p0 + deep))
            ok = torch.cat((torch.ones((b - a, p0), dtype=torch.bool, device="cuda"), seen), 1)
        else:
            pos, key_pos = p0 + torch.arange(b - a, device="cuda"), key
            ok = key_pos <= pos[:, None]
        far = (pos[:, None] - key_pos).abs().double()
        for h in range(case["q_heads"]):
            s = _scores64(st["q"][a:b, h].double(), k[:, h // grp], case, None if slopes is None else slopes[h], far)
            s = s.masked_fill(~ok, -math.inf)
            lse[a:b, h] = torch.logsumexp(s, -1)
            out[a:b, h] = torch.softmax(s, -1) @ v[:, h // grp]
    return [out, lse]


def _attend64(st, grp, slopes, cu):
    """A head at a time, its gradients by automatic differentiation of the definition."""
    case = st["case"]
    names = ("q", "k", "v", "gout")
    flat = st if case["packed"] else {x: st[x].transpose(1, 2).flatten(0, 1) for x in names}
    first = cu if case["packed"] else [i * case["seq"] for i in range(case["batch"])]
    flat = {x: flat[x].detach().double() for x in names}
    got = {x: torch.zeros_like(flat[x]) for x in ("q", "k", "v")}
    out = torch.zeros_like(flat["q"])
    lse = torch.full(out.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    for n, size in enumerate(st["sizes"]):
        a, b = first[n], first[n] + size
        at = torch.arange(size, device="cuda")
        ok = torch.ones((size, size), dtype=torch.bool, device="cuda")
        if case["causal"]:
            ok = at <= at[:, None]
            if st["prefix"] is not None:
                ok = ok | (at < st["prefix"][n])
        far = (at[:, None] - at).abs().double()
        for h in range(case["q_heads"]):
            q, k, v = (flat[x][a:b, j].clone().requires_grad_(case["grad"])
                       for x, j in (("q", h), ("k", h // grp), ("v", h // grp)))
            s = _scores64(q, k, case, None if slopes is None else slopes[h], far).masked_fill(~ok, -math.inf)
            o = torch.softmax(s, -1) @ v
            out[a:b, h] = o.detach()
            lse[a:b, h] = torch.logsumexp(s.detach(), -1)
            if case["grad"]:
                for x, j, y in zip("qkv", (h, h // grp, h // grp),
                                   torch.autograd.grad(o, (q, k, v), flat["gout"][a:b, h].contiguous())):
                    got[x][a:b, j] += y
    whole = [out, got["q"], got["k"], got["v"]] if case["grad"] else [out, lse]
    if case["packed"]:
        return whole
    return [x.unflatten(0, (case["batch"], case["seq"])).transpose(1, 2) for x in whole]
