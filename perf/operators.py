"""Serving a chunk of new tokens over a paged cache, as cases for timing and comparison.

The operators, in the order a serving step calls them: rotary positions (also as a training
step, with its gradients), new keys and values rotated into the pages of a cache, attention of
the chunk over that cache (dense or over a block mask), the attention weight every cached key
has received, and the eviction of the lightest keys. Head counts and lengths are those of
``perf/cases.py`` and ``tasft_amd.workloads`` (Llama-3-8B and Qwen-2.5-7B heads) and generic
ones beside them.

With ``own`` false ``run`` computes each operator in plain torch, in 32 bits (angles in 64);
with ``own`` true it calls ``tasft_amd``. ``exact`` is the definition in 64 bits.
"""
from __future__ import annotations

import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed() -> list[dict]:
    return [
        # A training step's rotation of a batch of long sequences, forward and backward, with
        # frequencies scaled for long contexts (Llama-3-8B heads).
        _case("rope", "rope_train", batch=4, seq=8192, scaling="llama3", base=500000.0, grad=True),
        # One short sequence of a model that rotates half of each head, interleaved: launches
        # and host time count.
        _case("rope", "rope_partial", batch=1, seq=1000, q_heads=16, kv_heads=16, head_dim=64,
              rotary=32, interleaved=True, scaling="yarn", dtype="fp16"),
        # One new token of each of 64 requests, rotated at a far position and written into the
        # pages (Qwen-2.5-7B heads).
        _case("append", "append_step", batch=64, chunk=1, kv=4100, ragged=True, q_heads=28, kv_heads=4,
              scaling="linear", far=1000000),
        # Four requests' chunks of a few thousand tokens, of different lengths.
        _case("append", "append_chunk", batch=4, chunk=4096, kv=8192, ragged=True, page=64, scaling="llama3",
              base=500000.0),
        # Chunked prefill of one long prompt: 2048 new tokens over a cache of 32768.
        _case("chunk", "chunk_long", batch=1, chunk=2048, kv=32768),
        # The same of several requests over block masks, a fifth of the blocks, a local band and
        # a first block kept (Qwen-2.5-7B heads).
        _case("chunk", "chunk_sparse", batch=4, chunk=2048, kv=16384, ragged=True, q_heads=28, kv_heads=4,
              page=64, keep=0.2),
        # One new token of each of 64 requests of different lengths over their whole caches.
        _case("chunk", "chunk_decode", batch=64, chunk=1, kv=16384, ragged=True),
        # Five drafted tokens of each of 8 requests checked at once, heads of 64 in fp16.
        _case("chunk", "chunk_verify", batch=8, chunk=5, kv=4001, ragged=True, q_heads=16, kv_heads=16,
              head_dim=64, page=32, dtype="fp16"),
        # The weights that the last 256 tokens of two long prompts give every cached key.
        _case("weights", "weights_window", batch=2, chunk=256, kv=32768, ragged=True),
        # The same for one new token of each of 32 requests at their budget.
        _case("weights", "weights_step", batch=32, chunk=1, kv=4097, page=32, dtype="fp16", q_heads=28, kv_heads=4),
        # Long prompts cut to a budget of 4096 keys per head.
        _case("evict", "evict_prompt", batch=4, kv=32768, budget=4096, recent=256, sinks=4, ragged=True),
        # 64 requests, a few tokens over their budget.
        _case("evict", "evict_step", batch=64, kv=1040, budget=1024, recent=64, sinks=4, page=32, head_dim=64),
    ]


def draw(rng) -> dict:
    heads, kv_heads = rng.choice([(32, 8), (28, 4), (16, 16), (8, 2), (12, 4)])
    f = {"q_heads": heads, "kv_heads": kv_heads, "head_dim": rng.choice([128, 128, 64]),
         "dtype": rng.choice(["bf16", "bf16", "fp16"]), "page": rng.choice([8, 16, 16, 32, 64, 128])}
    turn = {"scaling": rng.choice(["none", "linear", "llama3", "yarn"]), "base": rng.choice([10000.0, 500000.0]),
            "interleaved": rng.random() < 0.4, "rotary": rng.choice([0, 0, 16, 32, 64])}

    def length(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["rope", "append", "chunk", "chunk", "chunk", "weights", "evict"])
    if kind == "rope":
        seq = length(1, 8192)
        return _case(kind, None, batch=rng.randint(1, max(1, min(8, 32768 // seq))), seq=seq,
                     grad=rng.random() < 0.5, **f, **turn)
    if kind == "append":
        kv = length(16, 8192)
        batch = rng.randint(1, max(1, min(64, 65536 // kv)))
        return _case(kind, None, batch=batch, chunk=length(1, min(kv, max(1, 16384 // batch))), kv=kv,
                     ragged=rng.random() < 0.7, far=rng.choice([0, 0, 100000]), **f, **turn)
    if kind == "evict":
        kv = length(100, 32768)
        budget = min(kv, length(50, 8192))
        return _case(kind, None, batch=rng.randint(1, max(1, min(64, 131072 // kv))), kv=kv, budget=budget,
                     recent=rng.randint(0, budget // 2), sinks=rng.randint(0, min(8, budget // 4)),
                     ragged=rng.random() < 0.5, **f)
    kv = length(50, 32768)
    chunk = min(kv, rng.choice([1, length(2, 16), length(16, 2048)]))
    most = min(64, 500000 // kv, (1 << 26) // (chunk * kv))
    keep = rng.choice([0.0, 0.0, round(rng.uniform(0.1, 0.4), 3)])
    return _case(kind, None, batch=rng.randint(1, max(1, most)), chunk=chunk, kv=kv, ragged=rng.random() < 0.7,
                 keep=keep, block=rng.choice([64, 64, 32, 128]), **f)


def _case(kind, name, **fields):
    case = {"kind": kind, "q_heads": 32, "kv_heads": 8, "head_dim": 128, "dtype": "bf16"}
    if kind in ("rope", "append"):
        case.update(scaling="none", base=10000.0, interleaved=False, rotary=0)
    if kind == "rope":
        case.update(grad=False)
    else:
        case.update(page=16, ragged=False)
    if kind == "append":
        case.update(far=0)
    if kind in ("chunk", "weights"):
        case.update(keep=0.0, block=64)
    case.update(fields)
    if kind == "rope":
        case.pop("page", None)
    if name is not None:
        case["name"] = name
    return case


# ------------------------------------------------------------------------------- inputs
def _randn(g, shape, dtype):
    return torch.randn(shape, generator=g, device="cuda", dtype=dtype)


def _frequencies(case):
    """Inverse frequencies (64 bits) and the factor on cosine and sine, as a model's config
    gives them."""
    d = case["rotary"] or case["head_dim"]
    f = 1.0 / case["base"] ** (torch.arange(0, d, 2, dtype=torch.float64) / d)
    factor, old = 8.0, 8192
    if case["scaling"] == "linear":
        return f / factor, 1.0
    if case["scaling"] == "llama3":
        # Long wavelengths are stretched, short ones kept, those between blended.
        turns = old * f / (2 * math.pi)
        smooth = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return f / factor * (1 - smooth) + f * smooth, 1.0
    if case["scaling"] == "yarn":
        def dim_at(rotations):
            return d * math.log(old / (rotations * 2 * math.pi)) / (2 * math.log(case["base"]))
        low, high = max(0, math.floor(dim_at(32))), min(d - 1, math.ceil(dim_at(1)))
        ramp = ((torch.arange(d // 2, dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0, 1)
        return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1.0
    return f, 1.0


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind, dt = case["kind"], _DTYPES[case["dtype"]]
    hq, hkv, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    st = {"case": case}
    if kind in ("rope", "append"):
        st["inv_freq"], st["factor"] = _frequencies(case)
        st["inv_freq"] = st["inv_freq"].to("cuda")
    if kind == "rope":
        b, s = case["batch"], case["seq"]
        # Projections give [B, S, H, D]; attention takes the transposed view.
        st["q"] = _randn(g, (b, s, hq, d), dt).transpose(1, 2)
        st["k"] = _randn(g, (b, s, hkv, d), dt).transpose(1, 2)
        st["positions"] = torch.arange(s, device="cuda") + torch.randint(0, 4096, (b, 1), generator=g, device="cuda")
        if case["grad"]:
            st["gq"], st["gk"] = _randn(g, (b, hq, s, d), dt), _randn(g, (b, hkv, s, d), dt)
            st["q"].requires_grad_(True)
            st["k"].requires_grad_(True)
        return st
    n, ps, kv = case["batch"], case["page"], case["kv"]
    pages = -(-kv // ps)
    st["table"] = torch.randperm(n * pages, generator=g, device="cuda").view(n, pages).to(torch.int32)
    st["k_pages"] = _randn(g, (n * pages, ps, hkv, d), dt)
    st["v_pages"] = _randn(g, (n * pages, ps, hkv, d), dt)
    lens = torch.full((n,), kv, dtype=torch.int32, device="cuda")
    if case["ragged"]:
        lens = torch.randint(kv // 2 + 1, kv + 1, (n,), generator=g, device="cuda", dtype=torch.int32)
        lens[0] = kv
    st["kv_lens"] = lens
    if kind == "evict":
        cap = pages * ps
        # What accumulated weights look like: a few heavy keys, a long tail.
        st["scores"] = torch.rand((n, hkv, cap), generator=g, device="cuda").pow_(8) * 4
        # Positions as earlier evictions leave them: gaps, and no order among the older slots.
        pos = torch.randperm(4 * cap, generator=g, device="cuda")[:cap].sort().values
        st["positions"] = pos.to(torch.int32).expand(n, hkv, cap).contiguous()
        old = cap // 2
        shuffled = torch.rand((n, hkv, old), generator=g, device="cuda").argsort(-1)
        st["positions"][:, :, :old] = st["positions"][:, :, :old].gather(2, shuffled)
        return st
    chunk = case["chunk"]
    # The engine knows the chunks' lengths on the host too. They go by the case alone (and fit
    # the shortest cache above), so that outputs of every seed have one shape.
    sizes = [chunk] * n
    if case["ragged"]:
        rng = random.Random(chunk * 1000003 + kv)
        sizes = [chunk] + [rng.randint(min(chunk // 2 + 1, kv // 2 + 1), min(chunk, kv // 2 + 1)) for _ in range(n - 1)]
    t = sum(sizes)
    st["tokens"], st["max_seqlen"] = t, chunk
    new = torch.tensor(sizes, dtype=torch.int32, device="cuda")
    st["cu"] = torch.cat((new.new_zeros(1), new.cumsum(0))).to(torch.int32)
    st["q"] = _randn(g, (t, hq, d), dt)
    if kind == "append":
        st["k"], st["v"] = _randn(g, (t, hkv, d), dt), _randn(g, (t, hkv, d), dt)
        st["positions"] = None
        if case["far"]:
            st["positions"] = torch.randint(0, case["far"], (t,), generator=g, device="cuda")
        st["slots"] = torch.zeros((n, hkv, pages * ps), dtype=torch.int32, device="cuda")
        return st
    bs = case["block"]
    st["mask"] = None
    if case["keep"]:
        rows, nb = (st["max_seqlen"] + bs - 2) // bs + 1, -(-pages * ps // bs)
        m = torch.rand((n, hq, rows, nb), generator=g, device="cuda") < case["keep"]
        # The block of each row's own tokens, the one before it and the first are kept.
        own_block = ((lens - new) // bs).view(n, 1) + torch.arange(rows, device="cuda")
        j = torch.arange(nb, device="cuda")
        near = (j <= own_block[..., None]) & (j >= own_block[..., None] - 1)
        st["mask"] = m | near[:, None] | (j == 0)
    if kind == "weights":
        # What the attention before it returned.
        st["lse"] = _log_sums(st)
        # As much weight from earlier chunks as this one brings.
        st["scores"] = torch.rand((n, hkv, pages * ps), generator=g, device="cuda") * (2 * chunk * hq / (hkv * kv))
    return st


# ----------------------------------------------------------------------- the plain forms
def _turn(x, positions, inv_freq, factor, interleaved, back=False):
    """``x`` [..., D] rotated by ``positions`` (broadcast over the dims before the last) times
    the frequencies, in 32 bits; angles in 64."""
    angle = positions.double().unsqueeze(-1) * inv_freq
    cos, sin = (angle.cos() * factor).float(), (angle.sin() * factor).float()
    if back:
        sin = -sin
    r = 2 * inv_freq.numel()
    y = x.float()
    if interleaved:
        a, b = y[..., 0:r:2], y[..., 1:r:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = y[..., :r // 2], y[..., r // 2:r]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, y[..., r:]), -1).to(x.dtype)


def _sequence_of(cu, tokens):
    """Each token's sequence, and its place in it."""
    at = torch.arange(tokens, device=cu.device)
    seq = torch.searchsorted(cu[1:].long(), at, right=True)
    return seq, at - cu[seq]


def _scores(st):
    """Masked, scaled scores [N, Hkv, G, L, C] in 32 bits of the padded chunks, and each
    token's sequence and place."""
    case, cu, lens = st["case"], st["cu"], st["kv_lens"]
    n, ps, L = case["batch"], case["page"], st["max_seqlen"]
    hq, hkv, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    seq, place = _sequence_of(cu, st["tokens"])
    q = torch.zeros((n, L, hq, d), device="cuda")
    q[seq, place] = st["q"].float()
    k = st["k_pages"][st["table"].long()].flatten(1, 2).float().permute(0, 2, 3, 1)  # [N, Hkv, D, C]
    c = k.shape[-1]
    s = torch.matmul(q.permute(0, 2, 1, 3).reshape(n, hkv, hq // hkv * L, d), k)
    s = s.view(n, hq, L, c).mul_(1.0 / math.sqrt(d))
    start = (lens - (cu[1:] - cu[:-1])).view(n, 1).long()
    pos = start + torch.arange(L, device="cuda")
    key = torch.arange(c, device="cuda")
    dead = (key > pos[..., None]) | (key >= lens.view(n, 1, 1))
    if st["mask"] is not None:
        bs = case["block"]
        row = (torch.div(pos, bs, rounding_mode="floor") - torch.div(start, bs, rounding_mode="floor"))
        row = row.clamp(max=st["mask"].shape[2] - 1).view(n, 1, L, 1).expand(-1, hq, -1, st["mask"].shape[3])
        off = ~st["mask"].gather(2, row).repeat_interleave(bs, dim=3)[..., :c]
        dead = off | dead[:, None]
    else:
        dead = dead[:, None]
    return s.masked_fill_(dead, -math.inf), seq, place


def _log_sums(st):
    """log sum exp of every token's scores, [T, Hq]."""
    s, seq, place = _scores(st)
    return torch.logsumexp(s, -1)[seq, :, place].contiguous()


def _plain(st):
    case, kind = st["case"], st["case"]["kind"]
    n, hq, hkv, d = case["batch"], case["q_heads"], case["kv_heads"], case["head_dim"]
    if kind == "rope":
        with torch.no_grad():
            pos = st["positions"].unsqueeze(1)
            turn = (pos, st["inv_freq"], st["factor"], case["interleaved"])
            out = [_turn(st["q"], *turn), _turn(st["k"], *turn)]
            if case["grad"]:
                out += [_turn(st["gq"], *turn, back=True), _turn(st["gk"], *turn, back=True)]
            return out
    ps, lens, table = case["page"], st["kv_lens"], st["table"]
    if kind == "append":
        seq, place = _sequence_of(st["cu"], st["tokens"])
        slot = (lens - (st["cu"][1:] - st["cu"][:-1]))[seq] + place
        pos = slot if st["positions"] is None else st["positions"]
        turn = (pos.unsqueeze(1), st["inv_freq"], st["factor"], case["interleaved"])
        page = table[seq, torch.div(slot, ps, rounding_mode="floor")].long()
        st["k_pages"][page, slot % ps] = _turn(st["k"], *turn)
        st["v_pages"][page, slot % ps] = st["v"]
        st["slots"][seq, :, slot] = pos.to(torch.int32).unsqueeze(1)
        return [_turn(st["q"], *turn), st["k_pages"], st["v_pages"], st["slots"]]
    if kind == "chunk":
        s, seq, place = _scores(st)
        top = s.amax(-1, keepdim=True).nan_to_num_(neginf=0.0)
        p = s.sub_(top).exp_()
        total = p.sum(-1, keepdim=True)
        v = st["v_pages"][table.long()].flatten(1, 2).float().permute(0, 2, 1, 3)  # [N, Hkv, C, D]
        o = torch.matmul(p.view(n, hkv, -1, v.shape[2]), v).view(n, hq, -1, d)
        o = o / torch.where(total > 0, total, 1.0)
        lse = (top + total.log()).squeeze(-1)
        return [o[seq, :, place].to(st["q"].dtype), lse[seq, :, place]]
    if kind == "weights":
        s, seq, place = _scores(st)
        lse = torch.zeros((n, s.shape[2], hq), device="cuda")
        lse[seq, place] = st["lse"]
        live = torch.zeros((n, s.shape[2], 1), device="cuda")
        live[seq, place] = 1.0
        p = s.sub_(lse.transpose(1, 2).unsqueeze(-1)).exp_().mul_(live.transpose(1, 2).unsqueeze(-1))
        return [st["scores"] + p.view(n, hkv, -1, p.shape[-1]).sum(2)]
    # Eviction: the protected keys first, then by weight, ties to the lowest slot.
    scores, pos, budget = st["scores"], st["positions"], case["budget"]
    cap = scores.shape[-1]
    slot = torch.arange(cap, device="cuda")
    valid = (slot < lens.view(n, 1, 1)).expand_as(scores)
    newest = pos.masked_fill(~valid, -1).amax(-1, keepdim=True)
    guarded = (pos < case["sinks"]) | (pos > newest - case["recent"])
    key = scores.masked_fill(guarded, math.inf).masked_fill(~valid, -math.inf)
    order = key.sort(dim=-1, descending=True, stable=True).indices
    keep_n = lens.clamp(max=budget)
    kept = torch.zeros_like(valid).scatter_(2, order, slot < keep_n.view(n, 1, 1).expand_as(scores))
    # The kept keys behind the budget fill the holes before it, both in slot order.
    front = slot < keep_n.view(n, 1, 1)
    moving, hole = kept & ~front, front & ~kept
    by_rank = torch.full((n, hkv, cap + 1), cap, device="cuda")
    by_rank.scatter_(2, torch.where(moving, moving.cumsum(-1) - 1, cap), slot.expand_as(scores))
    src = torch.where(hole, by_rank.gather(2, (hole.cumsum(-1) - 1).clamp(min=0)), slot)
    src = torch.where(front, src, slot)
    head = torch.arange(hkv, device="cuda").view(1, hkv, 1)
    at = table.long()[torch.arange(n, device="cuda").view(n, 1, 1), torch.div(src, ps, rounding_mode="floor")]
    to = table.long()[:, torch.div(slot, ps, rounding_mode="floor")].unsqueeze(1).expand_as(at)
    for pool in (st["k_pages"], st["v_pages"]):
        pool[to, (slot % ps).expand_as(at), head] = pool[at, src % ps, head]
    return [keep_n, torch.where(front, scores.gather(2, src), 0.0), torch.where(front, pos.gather(2, src), -1),
            st["k_pages"], st["v_pages"]]


def run(st: dict):
    if not own:
        return _plain(st)
    from tasft_amd import kernels as K

    case, kind = st["case"], st["case"]["kind"]
    if kind == "rope":
        q, k = K.apply_rotary(st["q"], st["k"], st["positions"], st["inv_freq"], interleaved=case["interleaved"],
                              scale=st["factor"])
        if not case["grad"]:
            return [q, k]
        gq, gk = torch.autograd.grad((q, k), (st["q"], st["k"]), (st["gq"], st["gk"]))
        return [q.detach(), k.detach(), gq, gk]
    if kind == "append":
        q = K.append_paged(st["q"], st["k"], st["v"], st["k_pages"], st["v_pages"], st["table"], st["kv_lens"],
                           st["cu"], st["inv_freq"], positions=st["positions"], interleaved=case["interleaved"],
                           scale=st["factor"], slot_positions=st["slots"])
        return [q, st["k_pages"], st["v_pages"], st["slots"]]
    if kind == "chunk":
        attn = K.BlockSparseFlashAttention(block_size=case["block"], min_sparsity_for_speedup=0.0)
        out, lse = attn.forward_chunk_paged(st["q"], st["k_pages"], st["v_pages"], st["table"], st["kv_lens"],
                                            st["cu"], st["mask"], max_seqlen=st["max_seqlen"], return_lse=True)
        return [out, lse]
    if kind == "weights":
        return [K.accumulate_key_weights(st["q"], st["k_pages"], st["table"], st["kv_lens"], st["cu"], st["lse"],
                                         st["scores"], block_mask=st["mask"], block_size=case["block"],
                                         max_seqlen=st["max_seqlen"])]
    lens, scores, pos = K.evict_paged(st["k_pages"], st["v_pages"], st["table"], st["kv_lens"], st["scores"],
                                      st["positions"], case["budget"], recent=case["recent"], sinks=case["sinks"])
    return [lens, scores, pos, st["k_pages"], st["v_pages"]]


# --------------------------------------------------------------------------------- work
def work(case: dict) -> dict:
    kind = case["kind"]
    hq, hkv, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    if kind == "rope":
        x = case["batch"] * case["seq"] * (hq + hkv) * d
        passes = 2 if case["grad"] else 1
        return {"bytes": passes * x * 4, "flops": passes * x * 3}
    n, kv = case["batch"], case["kv"]
    # Ragged lengths spread evenly over the upper half; the first is the full one.
    mean_kv = kv if not case["ragged"] else (kv + (n - 1) * 0.75 * kv) / n
    if kind == "evict":
        per = min(mean_kv, case["budget"])
        moved = per * (1 - per / mean_kv)
        cap = -(-kv // case["page"]) * case["page"]
        return {"bytes": n * hkv * (8 * mean_kv + 8 * cap + moved * d * 8), "flops": n * hkv * 4 * mean_kv}
    chunk = case["chunk"]
    mean_new = chunk if not case["ragged"] or chunk == 1 else (chunk + (n - 1) * 0.75 * chunk) / n
    t = n * mean_new
    if kind == "append":
        return {"bytes": t * (2 * hq + 4 * hkv) * d * 2 + t * hkv * 4, "flops": t * (hq + hkv) * d * 3}
    pairs = n * mean_new * (mean_kv - (mean_new - 1) / 2)
    read = n * mean_kv
    if case["keep"]:
        # Kept blocks: the row's own, the one before and the first, and a share of the rest.
        bs = case["block"]
        fixed = min(mean_kv, 2.5 * bs)
        pairs = n * mean_new * (fixed + case["keep"] * max(0.0, mean_kv - mean_new / 2 - fixed))
        rows = (hq // hkv) * max(1.0, mean_new / bs)
        read = n * min(mean_kv, fixed + (1 - (1 - case["keep"]) ** rows) * max(0.0, mean_kv - fixed))
    if kind == "chunk":
        return {"bytes": read * hkv * d * 4 + 2 * t * hq * d * 2 + t * hq * 4, "flops": 4 * pairs * hq * d}
    cap = -(-kv // case["page"]) * case["page"]
    return {"bytes": read * hkv * d * 2 + t * hq * (2 * d + 4) + 2 * n * hkv * cap * 4,
            "flops": 2 * pairs * hq * d}


# ---------------------------------------------------------------------------- definition
def _turn64(x, positions, inv_freq, factor, interleaved, sign=1.0):
    """Pairs as complex numbers times factor * exp(i sign position frequency)."""
    x = x.detach().double()
    half = inv_freq.numel()
    angle = sign * positions.double()[..., None] * inv_freq
    w = torch.polar(torch.full_like(angle, factor), angle)
    y = x.clone()
    if interleaved:
        z = torch.complex(x[..., 0:2 * half:2], x[..., 1:2 * half:2]) * w
        y[..., 0:2 * half:2], y[..., 1:2 * half:2] = z.real, z.imag
    else:
        z = torch.complex(x[..., :half], x[..., half:2 * half]) * w
        y[..., :half], y[..., half:2 * half] = z.real, z.imag
    return y


def _allowed(st, i, h, start, length, kv, lo, hi):
    """Which of the keys 0 .. kv-1 the chunk's tokens lo .. hi-1 of sequence i see, head h."""
    pos = start + torch.arange(lo, hi, device="cuda")
    ok = torch.arange(kv, device="cuda")[None, :] <= pos[:, None]
    if st["mask"] is not None:
        bs = st["case"]["block"]
        rows = pos // bs - start // bs
        ok &= st["mask"][i, h][rows][:, torch.arange(kv, device="cuda") // bs]
    return ok


def exact(case: dict, seed: int):
    st = prepare(case, seed)
    kind = case["kind"]
    hq, hkv, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    if kind == "rope":
        turn = (st["positions"][:, None, :], st["inv_freq"], st["factor"], case["interleaved"])
        out = [_turn64(st["q"], *turn), _turn64(st["k"], *turn)]
        if case["grad"]:
            out += [_turn64(st["gq"], *turn, sign=-1.0), _turn64(st["gk"], *turn, sign=-1.0)]
        return out
    n, ps, cu, lens = case["batch"], case["page"], st.get("cu"), st["kv_lens"].tolist()
    if kind == "append":
        kp, vp = st["k_pages"].double(), st["v_pages"].double()
        cu = cu.tolist()
        qs = []
        for i in range(n):
            a, b = cu[i], cu[i + 1]
            slot = torch.arange(lens[i] - (b - a), lens[i], device="cuda")
            pos = slot if st["positions"] is None else st["positions"][a:b]
            turn = (pos[:, None], st["inv_freq"], st["factor"], case["interleaved"])
            page = st["table"][i].long()[slot // ps]
            kp[page, slot % ps] = _turn64(st["k"][a:b], *turn)
            vp[page, slot % ps] = st["v"][a:b].double()
            qs.append(_turn64(st["q"][a:b], *turn))
        return [torch.cat(qs), kp, vp, None]
    if kind == "evict":
        return None  # moves and comparisons: no computed numbers
    cu, grp = cu.tolist(), hq // hkv
    out = torch.zeros((st["tokens"], hq, d), dtype=torch.float64, device="cuda")
    lse = torch.full((st["tokens"], hq), -math.inf, dtype=torch.float64, device="cuda")
    sums = None if kind == "chunk" else st["scores"].double()
    for i in range(n):
        a, length, kv = cu[i], cu[i + 1] - cu[i], lens[i]
        pages = st["table"][i].long()
        k = st["k_pages"][pages].flatten(0, 1)[:kv].double()
        v = st["v_pages"][pages].flatten(0, 1)[:kv].double() if kind == "chunk" else None
        step = max(1, (1 << 27) // kv)
        for h in range(hq):
            kh = k[:, h // grp].t().contiguous()
            for lo in range(0, length, step):
                hi = min(length, lo + step)
                s = (st["q"][a + lo:a + hi, h].double() @ kh) / math.sqrt(d)
                s.masked_fill_(~_allowed(st, i, h, kv - length, length, kv, lo, hi), -math.inf)
                if kind == "chunk":
                    lse[a + lo:a + hi, h] = torch.logsumexp(s, -1)
                    out[a + lo:a + hi, h] = torch.softmax(s, -1) @ v[:, h // grp]
                else:
                    sums[i, h // grp, :kv] += torch.exp(s - st["lse"][a + lo:a + hi, h, None].double()).sum(0)
    return [out, lse] if kind == "chunk" else [sums]
