"""Attention over a paged cache with capped and biased scores or a tree of new tokens, and the plans of
such trees, in 64 bits and node by node on the CPU."""
from __future__ import annotations

import math
import random

import torch

from paged_ref import gather, half_step, visible


def random_parents(sizes, seed, roots=0.05, deep=0.5):
    """Parents of a tree (or several) of each sequence's nodes."""
    rng = random.Random(seed)
    out = []
    for n in sizes:
        for i in range(n):
            if i == 0 or rng.random() < roots:
                out.append(-1)
            else:
                out.append(i - 1 if rng.random() < deep else rng.randrange(i))
    return out


def chains(parents, cu):
    """For each node its ancestors and itself, from the root down, as indices within the sequence."""
    out = []
    for a, b in zip(cu[:-1], cu[1:]):
        rows = []
        for i in range(b - a):
            p = parents[a + i]
            rows.append((rows[p] if 0 <= p < i else []) + [i])
        out += rows
    return out


def bits(rows, words):
    """[T, words] int64 of lists of nodes."""
    t = torch.zeros((len(rows), words), dtype=torch.int64)
    for r, nodes in enumerate(rows):
        value = [0] * words
        for a in nodes:
            value[a // 64] |= 1 << (a % 64)
        t[r] = torch.tensor([v - (1 << 64) if v >> 63 else v for v in value])
    return t


def accept(parents, tokens, targets, cu, first, most):
    path, counts, following = [], [], []
    for n, (a, b) in enumerate(zip(cu[:-1], cu[1:])):
        kept = []
        for i, row in enumerate(chains(parents[a:b], [0, b - a])):
            ok = first is None or tokens[a + row[0]] == first[n]
            ok = ok and all(tokens[a + j] == targets[a + i0] for i0, j in zip(row, row[1:]))
            if ok:
                kept.append((-len(row), i, row))
        row = min(kept)[2] if kept else []
        path.append(row + [-1] * (most - len(row)))
        counts.append(len(row))
        following.append(targets[a + row[-1]] if row else (-1 if first is None else first[n]))
    return path, counts, following


def attention(q, k, v, table, kv_lens, cu, *, cap=0.0, slopes=None, rows=None, mask=None, bs=64, causal=True, slots=None):
    """out, lse and their bounds; ``rows``: the chains of a tree's nodes; ``slots``: keys behind are not
    there.

    A score's error: D products in fp32 (at most (D + 3) 2^-24 of their absolute sum), 4 2^-24 of its size and
    the bias's, with a cap 2^-21 of the cap (from 128 on 2^-19 of the score). The largest in a row is delta;
    a weight is off by 2 delta and the fp32 sums (keys 2^-24) twice; P and the output are rounded once each.
    """
    t, hq, d = q.shape
    page, hkv = k.shape[1], k.shape[2]
    u = half_step(q.dtype)
    out, e_out = torch.zeros(2, t, hq, d, dtype=torch.float64)
    lse, e_lse = torch.full((t, hq), -math.inf, dtype=torch.float64), torch.zeros(t, hq, dtype=torch.float64)
    for n in range(len(cu) - 1):
        a, b, full = int(cu[n]), int(cu[n + 1]), int(kv_lens[n])
        kv = full if slots is None else min(full, slots)
        if b == a or kv <= 0:
            continue
        p0 = full - (b - a)
        kk, vv = gather(k, table, n, kv, page), gather(v, table, n, kv, page)
        key_pos = torch.arange(kv)
        pos = p0 + torch.arange(b - a)
        if rows is not None:
            pos = p0 + torch.tensor([len(r) - 1 for r in rows[a:b]])
            key_pos = torch.cat((torch.arange(max(p0, 0)), pos[max(-p0, 0):]))[:kv]
        for h in range(hq):
            if rows is None:
                ok = visible(p0, b - a, kv, causal, None if mask is None else mask[n], bs, h)
            else:
                ok = torch.zeros(b - a, kv, dtype=torch.bool)
                ok[:, :max(p0, 0)] = True
                for i, r in enumerate(rows[a:b]):
                    ok[i, [p0 + j for j in r if 0 <= p0 + j < kv]] = True
            qh, kh, vh = q[a:b, h].double(), kk[:, h // (hq // hkv)], vv[:, h // (hq // hkv)]
            s = qh @ kh.t() / math.sqrt(d)
            size = qh.abs() @ kh.abs().t() / math.sqrt(d)
            if cap:
                s = cap * torch.tanh(s / cap)
            far = torch.zeros_like(s)
            if slopes is not None:
                far = float(slopes[h]) * (pos[:, None] - key_pos[None]).abs().double()
                s = s - far
            err = ((d + 3) * size + 4 * (1 + size + far)) * 2.0 ** -24
            if cap:
                err = err + (cap * 2.0 ** -21 if cap <= 128 else s.abs() * 2.0 ** -19 + 2.0 ** -21)
            for i in range(b - a):
                see = ok[i]
                if not see.any():
                    continue
                p = torch.softmax(s[i, see], 0)
                delta, sums = float(err[i, see].max()), kv * 2.0 ** -24
                o = (p[:, None] * vh[see]).sum(0)
                mag = (p[:, None] * vh[see].abs()).sum(0)
                l = torch.logsumexp(s[i, see], 0)
                out[a + i, h], lse[a + i, h] = o, l
                e_out[a + i, h] = (u + 2 * delta + 2 * sums) * 1.01 * mag + u * o.abs() * 1.01
                e_lse[a + i, h] = 2 * delta + sums + 4 * 2.0 ** -24 * (1 + l.abs())
                if q.dtype == torch.float16:
                    e_out[a + i, h] += kv * 2.0 ** -25 * 8 + 2.0 ** -25
    return out, lse, e_out, e_lse


def commit(k, v, table, kv_lens, cu, path, counts, positions=None):
    """In place on copies, token by token: (k, v, kv_lens, positions)."""
    k, v = k.clone(), v.clone()
    positions = None if positions is None else positions.clone()
    page, out = k.shape[1], []
    for n in range(len(cu) - 1):
        start = int(kv_lens[n]) - (int(cu[n + 1]) - int(cu[n]))
        where = lambda s: (int(table[n, s // page]), s % page)  # noqa: E731
        for j in range(int(counts[n])):
            src, to = start + int(path[n][j]), start + j
            k[where(to)], v[where(to)] = k[where(src)].clone(), v[where(src)].clone()
            if positions is not None:
                positions[n, :, to] = positions[n, :, src]
        out.append(start + int(counts[n]))
    return k, v, torch.tensor(out, dtype=torch.int32), positions
