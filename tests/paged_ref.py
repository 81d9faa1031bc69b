"""Plain 64-bit forms of the paged-cache operators, on the CPU, and their inputs.

``attention`` gives, next to output and log-sum-exp, what a bound on the kernel's error needs: the
softmax-weighted magnitude of V and the largest error of a score.
"""
from __future__ import annotations

import math

import torch


def half_step(dtype: torch.dtype) -> float:
    """The largest relative error of one rounding."""
    return torch.finfo(dtype).eps / 2


def make(lens, kv, hq, hkv, d, page, dtype, seed, spare_pages=2, pad=0, max_pages=None, scale=1.0):
    """q [T, Hq, D], pools, table [N, max_pages], kv_lens, cu on the CPU. Pages are shuffled; those
    that no sequence uses (and table entries behind a sequence's pages) hold NaN or are invalid."""
    g = torch.Generator().manual_seed(seed)
    n = len(lens)
    per = [max(1, math.ceil(max(x, 1) / page)) for x in kv]
    max_pages = max_pages or max(per) + 1
    num = sum(per) + spare_pages
    order = torch.randperm(num, generator=g)
    table = torch.full((n, max_pages), num + 5, dtype=torch.int32)  # out of the pool behind the used ones
    k = torch.full((num, page, hkv, d), float("nan"), dtype=dtype)
    v = k.clone()
    at = 0
    for i in range(n):
        ids = order[at:at + per[i]]
        at += per[i]
        table[i, :per[i]] = ids.to(torch.int32)
        kk = torch.randn((per[i] * page, hkv, d), generator=g) * scale
        vv = torch.randn((per[i] * page, hkv, d), generator=g)
        kk[kv[i]:] = float("nan")
        vv[kv[i]:] = float("inf")
        k[ids] = kk.to(dtype).view(per[i], page, hkv, d)
        v[ids] = vv.to(dtype).view(per[i], page, hkv, d)
    t = sum(lens) + pad
    q = torch.randn((t, hq, d), generator=g).mul_(scale).to(dtype)
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32)
    return q, k, v, table, torch.tensor(kv, dtype=torch.int32), cu


def gather(pool, table, n, length, page):
    """The first ``length`` slots of sequence n, [length, Hkv, D] in 64 bits."""
    s = torch.arange(length)
    return pool[table[n, s // page].long(), s % page].double()


def visible(start, length, kv, causal, mask, bs, h):
    """[length, kv] bool: which keys each token of a chunk sees (mask [Hq, R, NB] or None)."""
    pos = start + torch.arange(length)
    key = torch.arange(kv)
    ok = torch.ones(length, kv, dtype=torch.bool)
    if causal:
        ok &= key[None] <= pos[:, None]
    if mask is not None:
        rows = (torch.div(pos, bs, rounding_mode="floor") - math.floor(start / bs)).clamp(max=mask.shape[1] - 1)
        ok &= mask[h][rows][:, key // bs]
    return ok


def attention(q, k, v, table, kv_lens, cu, mask=None, bs=64, causal=True):
    """out, lse, weighted |v|, score error factor sum|q k| (largest seen), all [T, Hq, ...]."""
    t, hq, d = q.shape
    page, hkv = k.shape[1], k.shape[2]
    out = torch.zeros(t, hq, d, dtype=torch.float64)
    lse = torch.full((t, hq), -math.inf, dtype=torch.float64)
    mag = torch.zeros(t, hq, d, dtype=torch.float64)
    dot = torch.zeros(t, hq, dtype=torch.float64)
    for n in range(len(cu) - 1):
        a, b, kv = int(cu[n]), int(cu[n + 1]), int(kv_lens[n])
        if b == a or kv == 0:
            continue
        kk, vv = gather(k, table, n, kv, page), gather(v, table, n, kv, page)
        for h in range(hq):
            ok = visible(kv - (b - a), b - a, kv, causal, None if mask is None else mask[n], bs, h)
            qh, kh, vh = q[a:b, h].double(), kk[:, h // (hq // hkv)], vv[:, h // (hq // hkv)]
            s = (qh @ kh.t()) / math.sqrt(d)
            size = (qh.abs() @ kh.abs().t()) / math.sqrt(d)
            for i in range(b - a):
                see = ok[i]
                if not see.any():
                    continue
                p = torch.softmax(s[i, see], 0)
                out[a + i, h] = (p[:, None] * vh[see]).sum(0)
                mag[a + i, h] = (p[:, None] * vh[see].abs()).sum(0)
                lse[a + i, h] = torch.logsumexp(s[i, see], 0)
                dot[a + i, h] = size[i, see].max()
    return out, lse, mag, dot


def attention_bounds(out, lse, mag, dot, dtype, d, keys):
    """Largest errors of the kernel's output and log-sum-exp.

    A score is a sum of d products in fp32, off by at most (d + 3) 2^-24 of its absolute sum, and
    the exponential and its argument add 4 2^-24 (1 + |score|); the error of a weight is that
    relative, twice (its own and the sum's). P is rounded once (half a step u), the output once more.
    fp16 probabilities below its normal range are off by at most 2^-25 of a sum that is at least 1.
    """
    u = half_step(dtype)
    delta = ((d + 3) * dot + 4 * (1 + dot)) * 2.0 ** -24
    sums = keys * 2.0 ** -24  # fp32 sums over the keys
    o = (u + 2 * delta[..., None] + 2 * sums) * 1.01 * mag + u * out.abs() * 1.01
    if dtype == torch.float16:
        o = o + keys * 2.0 ** -25 * 8 + 2.0 ** -25
    return o, 2 * delta + sums + 4 * 2.0 ** -24 * (1 + lse.abs().nan_to_num(posinf=0.0, neginf=0.0))


def key_weights(q, k, table, kv_lens, cu, lse, scores, mask=None, bs=64, causal=True):
    """scores + weights [N, Hkv, cap] in 64 bits, the weights alone, and the largest score size."""
    t, hq, d = q.shape
    page, hkv = k.shape[1], k.shape[2]
    total = scores.double().clone()
    dot = 0.0
    for n in range(len(cu) - 1):
        a, b, kv = int(cu[n]), int(cu[n + 1]), int(kv_lens[n])
        if b == a or kv == 0:
            continue
        kk = gather(k, table, n, kv, page)
        for h in range(hq):
            g = h // (hq // hkv)
            ok = visible(kv - (b - a), b - a, kv, causal, None if mask is None else mask[n], bs, h)
            s = (q[a:b, h].double() @ kk[:, g].t()) / math.sqrt(d)
            dot = max(dot, float((q[a:b, h].double().abs() @ kk[:, g].abs().t()).max()) / math.sqrt(d))
            ok = ok & (lse[a:b, h, None] != -math.inf)
            total[n, g, :kv] += torch.where(ok, torch.exp(s - lse[a:b, h, None].double()), 0.0).sum(0)
    return total, dot


def rotate(x, positions, inv_freq, scale=1.0, interleaved=False, inverse=False):
    """x [..., D] in 64 bits, positions broadcast over x's dims but the last."""
    y = x.double().clone()
    half = inv_freq.numel()
    angle = positions.double()[..., None] * inv_freq.double()
    c, s = angle.cos() * scale, angle.sin() * (-scale if inverse else scale)
    if interleaved:
        a, b = x[..., 0:2 * half:2].double(), x[..., 1:2 * half:2].double()
        y[..., 0:2 * half:2], y[..., 1:2 * half:2] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., :half].double(), x[..., half:2 * half].double()
        y[..., :half], y[..., half:2 * half] = a * c - b * s, b * c + a * s
    return y


def rotate_bound(x, want, inv_freq, scale, interleaved, dtype):
    """One rounding of the result, and of the fp32 arithmetic: the reduced angle is rounded (2^-24
    of half a turn: 2^-22.3 rad), sine and cosine are off by 2^-23, the products and their sum by
    three more roundings of 2^-24 each; together under 2^-20 of |a| + |b|. The copied dims are exact."""
    half = inv_freq.numel()
    size = torch.zeros_like(want)
    y = x.double().abs()
    if interleaved:
        both = y[..., 0:2 * half:2] + y[..., 1:2 * half:2]
        size[..., 0:2 * half:2] = size[..., 1:2 * half:2] = both
    else:
        size[..., :half] = size[..., half:2 * half] = y[..., :half] + y[..., half:2 * half]
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    return half_step(dtype) * want.abs() * 1.001 + 2.0 ** -20 * abs(scale) * size + tiny * (size > 0)


def evict(k, v, table, kv_lens, scores, positions, budget, recent, sinks):
    """In place on copies, key by key: (k, v, kv_lens, scores, positions)."""
    k, v = k.clone(), v.clone()
    n, hkv, cap = scores.shape
    page = k.shape[1]
    s_out, p_out = torch.zeros_like(scores), torch.full_like(positions, -1)
    lens = kv_lens.clamp(0, cap)
    for i in range(n):
        length = int(lens[i])
        keep = min(length, budget)
        for h in range(hkv):
            pos, w = positions[i, h, :length].tolist(), scores[i, h, :length].tolist()
            newest = max(pos, default=0)

            def rank(j):
                guarded = pos[j] < sinks or pos[j] > newest - recent
                nan = math.isnan(w[j])
                return (not guarded, not nan, 0.0 if guarded or nan else -w[j], j)

            kept = sorted(sorted(range(length), key=rank)[:keep])
            held = set(kept)
            holes = [j for j in range(keep) if j not in held]
            movers = [j for j in kept if j >= keep]
            src = list(range(keep))
            for a, b in zip(holes, movers):
                src[a] = b
            pages = table[i].tolist()
            rows = [(pages[j // page], j % page) for j in range(length)]
            for a, b in zip(holes, movers):
                k[rows[a][0], rows[a][1], h] = k[rows[b][0], rows[b][1], h]
                v[rows[a][0], rows[a][1], h] = v[rows[b][0], rows[b][1], h]
            s_out[i, h, :keep], p_out[i, h, :keep] = scores[i, h, src], positions[i, h, src]
    return k, v, lens.clamp(max=budget), s_out, p_out
