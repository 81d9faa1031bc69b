"""Chunk attention over a paged cache and the key weights, against the 64-bit form."""
from __future__ import annotations

import math

import pytest
import torch

import paged_ref as ref
from helpers import require_gpu
from tasft_amd import _native
from tasft_amd.kernels import BlockSparseFlashAttention, accumulate_key_weights

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16

# lens, kv_lens, Hq, Hkv, D, page, dtype, causal
CASES = [
    ([1], [1], 1, 1, 128, 16, BF, True),
    ([1], [1], 4, 4, 64, 8, HF, True),
    ([1, 1, 1], [65, 700, 64], 8, 2, 128, 16, BF, True),
    ([1, 1], [333, 20], 28, 4, 128, 32, HF, True),
    ([1, 1], [130, 513], 16, 1, 64, 128, BF, True),
    ([1], [300], 40, 1, 128, 16, BF, True),            # 40 query heads of one KV head
    ([5, 3, 0, 8], [700, 64, 40, 8], 8, 2, 128, 16, BF, True),
    ([5, 4], [129, 1000], 16, 16, 64, 32, HF, True),
    ([2, 1, 7], [64, 65, 71], 6, 2, 128, 8, HF, True),
    ([70, 1, 33], [70, 500, 300], 8, 2, 128, 16, BF, True),
    ([130, 200], [130, 515], 4, 2, 64, 64, BF, True),
    ([129], [1000], 7, 1, 128, 256, HF, True),
    ([40, 64], [200, 64], 4, 1, 128, 16, BF, False),
    ([3, 1], [77, 400], 8, 8, 64, 8, HF, False),
    ([9, 70], [4, 50], 4, 2, 128, 16, BF, True),       # fewer cached keys than new tokens
    ([300], [900], 2, 1, 64, 8, HF, True),
]


def _put(t, dev):
    return [x.to(dev) for x in t]


def _mask(case, seed, bs, density, rows=None, blocks=None):
    lens, kv, hq = case[0], case[1], case[2]
    page = case[5]
    longest = max(lens)
    r = rows or (longest + bs - 2) // bs + 1
    cap = (max(max(1, -(-max(x, 1) // page)) for x in kv) + 1) * page
    g = torch.Generator().manual_seed(seed)
    return torch.rand((len(lens), hq, r, blocks or -(-cap // bs)), generator=g) < density


def _check(out, lse, want, dtype, d, keys, what):
    o, e = ref.attention_bounds(*want, dtype, d, keys)
    err = (out.cpu().double() - want[0]).abs()
    assert bool((err <= o).all()), f"{what}: output {float((err - o).max()):.3e} over the bound"
    empty = want[1] == -math.inf
    assert torch.equal(lse.cpu() == -math.inf, empty), f"{what}: empty rows"
    le = (lse.cpu().double() - want[1])[~empty].abs()
    assert bool((le <= e[~empty]).all()), f"{what}: log-sum {float((le - e[~empty]).max()):.3e} over the bound"


@pytest.mark.parametrize("index", range(len(CASES)))
def test_dense(index):
    lens, kv, hq, hkv, d, page, dtype, causal = CASES[index]
    dev = require_gpu()
    t = ref.make(lens, kv, hq, hkv, d, page, dtype, seed=index, pad=3)
    want = ref.attention(*t, causal=causal)
    q, k, v, table, kvl, cu = _put(t, dev)
    attn = BlockSparseFlashAttention(min_sparsity_for_speedup=0.0)
    for splits in (None, 1, 3):
        print(f"chunk {CASES[index]} splits={splits}", flush=True)
        out, lse = attn.forward_chunk_paged(q, k, v, table, kvl, cu, max_seqlen=max(max(lens), 1), causal=causal,
                                            return_lse=True, num_splits=splits)
        torch.cuda.synchronize()
        _check(out, lse, want, dtype, d, max(kv), f"splits {splits}")
    assert torch.equal(out[-3:], torch.zeros_like(out[-3:]))
    alone = attn.forward_chunk_paged(q, k, v, table, kvl, cu.cpu(), causal=causal, num_splits=3)
    assert torch.equal(alone, out)


@pytest.mark.parametrize("bs", [32, 64, 128])
@pytest.mark.parametrize("index", range(2, len(CASES)))
def test_block_mask(index, bs):
    lens, kv, hq, hkv, d, page, dtype, causal = CASES[index]
    dev = require_gpu()
    t = ref.make(lens, kv, hq, hkv, d, page, dtype, seed=50 + index, pad=1)
    attn = BlockSparseFlashAttention(block_size=bs, min_sparsity_for_speedup=0.0)
    for density in (0.4, 0.05):  # at the second many rows see nothing
        mask = _mask(CASES[index], index, bs, density)
        want = ref.attention(*t, mask=mask, bs=bs, causal=causal)
        q, k, v, table, kvl, cu = _put(t, dev)
        for splits, m in ((None, mask.to(dev)), (2, mask.to(dev).transpose(1, 2).contiguous().transpose(1, 2)),
                          (1, mask.to(torch.int32))):
            print(f"chunk {CASES[index]} block {bs} density {density} splits={splits}", flush=True)
            out, lse = attn.forward_chunk_paged(q, k, v, table, kvl, cu, m, max_seqlen=max(lens), causal=causal,
                                                return_lse=True, num_splits=splits)
            torch.cuda.synchronize()
            _check(out, lse, want, dtype, d, max(kv), f"block {bs} splits {splits}")


@pytest.mark.parametrize("bs", [32, 64, 128])
@pytest.mark.parametrize(("lens", "hq", "hkv", "d"), [([1, 1], 14, 2, 128), ([5, 2], 8, 2, 64), ([1, 0], 32, 1, 64),
                                                       ([40, 3], 4, 2, 128)])
def test_block_mask_of_a_long_cache(lens, hq, hkv, d, bs):
    """More key tiles than a wave looks over at once, whole stretches of them left out."""
    dev = require_gpu()
    kv, page = [9500, 13000], 16
    t = ref.make(lens, kv, hq, hkv, d, page, BF, seed=bs)
    mask = _mask((lens, kv, hq, hkv, d, page), bs, bs, 0.05, blocks=-(-t[3].shape[1] * page // bs))
    mask[:, :, :, 4200 // bs:8400 // bs] = False
    mask[0, 0] = False
    want = ref.attention(*t, mask=mask, bs=bs)
    q, k, v, table, kvl, cu = _put(t, dev)
    attn = BlockSparseFlashAttention(block_size=bs, min_sparsity_for_speedup=0.0)
    for splits in (None, 1, 5):
        print(f"chunk long masked lens={lens} heads={hq}/{hkv} block={bs} splits={splits}", flush=True)
        out, lse = attn.forward_chunk_paged(q, k, v, table, kvl, cu, mask.to(dev), max_seqlen=max(lens), return_lse=True,
                                            num_splits=splits)
        _check(out, lse, want, BF, d, max(kv), f"splits {splits}")


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize(("lens", "kv"), [([100], [230]), ([6], [200]), ([1], [100])])
def test_what_a_row_does_not_see_does_not_reach_it(lens, kv, masked, dtype):
    """NaN and infinities in keys and values behind a token, in blocks its mask leaves out and
    behind the cache's end change nothing; those it sees do."""
    dev = require_gpu()
    hq, hkv, d, page, bs = 4, 2, 128, 16, 32
    t = ref.make(lens, kv, hq, hkv, d, page, dtype, seed=7)
    q, k, v, table, kvl, cu = t
    mask = _mask((lens, kv, hq, hkv, d, page), 5, bs, 0.5) if masked else None
    if masked:
        mask[..., 0] = True
    attn = BlockSparseFlashAttention(block_size=bs, min_sparsity_for_speedup=0.0)

    def run():
        a = _put((q, k, v, table, kvl, cu), dev)
        return attn.forward_chunk_paged(*a, None if mask is None else mask.to(dev), max_seqlen=max(lens),
                                        return_lse=True)

    print(f"chunk unseen values lens={lens} masked={masked} {dtype}", flush=True)
    clean, clean_lse = run()
    length, cached = lens[0], kv[0]
    poison = [cached - 1, cached - length + length // 2, 40]
    for slot in poison:
        pg, row = int(table[0, slot // page]), slot % page
        for g in range(hkv):
            v[pg, row, g, 3] = float("inf")
            v[pg, row, g, 70] = float("nan")
            k[pg, row, g, 1] = float("nan") if slot != 40 else k[pg, row, g, 1]
    out, lse = run()
    for h in range(hq):
        see = ref.visible(cached - length, length, cached, True, None if mask is None else mask[0], bs, h)
        for i in range(length):
            if not see[i, poison].any():
                assert torch.equal(out[i, h], clean[i, h]) and torch.equal(lse[i, h], clean_lse[i, h])
            elif see[i, 40] and not see[i, poison[:2]].any():
                assert out[i, h, 3] == math.inf and bool(torch.isnan(out[i, h, 70]))
                rest = torch.ones(d, dtype=torch.bool)
                rest[[3, 70]] = False
                assert torch.equal(out[i, h].cpu()[rest], clean[i, h].cpu()[rest])
            else:
                assert bool(torch.isnan(out[i, h]).all()) and bool(torch.isnan(lse[i, h]))


@pytest.mark.parametrize("lens", [[1, 1], [6, 3], [90, 130]])
def test_strides_and_large_scores(lens):
    """Queries cut from a wider projection, head-major pools, a table with a row stride, and scores
    whose running maximum moves far: equal to contiguous copies, and to the 64-bit form."""
    dev = require_gpu()
    hq, hkv, d, page = 8, 2, 64, 16
    kv = [400, 333]
    t = ref.make(lens, kv, hq, hkv, d, page, BF, seed=3, scale=4.0)
    q, k, v, table, kvl, cu = t
    for n in range(2):
        for slot in range(kv[n]):  # growing keys
            k[int(table[n, slot // page]), slot % page] *= 1.0 + slot / 100
    want = ref.attention(*t)
    q, k, v, table, kvl, cu = _put(t, dev)
    attn = BlockSparseFlashAttention(min_sparsity_for_speedup=0.0)
    print(f"chunk strides lens={lens}", flush=True)
    out, lse = attn.forward_chunk_paged(q, k, v, table, kvl, cu, max_seqlen=max(lens), return_lse=True)
    _check(out, lse, want, BF, d, max(kv), "large scores")
    wide = torch.randn(q.shape[0], hq + 2 * hkv, d, device=dev).bfloat16()
    wide[:, :hq] = q
    hm = [x.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for x in (k, v)]
    big = torch.zeros((2, table.shape[1] + 5), dtype=torch.int32, device=dev)
    big[:, :table.shape[1]] = table
    again = attn.forward_chunk_paged(wide[:, :hq], *hm, big[:, :table.shape[1]], kvl.long(), cu, max_seqlen=max(lens))
    assert torch.equal(again, out)
    odd = torch.empty(q.numel() + 1, dtype=BF, device=dev)[1:].view(q.shape).copy_(q)  # two bytes off
    assert torch.equal(attn.forward_chunk_paged(odd, k, v, table, kvl, cu, max_seqlen=max(lens)), out)


@pytest.mark.parametrize("lens", [[1], [4], [80]])
def test_lengths_are_clamped(lens):
    """A length past the table and table entries outside the pool read pages that exist; a negative
    length reads nothing."""
    dev = require_gpu()
    t = ref.make(lens, [90], 4, 2, 128, 16, BF, seed=1)
    q, k, v, table, kvl, cu = _put(t, dev)
    k, v = k.nan_to_num(0.5), v.nan_to_num(0.5, posinf=0.5)
    attn = BlockSparseFlashAttention(min_sparsity_for_speedup=0.0)
    print(f"chunk clamped lens={lens}", flush=True)
    over = attn.forward_chunk_paged(q, k, v, table, kvl + 100000, cu, max_seqlen=lens[0])
    assert bool(torch.isfinite(over).all())
    wild = table.clone()
    wild[0, 0], wild[0, 1] = -7, 1 << 30
    assert bool(torch.isfinite(attn.forward_chunk_paged(q, k, v, wild, kvl, cu, max_seqlen=lens[0])).all())
    out, lse = attn.forward_chunk_paged(q, k, v, table, kvl - 1000, cu, max_seqlen=lens[0], return_lse=True)
    assert not out.any() and bool((lse == -math.inf).all())


@pytest.mark.parametrize("masked", [0, 32, 64, 128])
@pytest.mark.parametrize("index", range(len(CASES)))
def test_key_weights(index, masked):
    _check_weights(index, masked, None)


@pytest.mark.parametrize("masked", [0, 32, 64, 128])
@pytest.mark.parametrize("index", range(len(CASES)))
def test_key_weights_of_a_wide_table(index, masked):
    # Room for 512 workgroups of 256 keys: the kernel for many keys.
    lens, _, _, hkv, _, page = CASES[index][:6]
    _check_weights(index, masked, -(-512 // (len(lens) * hkv)) * 256 // page)


@pytest.mark.parametrize("masked", [0, 32, 64, 128])
@pytest.mark.parametrize("index", range(len(CASES)))
def test_key_weights_of_many_rows(index, masked):
    # As many rows as the kernel for few keys and many rows asks for, most of them padding.
    _check_weights(index, masked, None, pad=1024, longest=1024)


@pytest.mark.parametrize("masked", [0, 64])
@pytest.mark.parametrize("case", [([700, 513], [700, 1500], 4, 2, 128, 16, BF, True),
                                  ([2100, 1], [2300, 900], 3, 3, 64, 64, HF, True)])
def test_key_weights_of_long_chunks(case, masked):
    _check_weights(case, masked, None)


def _check_weights(index, masked, max_pages, pad=2, longest=None):
    case = CASES[index] if isinstance(index, int) else index
    index = index if isinstance(index, int) else 50
    lens, kv, hq, hkv, d, page, dtype, causal = case
    dev = require_gpu()
    longest = longest or max(lens)
    t = ref.make(lens, kv, hq, hkv, d, page, dtype, seed=100 + index, pad=pad, max_pages=max_pages)
    q, k, v, table, kvl, cu = t
    cap = table.shape[1] * page
    mask = _mask(case, index, masked, 0.3, (longest + masked - 2) // masked + 1, -(-cap // masked)) if masked else None
    lse = ref.attention(*t, mask=mask, bs=masked or 64, causal=causal)[1].float()
    before = torch.rand((len(lens), hkv, cap), generator=torch.Generator().manual_seed(index))
    total, dot = ref.key_weights(q, k, table, kvl, cu, lse, before, mask, masked or 64, causal)
    weight = total - before.double()
    print(f"key weights {case} mask {masked}", flush=True)
    a = [x.to(dev) for x in (q, k, table, kvl, cu, lse)]
    md = None if mask is None else mask.to(dev)
    got = accumulate_key_weights(*a, before.to(dev), block_mask=md, block_size=masked or 64, causal=causal,
                                 max_seqlen=longest)
    torch.cuda.synchronize()
    # Scores as in the attention's bound, twice for the exponent's own rounding; fp32 sums over rows.
    rel = 2 * ((d + 3) * dot + 8 * (1 + dot)) * 2.0 ** -24 + (max(lens) * hq // hkv + 2) * 2.0 ** -24
    err = (got.cpu().double() - total).abs()
    assert bool((err <= rel * weight + 2.0 ** -23 * total).all()), float((err - rel * weight).max())
    for n in range(len(lens)):
        assert torch.equal(got[n, :, max(kv[n], 0):].cpu(), before[n, :, max(kv[n], 0):])
    bare = accumulate_key_weights(*a, block_mask=md, block_size=masked or 64, causal=causal, max_seqlen=longest)
    assert bool(((bare.cpu().double() - weight).abs() <= rel * weight + 2.0 ** -23 * weight).all())
    # The weights of a row add up to one.
    rows = int((lse[:int(cu[-1])] != -math.inf).sum())
    assert abs(float(bare.double().sum()) - rows) <= (rel + 1e-5) * max(rows, 1)


@pytest.mark.parametrize("masked", [0, 64])
def test_longer_than_max_seqlen(masked):
    """A sequence's tokens behind its first max_seqlen are left out; those before keep their place."""
    dev = require_gpu()
    lens, kv, cut = [150, 3, 40], [400, 90, 40], 70
    t = ref.make(lens, kv, 4, 2, 128, 16, BF, seed=3)
    case = (lens, kv, 4, 2, 128, 16)
    rows = (cut + 62) // 64 + 1
    mask = _mask(case, 1, 64, 0.4, blocks=-(-t[3].shape[1] * 16 // 64)) if masked else None
    want = ref.attention(*t, mask=mask)
    q, k, v, table, kvl, cu = _put(t, dev)
    md = None if mask is None else mask[:, :, :rows].to(dev)
    attn = BlockSparseFlashAttention(min_sparsity_for_speedup=0.0)
    print(f"chunk longer than max_seqlen, masked={masked}", flush=True)
    out, lse = attn.forward_chunk_paged(q, k, v, table, kvl, cu, md, max_seqlen=cut, return_lse=True)
    kept = torch.cat([torch.arange(min(x, cut)) + int(a) for x, a in zip(lens, t[5])])
    _check(out[kept], lse[kept], [x[kept] for x in want], BF, 128, max(kv), "kept")
    # Their weights alone, each row's adding up to one.
    w = accumulate_key_weights(q, k, table, kvl, cu, lse, block_mask=md, max_seqlen=cut)
    short = want[1].float()
    short[[i for i in range(sum(lens)) if i not in set(kept.tolist())]] = -math.inf
    zeros = torch.zeros(w.shape)
    total, dot = ref.key_weights(*[t[i] for i in (0, 1, 3, 4, 5)], short, zeros, mask)
    rel = 4 * ((128 + 3) * dot + 8 * (1 + dot)) * 2.0 ** -24 + (cut * 2 + max(kv)) * 2.0 ** -24
    assert bool(((w.cpu().double() - total).abs() <= rel * total).all())


@pytest.mark.parametrize("masked", [0, 64])
@pytest.mark.parametrize("lens", [[1, 1], [5, 300]])
def test_offsets_past_32_bits(lens, masked):
    """Pools whose pages lie 128 MB apart, 5 GB in all: the same bits as in close pools."""
    dev = require_gpu()
    kv, page = [300, 700], 32
    t = ref.make(lens, kv, 4, 2, 128, page, BF, seed=4)
    mask = _mask((lens, kv, 4, 2, 128, page), 2, 64, 0.5, blocks=-(-t[3].shape[1] * page // 64)) if masked else None
    q, k, v, table, kvl, cu = _put(t, dev)
    md = None if mask is None else mask.to(dev)
    far = []
    for x in (k, v):
        room = torch.empty((x.shape[0], 1 << 26), dtype=BF, device=dev)
        far.append(room[:, :x[0].numel()].view(x.shape).copy_(x))
    assert (k.shape[0] - 1) << 26 > 1 << 31
    attn = BlockSparseFlashAttention(min_sparsity_for_speedup=0.0)
    print(f"chunk far pages lens={lens} masked={masked}", flush=True)
    out, lse = attn.forward_chunk_paged(q, k, v, table, kvl, cu, md, max_seqlen=max(lens), return_lse=True)
    o2, l2 = attn.forward_chunk_paged(q, *far, table, kvl, cu, md, max_seqlen=max(lens), return_lse=True)
    assert torch.equal(out, o2) and torch.equal(lse, l2)
    w = accumulate_key_weights(q, k, table, kvl, cu, lse, block_mask=md, max_seqlen=max(lens))
    assert torch.equal(w, accumulate_key_weights(q, far[0], table, kvl, cu, lse, block_mask=md, max_seqlen=max(lens)))


@pytest.mark.parametrize("masked", [0, 64])
@pytest.mark.parametrize(("lens", "over"), [([1, 1], [1, 0]), ([5, 3], [2, 300]), ([70, 130], [33, 1])])
def test_lengths_past_the_table(lens, over, masked):
    """Lengths (on the device) that pass the table: the chunk's tokens keep the positions they were
    written at, and the keys are those that the table holds. The oracle has a longer table, whose blocks
    behind the short one's end no row sees."""
    dev = require_gpu()
    hq, hkv, d, page, cap = 4, 2, 128, 16, 256
    kv = [cap + x for x in over]
    t = ref.make(lens, kv, hq, hkv, d, page, BF, seed=12)
    rows, blocks = (max(lens) + 62) // 64 + 1, -(-t[3].shape[1] * page // 64)
    mask = _mask((lens, kv, hq, hkv, d, page), 4, 64, 0.5 if masked else 2.0, blocks=blocks)
    mask[..., cap // 64:] = False
    want = ref.attention(*t, mask=mask)
    q, k, v, table, kvl, cu = _put(t, dev)
    short = table[:, :cap // page].contiguous()
    md = mask[..., :cap // 64].contiguous().to(dev) if masked else None
    attn = BlockSparseFlashAttention(min_sparsity_for_speedup=0.0)
    for splits in (None, 3):
        print(f"chunk past the table lens={lens} over={over} masked={masked} splits={splits}", flush=True)
        out, lse = attn.forward_chunk_paged(q, k, v, short, kvl, cu, md, max_seqlen=max(lens), return_lse=True,
                                            num_splits=splits)
        _check(out, lse, want, BF, d, cap, f"splits {splits}")
    exact = want[1].float()
    got = accumulate_key_weights(q, k, short, kvl, cu, exact.to(dev), block_mask=md, max_seqlen=max(lens))
    total, dot = ref.key_weights(t[0], t[1], *t[3:], exact, torch.zeros(len(lens), hkv, t[3].shape[1] * page), mask)
    rel = 2 * ((d + 3) * dot + 8 * (1 + dot)) * 2.0 ** -24 + (max(lens) * hq // hkv + 2) * 2.0 ** -24
    assert bool(((got.cpu().double() - total[..., :cap]).abs() <= (rel + 2.0 ** -23) * total[..., :cap]).all())


@pytest.mark.parametrize("splits", [1, 3, 9])
@pytest.mark.parametrize(("hq", "cut", "masked"), [(4, 70, 0), (4, 70, 64), (4, 8, 64), (32, 8, 0)])
def test_rows_behind_max_seqlen_are_not_written(hq, cut, masked, splits):
    """The C entry leaves the output rows of tokens behind max_seqlen as they were, with one split and with
    several joined."""
    dev = require_gpu()
    lens, kv, hkv, d, page = [150, 3, 75, 1], [400, 90, 75, 30], 2, 128, 16
    t = ref.make(lens, kv, hq, hkv, d, page, BF, seed=3, pad=2)
    blocks = -(-t[3].shape[1] * page // 64)
    mask = _mask((lens, kv, hq, hkv, d, page), 1, 64, 0.4, blocks=blocks) if masked else None
    want = ref.attention(*t, mask=mask)
    q, k, v, table, kvl, cu = _put(t, dev)
    md = None if mask is None else mask[:, :, :(cut + 62) // 64 + 1].contiguous().to(dev)
    out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device=dev)
    lib = _native.load_library()
    size = lib.tasft_chunk_workspace_bytes(q.shape[0], hq, d, splits)
    ws = torch.full((max(size, 4) // 4,), 3.0, device=dev)
    print(f"chunk cut at {cut}, heads {hq}, masked={masked} splits={splits}", flush=True)
    status = lib.tasft_chunk_paged_fwd(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(), _native.ptr(md), table.data_ptr(),
        kvl.data_ptr(), cu.data_ptr(), ws.data_ptr(), size, len(lens), q.shape[0], hq, hkv, cut, d, 64,
        0 if md is None else md.shape[2], page, k.shape[0], table.shape[1], splits, _native.strides(q),
        _native.strides(k), _native.strides(v), _native.strides(out), None if md is None else _native.strides(md),
        table.stride(0), 1.0 / math.sqrt(d), 1, _native.DTYPE_BF16, _native.stream_handle(q.device))
    _native.check(status, "tasft_chunk_paged_fwd")
    torch.cuda.synchronize()
    kept = torch.cat([torch.arange(min(x, cut)) + int(a) for x, a in zip(lens, t[5])] + [torch.arange(2) + sum(lens)])
    _check(out[kept], lse[kept], [x[kept] for x in want], BF, d, max(kv), "kept")
    rest = torch.ones(q.shape[0], dtype=torch.bool)
    rest[kept] = False
    assert rest.any() and bool((out.cpu()[rest] == 7.0).all()) and bool((lse.cpu()[rest] == 7.0).all())
