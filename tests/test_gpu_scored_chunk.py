"""Chunk attention over a paged cache with capped and biased scores and over trees of new tokens, against the
64-bit form."""
from __future__ import annotations

import math

import pytest
import torch

import paged_ref
import scored_ref as ref
from helpers import require_gpu
from tasft_amd.exceptions import KernelError
from tasft_amd.kernels import BlockSparseFlashAttention, append_paged, dense_attention, rotary_frequencies

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16

# lens, kv_lens, Hq, Hkv, D, page, dtype, softcap, slopes
CASES = [
    ([1], [1], 1, 1, 128, 16, BF, 30.0, False),
    ([1, 1, 1], [65, 700, 64], 8, 2, 128, 16, BF, 50.0, False),
    ([1, 1], [333, 20], 28, 4, 128, 8, HF, 0, True),
    ([5, 3, 0, 8], [700, 64, 40, 8], 8, 2, 128, 16, BF, 10.0, True),
    ([2, 1, 7], [64, 65, 71], 6, 2, 64, 8, HF, 20.0, True),
    ([70, 1, 33], [70, 500, 300], 8, 2, 128, 32, BF, 0, True),
    ([130, 200], [130, 515], 4, 2, 64, 64, HF, 500.0, False),
    ([9, 70], [4, 50], 4, 2, 128, 16, BF, 15.0, True),       # fewer cached keys than new tokens
    ([150], [1000], 7, 1, 128, 256, BF, 30.0, True),
]


def slopes_of(hq):
    return torch.tensor([2.0 ** (-8.0 * (i + 1) / hq) for i in range(hq)])


def check(out, lse, want, what):
    o, l, e_o, e_l = want
    err = (out.cpu().double() - o).abs()
    assert bool((err <= e_o).all()), f"{what}: output {float((err - e_o).max()):.3e} over the bound"
    empty = l == -math.inf
    assert torch.equal(lse.cpu() == -math.inf, empty), f"{what}: empty rows"
    err = (lse.cpu().double() - l)[~empty].abs()
    assert bool((err <= e_l[~empty]).all()), f"{what}: log-sum {float((err - e_l[~empty]).max()):.3e} over the bound"


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("index", range(len(CASES)))
def test_scores(index, causal):
    lens, kv, hq, hkv, d, page, dtype, cap, biased = CASES[index]
    dev = require_gpu()
    t = paged_ref.make(lens, kv, hq, hkv, d, page, dtype, seed=index, pad=2, scale=2.0)
    slopes = slopes_of(hq) if biased else None
    want = ref.attention(*t, cap=cap, slopes=slopes, causal=causal)
    a = [x.to(dev) for x in t]
    attn = BlockSparseFlashAttention(min_sparsity_for_speedup=0.0)
    for splits in (None, 1, 3, 9):
        print(f"scored {CASES[index]} causal={causal} splits={splits}", flush=True)
        out, lse = attn.forward_chunk_paged(*a, max_seqlen=max(lens), causal=causal, return_lse=True, num_splits=splits,
                                            softcap=cap or None, alibi_slopes=None if slopes is None else slopes.to(dev))
        torch.cuda.synchronize()
        check(out, lse, want, f"splits {splits}")
    assert not out[-2:].any()


@pytest.mark.parametrize("bs", [32, 64, 128])
@pytest.mark.parametrize("index", [1, 2, 3, 4, 5, 6, 8])
def test_scores_under_a_block_mask(index, bs):
    lens, kv, hq, hkv, d, page, dtype, cap, biased = CASES[index]
    dev = require_gpu()
    t = paged_ref.make(lens, kv, hq, hkv, d, page, dtype, seed=20 + index, pad=1)
    slopes = slopes_of(hq) if biased else None
    rows, cap_slots = (max(lens) + bs - 2) // bs + 1, t[3].shape[1] * page
    g = torch.Generator().manual_seed(index)
    mask = torch.rand((len(lens), hq, rows, -(-cap_slots // bs)), generator=g) < 0.4
    want = ref.attention(*t, cap=cap, slopes=slopes, mask=mask, bs=bs)
    a = [x.to(dev) for x in t]
    attn = BlockSparseFlashAttention(block_size=bs, min_sparsity_for_speedup=0.0)
    for splits in (None, 2):
        print(f"scored {CASES[index]} block {bs} splits={splits}", flush=True)
        out, lse = attn.forward_chunk_paged(*a, mask.to(dev), max_seqlen=max(lens), return_lse=True, num_splits=splits,
                                            softcap=cap or None, alibi_slopes=None if slopes is None else slopes.to(dev))
        torch.cuda.synchronize()
        check(out, lse, want, f"block {bs} splits {splits}")


# lens, kv_lens, Hq, Hkv, D, page, dtype, softcap, slopes
TREES = [
    ([1], [1], 1, 1, 128, 16, BF, 0, False),
    ([2, 1, 3], [2, 40, 100], 4, 2, 64, 8, HF, 0, True),
    ([25], [1000], 16, 16, 64, 32, HF, 30.0, True),
    ([64, 63, 0, 33], [64, 300, 10, 97], 8, 2, 128, 16, BF, 0, False),
    ([65, 64], [129, 128], 4, 1, 128, 16, BF, 0, True),
    ([130, 7, 200], [700, 70, 333], 4, 2, 128, 64, HF, 20.0, True),
    ([300], [301], 3, 1, 64, 16, BF, 0, True),
    ([9, 70], [4, 50], 4, 2, 128, 16, BF, 0, True),          # the first nodes are not cached
    ([17] * 5, [5000, 16, 900, 17, 200], 28, 4, 128, 16, BF, 0, False),
]


def tree_of(lens, seed, extra=0):
    cu = torch.tensor([0] + lens).cumsum(0).tolist()
    rows = ref.chains(ref.random_parents(lens, seed), cu)
    return rows, ref.bits(rows, -(-max(lens) // 64) + extra)


@pytest.mark.parametrize("index", range(len(TREES)))
def test_trees(index):
    lens, kv, hq, hkv, d, page, dtype, cap, biased = TREES[index]
    dev = require_gpu()
    pad = 3
    t = paged_ref.make(lens, kv, hq, hkv, d, page, dtype, seed=40 + index, pad=pad)
    rows, words = tree_of(lens, index, extra=index % 2)
    words = torch.cat((words, torch.full((pad, words.shape[1]), -1))).to(dev)
    slopes = slopes_of(hq) if biased else None
    want = ref.attention(*t, cap=cap, slopes=slopes, rows=rows)
    a = [x.to(dev) for x in t]
    attn = BlockSparseFlashAttention(min_sparsity_for_speedup=0.0)
    for splits in (None, 1, 3, 9):
        print(f"tree {TREES[index]} splits={splits}", flush=True)
        out, lse = attn.forward_chunk_paged(*a, max_seqlen=max(lens), return_lse=True, num_splits=splits, ancestors=words,
                                            softcap=cap or None, alibi_slopes=None if slopes is None else slopes.to(dev))
        torch.cuda.synchronize()
        check(out, lse, want, f"splits {splits}")
    assert not out[-pad:].any()


@pytest.mark.parametrize("biased", [False, True])
def test_what_a_node_does_not_see_does_not_reach_it(biased):
    """NaN and infinities of other branches and of keys behind the cache's end."""
    dev = require_gpu()
    n, kv, hq, hkv, d, page = 90, 230, 4, 2, 128, 16
    t = paged_ref.make([n], [kv], hq, hkv, d, page, BF, seed=1)
    q, k, v, table, lens, cu = t
    rows, words = tree_of([n], 3)
    slopes = slopes_of(hq).to(dev) if biased else None
    attn = BlockSparseFlashAttention(min_sparsity_for_speedup=0.0)

    def run():
        a = [x.to(dev) for x in (q, k, v, table, lens, cu)]
        return [x.cpu() for x in attn.forward_chunk_paged(*a, max_seqlen=n, ancestors=words.to(dev), return_lse=True,
                                                          alibi_slopes=slopes)]

    print(f"tree unseen values biased={biased}", flush=True)
    clean, clean_lse = run()
    bad_v, bad_k = 40, 71
    at = [int(table[0, (kv - n + x) // page]) for x in (bad_v, bad_k)]
    v[at[0], (kv - n + bad_v) % page, :, 3] = float("inf")
    k[at[1], (kv - n + bad_k) % page, :, 1] = float("nan")
    out, lse = run()
    touched = 0
    for i in range(n):
        if bad_k in rows[i]:
            assert bool(torch.isnan(out[i]).all()) and bool(torch.isnan(lse[i]).all())
        elif bad_v in rows[i]:
            rest = [x for x in range(d) if x != 3]
            assert bool((out[i, :, 3] == math.inf).all()) and torch.equal(out[i][:, rest], clean[i][:, rest])
            touched += 1
        else:
            assert torch.equal(out[i], clean[i]) and torch.equal(lse[i], clean_lse[i])
    assert touched


@pytest.mark.parametrize("biased", [False, True])
def test_trees_cut_and_past_the_table(biased):
    """Nodes behind max_seqlen are left out, and slots behind the table are not there."""
    dev = require_gpu()
    lens, hq, hkv, d, page = [100, 20], 4, 2, 64, 16
    slopes = slopes_of(hq) if biased else None
    sd = None if slopes is None else slopes.to(dev)
    t = paged_ref.make(lens, [180, 300], hq, hkv, d, page, BF, seed=2)
    rows, words = tree_of(lens, 5)
    want = ref.attention(*t, slopes=slopes, rows=rows)
    a = [x.to(dev) for x in t]
    attn = BlockSparseFlashAttention(min_sparsity_for_speedup=0.0)
    print(f"tree cut biased={biased}", flush=True)
    out, lse = attn.forward_chunk_paged(*a, max_seqlen=50, ancestors=words.to(dev), return_lse=True, alibi_slopes=sd)
    kept = list(range(50)) + list(range(100, 120))
    check(out[kept], lse[kept], [x[kept] for x in want], "cut")
    for cap in (160, 64):  # within the tree, and before it
        want = ref.attention(*t, slopes=slopes, rows=rows, slots=cap)
        for splits in (None, 4):
            out, lse = attn.forward_chunk_paged(*a[:3], a[3][:, :cap // page].contiguous(), *a[4:], max_seqlen=100,
                                                ancestors=words.to(dev), return_lse=True, alibi_slopes=sd,
                                                num_splits=splits)
            check(out, lse, want, f"table of {cap}")


def test_refusals():
    dev = require_gpu()
    t = paged_ref.make([5, 3], [70, 64], 4, 2, 64, 16, BF, seed=0)
    a = [x.to(dev) for x in t]
    attn = BlockSparseFlashAttention(min_sparsity_for_speedup=0.0)
    words = torch.ones((8, 1), dtype=torch.int64, device=dev)
    slopes = slopes_of(4).to(dev)

    def refused(error, match, **options):
        with pytest.raises(error, match=match):
            attn.forward_chunk_paged(*a, max_seqlen=options.pop("max_seqlen", 5), **options)

    refused(ValueError, "softcap", softcap=0.0)
    refused(ValueError, "softcap", softcap=-3.0)
    refused(ValueError, "softcap", softcap=math.nan)
    refused(KernelError, "alibi_slopes", alibi_slopes=slopes[:3])
    refused(KernelError, "alibi_slopes", alibi_slopes=slopes.int())
    refused(KernelError, "require grad", alibi_slopes=slopes.clone().requires_grad_(True))
    refused(ValueError, "causal", ancestors=words, causal=False)
    mask = torch.ones((2, 4, 2, 2), dtype=torch.bool, device=dev)
    refused(ValueError, "block_mask", ancestors=words, block_mask=mask)
    refused(KernelError, "ancestors", ancestors=words[:7])
    refused(KernelError, "ancestors", ancestors=words.int())
    refused(KernelError, "ancestors", ancestors=words.cpu())
    refused(KernelError, "ancestors", ancestors=words[:, :0])
    # Slopes of another type or place are converted.
    want = attn.forward_chunk_paged(*a, max_seqlen=5, alibi_slopes=slopes)
    assert torch.equal(attn.forward_chunk_paged(*a, max_seqlen=5, alibi_slopes=slopes.double().cpu()), want)


def test_offsets_past_32_bits():
    """Pools whose pages lie 128 MB apart: the same bits as in close pools."""
    dev = require_gpu()
    lens, kv, page = [20, 70], [300, 700], 32
    t = paged_ref.make(lens, kv, 4, 2, 128, page, BF, seed=4)
    a = [x.to(dev) for x in t]
    far = []
    for x in a[1:3]:
        room = torch.empty((x.shape[0], 1 << 26), dtype=BF, device=dev)
        far.append(room[:, :x[0].numel()].view(x.shape).copy_(x))
    words = tree_of(lens, 1)[1].to(dev)
    slopes = slopes_of(4).to(dev)
    attn = BlockSparseFlashAttention(min_sparsity_for_speedup=0.0)
    print("scored far pages", flush=True)
    for options in ({"ancestors": words}, {"softcap": 20.0, "alibi_slopes": slopes}):
        want = attn.forward_chunk_paged(*a, max_seqlen=70, return_lse=True, **options)
        got = attn.forward_chunk_paged(a[0], *far, *a[3:], max_seqlen=70, return_lse=True, **options)
        assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])


def test_serving_agrees_with_training():
    """A prompt in chunks over pages and then token by token, capped and biased: the training form's rows."""
    dev = require_gpu()
    hq, hkv, d, page, n = 8, 2, 128, 16, 150
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn((n, h, d), generator=g).to(BF).to(dev) for h in (hq, hkv, hkv))
    slopes = slopes_of(hq).to(dev)
    inv, factor = rotary_frequencies(d, device=dev)
    zero = torch.zeros(n, dtype=torch.int32, device=dev)  # not turned: position 0
    pools = [torch.zeros((10, page, hkv, d), dtype=BF, device=dev) for _ in range(2)]
    table = torch.randperm(10, generator=g).to(torch.int32)[None].to(dev)
    attn = BlockSparseFlashAttention(min_sparsity_for_speedup=0.0)
    whole, lse = dense_attention(q, k, v, cu_seqlens=torch.tensor([0, n]), softcap=25.0, alibi_slopes=slopes,
                                 return_lse=True)
    print("scored serving and training", flush=True)
    at = 0
    for step in (70, 64, 9, 1, 1, 1, 1, 1, 1, 1):
        lens = torch.tensor([at + step], dtype=torch.int32, device=dev)
        cu = torch.tensor([0, step], dtype=torch.int32, device=dev)
        s = slice(at, at + step)
        turned = append_paged(q[s], k[s], v[s], *pools, table, lens, cu, inv, scale=1.0, positions=zero[s])
        assert torch.equal(turned, q[s])
        out, part = attn.forward_chunk_paged(turned, *pools, table, lens, cu, max_seqlen=step, softcap=25.0,
                                             alibi_slopes=slopes, return_lse=True)
        # Both are within the bounds of tests/dense_ref.py of the same value: two roundings of P and two of
        # the output apart, of values of about 1 (weighted magnitudes of V).
        assert float((out.float() - whole[s].float()).abs().max()) <= 4 * 2.0 ** -8 * float(v.float().abs().max())
        assert float((part - lse[s]).abs().max()) <= 1e-4
        at += step
    assert at == n
