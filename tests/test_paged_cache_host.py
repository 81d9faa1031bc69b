"""Rotary frequencies, and the refusals of the rotary and paged-cache calls, on the CPU: every
check comes before any kernel (a valid call on CPU tensors ends at the device check)."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

import paged_ref as ref
from tasft_amd import _native
from tasft_amd.exceptions import KernelError
from tasft_amd.kernels import (
    BlockSparseFlashAttention,
    accumulate_key_weights,
    append_paged,
    apply_rotary,
    default_chunk_splits,
    evict_paged,
    rotary_frequencies,
)

BF = torch.bfloat16


# --------------------------------------------------------------------------- frequencies
def test_default_and_linear_frequencies():
    f, a = rotary_frequencies(64, 10000.0)
    assert f.dtype == torch.float64 and a == 1.0
    assert torch.equal(f, torch.tensor([10000.0 ** (-2.0 * j / 64) for j in range(32)], dtype=torch.float64))
    assert f[0] == 1.0
    g, a = rotary_frequencies(64, 10000.0, {"rope_type": "linear", "factor": 4.0})
    assert a == 1.0 and torch.equal(g, f / 4.0)
    assert torch.equal(rotary_frequencies(64, 10000.0, {"type": "default"})[0], f)


def test_llama3_frequencies():
    """The published values: wavelengths under original / high stay, over original / low are divided,
    between them the frequency is a mix linear in original / wavelength."""
    cfg = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
           "original_max_position_embeddings": 8192}
    plain, _ = rotary_frequencies(128, 500000.0)
    got, a = rotary_frequencies(128, 500000.0, cfg)
    assert a == 1.0
    for f, x in zip(plain.tolist(), got.tolist()):
        wave = 2 * math.pi / f
        if wave < 8192 / 4.0:
            want = f
        elif wave > 8192 / 1.0:
            want = f / 8.0
        else:
            s = (8192 / wave - 1.0) / 3.0
            want = (1 - s) * f / 8.0 + s * f
        assert abs(x - want) <= 1e-14 * want


def test_yarn_frequencies():
    cfg = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 4096}
    plain, _ = rotary_frequencies(128, 10000.0)
    got, a = rotary_frequencies(128, 10000.0, cfg)
    assert abs(a - (0.1 * math.log(4.0) + 1.0)) < 1e-15
    # 32 turns over 4096 positions at pair 128 ln(4096 / (64 pi)) / (2 ln 10000) = 20.9, one turn at 45.03.
    low, high = 20, 46
    for j, (f, x) in enumerate(zip(plain.tolist(), got.tolist())):
        r = min(1.0, max(0.0, (j - low) / (high - low)))
        assert abs(x - (f / 4.0 * r + f * (1 - r))) <= 1e-15
    assert rotary_frequencies(128, 10000.0, {**cfg, "attention_factor": 1.5})[1] == 1.5


@pytest.mark.parametrize(("args", "match"), [
    ((63,), "even"), ((0,), "even"), ((64, 0.0), "base"), ((64, math.inf), "base"),
    ((64, 1e4, {"rope_type": "dynamic", "factor": 2.0}), "rope_type"),
    ((64, 1e4, {"rope_type": "linear"}), "factor"),
    ((64, 1e4, {"rope_type": "linear", "factor": 0.0}), "factor"),
    ((64, 1e4, {"rope_type": "yarn", "factor": 2.0}), "original_max"),
    ((64, 1e4, {"rope_type": "llama3", "factor": 2.0, "original_max_position_embeddings": 64,
                "low_freq_factor": 4.0, "high_freq_factor": 1.0}), "low_freq"),
])
def test_frequency_refusals(args, match):
    with pytest.raises(ValueError, match=match):
        rotary_frequencies(*args)


def test_yarn_factor_of_mscale():
    """The published factor on cosine and sine: (0.1 m ln(factor) + 1) of mscale over that of
    mscale_all_dim."""
    cfg = {"type": "yarn", "factor": 40.0, "original_max_position_embeddings": 4096, "beta_fast": 32, "beta_slow": 1}
    both = {**cfg, "mscale": 1.0, "mscale_all_dim": 1.0}
    assert rotary_frequencies(64, 10000.0, both)[1] == 1.0
    assert rotary_frequencies(64, 10000.0, {**cfg, "mscale": 0.707, "mscale_all_dim": 0.707})[1] == 1.0
    got = rotary_frequencies(64, 10000.0, {**cfg, "mscale": 1.0, "mscale_all_dim": 0.5})[1]
    assert abs(got - (0.1 * math.log(40.0) + 1.0) / (0.05 * math.log(40.0) + 1.0)) < 1e-15
    assert abs(rotary_frequencies(64, 10000.0, {**cfg, "mscale": 1.0, "mscale_all_dim": 0.0})[1]
               - (0.1 * math.log(40.0) + 1.0)) < 1e-15
    assert rotary_frequencies(64, 10000.0, {**both, "attention_factor": 1.25})[1] == 1.25  # given: taken as it is
    assert rotary_frequencies(64, 10000.0, {**both, "factor": 1.0, "mscale": 2.0})[1] == 1.0
    assert torch.equal(rotary_frequencies(64, 10000.0, both)[0], rotary_frequencies(64, 10000.0, cfg)[0])


def test_yarn_range_without_rounding():
    cfg = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 4096, "truncate": False}
    plain, _ = rotary_frequencies(128, 10000.0)
    got, a = rotary_frequencies(128, 10000.0, cfg)
    assert abs(a - (0.1 * math.log(4.0) + 1.0)) < 1e-15
    low, high = (128 * math.log(4096 / (t * 2 * math.pi)) / (2 * math.log(10000.0)) for t in (32.0, 1.0))
    for j, (f, x) in enumerate(zip(plain.tolist(), got.tolist())):
        r = min(1.0, max(0.0, (j - low) / (high - low)))
        assert abs(x - (f / 4.0 * r + f * (1 - r))) <= 1e-15
    rounded = rotary_frequencies(128, 10000.0, {**cfg, "truncate": True})[0]
    assert not torch.equal(got, rounded)
    assert torch.equal(rounded, rotary_frequencies(128, 10000.0, {k: v for k, v in cfg.items() if k != "truncate"})[0])


_YARN = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 4096}


@pytest.mark.parametrize(("base", "scaling", "match"), [
    (1.0, _YARN, "base"), (0.5, _YARN, "base"),
    (1e4, {**_YARN, "mscale": 0.707}, "mscale"), (1e4, {**_YARN, "mscale_all_dim": 1.0}, "mscale"),
    (1e4, {**_YARN, "original_max_position_embeddings": 0}, "original_max"),
    (1e4, {**_YARN, "beta_fast": -1.0}, "beta"),
    (1e4, {**_YARN, "beta_slow": math.inf}, "beta"),
    (1e4, {**_YARN, "factor": math.inf}, "factor"),
    (1e4, {**_YARN, "short_factor": [1.0]}, "short_factor"),
    (1e4, {"rope_type": "default", "long_factor": [1.0, 2.0]}, "long_factor"),
    (1e4, {"rope_type": "linear", "factor": 2.0, "rope_theta": 5e5}, "rope_theta"),
])
def test_scaling_entries_that_would_be_ignored(base, scaling, match):
    with pytest.raises(ValueError, match=match):
        rotary_frequencies(64, base, scaling)


def test_scaling_entries_without_effect():
    """Entries of other types, and those that only describe, are read past as before."""
    plain = rotary_frequencies(64, 1e4, {"rope_type": "linear", "factor": 2.0})
    more = {"rope_type": "linear", "factor": 2.0, "original_max_position_embeddings": 4096, "rope_theta": 1e4,
            "finetuned": True, "attention_factor": None, "partial_rotary_factor": 0.5, "mrope_section": [8, 12, 12],
            "short_factor": None}
    got = rotary_frequencies(64, 1e4, more)
    assert torch.equal(got[0], plain[0]) and got[1] == plain[1]
    assert torch.equal(rotary_frequencies(64, 1e4, {})[0], rotary_frequencies(64, 1e4)[0])


def test_a_lone_mscale_of_its_default():
    """One of the two entries at the value that leaving it out means: the plain factor."""
    cfg = {"rope_type": "yarn", "factor": 40.0, "original_max_position_embeddings": 4096}
    plain = rotary_frequencies(64, 10000.0, cfg)[1]
    assert rotary_frequencies(64, 10000.0, {**cfg, "mscale": 1.0})[1] == plain
    assert rotary_frequencies(64, 10000.0, {**cfg, "mscale_all_dim": 0})[1] == plain


# ------------------------------------------------------------------------------ refusals
def _rope(**over):
    a = {"q": torch.zeros(2, 4, 5, 64, dtype=BF), "k": torch.zeros(2, 2, 5, 64, dtype=BF),
         "positions": torch.arange(5), "inv_freq": rotary_frequencies(64)[0]}
    a.update(over)
    return apply_rotary(a["q"], a["k"], a["positions"], a["inv_freq"])


@pytest.mark.parametrize(("over", "match"), [
    ({}, "CUDA"),
    ({"q": torch.zeros(5, 64, dtype=BF)}, "Expected q"),
    ({"q": torch.zeros(2, 0, 5, 64, dtype=BF)}, "one head"),
    ({"q": torch.zeros(2, 4, 5, 64)}, "bf16 or fp16"),
    ({"k": torch.zeros(2, 2, 5, 64, dtype=torch.float16)}, "one dtype"),
    ({"k": torch.zeros(2, 2, 6, 64, dtype=BF)}, "incompatible"),
    ({"k": torch.zeros(5, 2, 64, dtype=BF)}, "incompatible"),
    ({"k": torch.zeros(2, 0, 5, 64, dtype=BF)}, "incompatible"),
    ({"positions": torch.arange(6)}, "positions"),
    ({"positions": torch.zeros(3, 5, dtype=torch.int64)}, "positions"),
    ({"positions": torch.zeros(5)}, "int32 or int64"),
    ({"inv_freq": torch.zeros(33, dtype=torch.float64)}, "inv_freq"),
    ({"inv_freq": torch.zeros(0, dtype=torch.float64)}, "inv_freq"),
    ({"inv_freq": torch.zeros(32, dtype=torch.int64)}, "inv_freq"),
    ({"inv_freq": torch.zeros(32, dtype=torch.float64, requires_grad=True)}, "grad"),
    ({"q": torch.zeros(1, 1, 5, 320, dtype=BF), "k": None}, "head_dim"),
])
def test_rotary_refusals(over, match):
    with pytest.raises(KernelError, match=match):
        _rope(**over)


def _chunk_args(**over):
    q, k, v, table, kvl, cu = ref.make([5, 3], [70, 40], 4, 2, 64, 16, BF, seed=0)
    a = {"q": q, "k_pages": k, "v_pages": v, "block_table": table, "kv_lens": kvl, "cu_seqlens": cu}
    a.update(over)
    return a


_COMMON = [
    ({}, "CUDA"),
    ({"q": torch.zeros(8, 64, dtype=BF)}, "packed q"),
    ({"q": torch.zeros(8, 4, 64, dtype=torch.float16)}, "q is"),
    ({"q": torch.zeros(8, 3, 64, dtype=BF)}, "Hq % Hkv"),
    ({"q": torch.zeros(8, 4, 128, dtype=BF)}, "head_dim"),
    ({"cu_seqlens": torch.tensor([0])}, "cu_seqlens"),
    ({"cu_seqlens": torch.tensor([0, 5, 4])}, "non-decreasing"),
    ({"cu_seqlens": torch.tensor([1, 5, 8])}, "start at 0"),
    ({"cu_seqlens": torch.tensor([0, 5, 9])}, "end at"),
    ({"block_table": torch.zeros(3, 6, dtype=torch.int32)}, "block_table"),
    ({"kv_lens": torch.tensor([70, 40, 1])}, "kv_lens"),
    ({"kv_lens": torch.tensor([70, 2])}, "hold the chunk"),
    ({"kv_lens": torch.tensor([70, 1000])}, "at most"),
]


@pytest.mark.parametrize(("over", "match"), [*_COMMON,
    ({"k_pages": torch.zeros(9, 16, 2, 64, dtype=BF)}, "page pools"),
    ({"max_seqlen": 4}, "more than max_seqlen"),
    ({"max_seqlen": 0}, "max_seqlen"),
    ({"k_pages": torch.zeros(9, 4, 2, 64, dtype=BF), "v_pages": torch.zeros(9, 4, 2, 64, dtype=BF)}, "page_size"),
    ({"k_pages": torch.zeros(9, 24, 2, 64, dtype=BF), "v_pages": torch.zeros(9, 24, 2, 64, dtype=BF)}, "page_size"),
])
def test_chunk_refusals(over, match):
    a = _chunk_args(**over)
    extra = {"max_seqlen": a.pop("max_seqlen")} if "max_seqlen" in a else {}
    with pytest.raises(KernelError, match=match):
        BlockSparseFlashAttention().forward_chunk_paged(**a, **extra)


@pytest.mark.parametrize(("over", "match"), _COMMON)
def test_key_weight_refusals(over, match):
    a = _chunk_args(**over)
    a.pop("v_pages")
    with pytest.raises(KernelError, match=match):
        accumulate_key_weights(**a, lse=torch.zeros(8, 4))


@pytest.mark.parametrize(("over", "match"), _COMMON)
def test_append_refusals(over, match):
    a = _chunk_args(**over)
    kv = torch.zeros(8, 2, 64, dtype=BF)
    with pytest.raises(KernelError, match=match):
        append_paged(a["q"], kv, kv, a["k_pages"], a["v_pages"], a["block_table"], a["kv_lens"], a["cu_seqlens"],
                     rotary_frequencies(64)[0])


@pytest.mark.parametrize(("over", "error", "match"), [
    ({}, KernelError, "CUDA"),
    ({"budget": 0}, ValueError, "budget"),
    ({"recent": 9, "sinks": 2}, ValueError, "fit the budget"),
    ({"recent": -1}, ValueError, "non-negative"),
    ({"scores": torch.zeros(2, 2, 95)}, KernelError, "scores"),
    ({"scores": torch.zeros(2, 2, 96, dtype=torch.float64)}, KernelError, "scores"),
    ({"slot_positions": torch.zeros(2, 2, 96, dtype=torch.int64)}, KernelError, "slot_positions"),
    ({"kv_lens": torch.zeros(3, dtype=torch.int32)}, KernelError, "kv_lens"),
    ({"block_table": torch.zeros(2, dtype=torch.int32)}, KernelError, "block_table"),
    ({"k_pages": torch.zeros(1, 16, 2, 64, dtype=BF).expand(10, 16, 2, 64)}, KernelError, "overlap"),
    ({"v_pages": torch.zeros(10, 16, 2, 128, dtype=BF)[..., ::2]}, KernelError, "contiguous rows"),
    ({"v_pages": torch.zeros(10, 16, 2, 64)}, KernelError, "v_pages is"),
])
def test_evict_refusals(over, error, match):
    a = {"k_pages": torch.zeros(10, 16, 2, 64, dtype=BF), "v_pages": torch.zeros(10, 16, 2, 64, dtype=BF),
         "block_table": torch.zeros(2, 6, dtype=torch.int32), "kv_lens": torch.tensor([50, 20]),
         "scores": torch.zeros(2, 2, 96), "slot_positions": torch.zeros(2, 2, 96, dtype=torch.int32), "budget": 10}
    a.update(over)
    with pytest.raises(error, match=match):
        evict_paged(**a)


def test_chunk_splits():
    assert default_chunk_splits(1, 8, 4, 2048, 32768) == 1
    assert default_chunk_splits(1, 8, 4, 1, 64) == 1
    assert default_chunk_splits(1, 8, 4, 2100, 32768) == 3 and default_chunk_splits(1, 8, 4, 2100, 4096) == 1
    assert default_chunk_splits(1, 1, 8, 300, 131072) == 26 and default_chunk_splits(64, 8, 4, 1, 16384) == 4
    for n, hkv, g, chunk, slots in ((1, 8, 4, 1, 32768), (64, 8, 4, 1, 16384), (2, 4, 7, 256, 32768), (1, 1, 1, 1, 8)):
        for masked in (False, True):
            s = default_chunk_splits(n, hkv, g, chunk, slots, masked)
            assert 1 <= s <= 64 and s <= max(1, math.ceil(slots / 64))


def test_chunk_splits_of_an_empty_chunk():
    for masked in (False, True):
        assert default_chunk_splits(1, 8, 4, 0, 4096, masked) == 1
        assert default_chunk_splits(64, 2, 1, 0, 1 << 20, masked, 64) == 1


# ------------------------------------------------------------------------- the C entries
def _i64(*vals):
    return (ctypes.c_int64 * 4)(*vals)


FAKE = ctypes.c_void_p(16)  # never dereferenced: validation fails first
ODD = ctypes.c_void_p(18)


def _err():
    return _native.load_library().tasft_last_error()


def test_rotary_entry_refusals():
    lib = _native.load_library()
    st = _i64(4096, 1024, 128, 1)

    def call(q=FAKE, heads=4, kv=2, seq=8, d=128, r=128, sq=st, so=st, dtype=0, pos=FAKE):
        return lib.tasft_rotary(q, FAKE, FAKE, FAKE, pos, 1, FAKE, 2, heads, kv, seq, d, r, sq, st, so, st,
                                _i64(0, 1), 0, 0, 1.0, dtype, None)

    for args, rc, text in (({"q": None}, -1, b"null"), ({"pos": None}, -1, b"null"), ({"dtype": 2}, -2, b"dtype"),
                           ({"heads": 0}, -1, b"positive"), ({"d": 320, "r": 64}, -2, b"head_dim"),
                           ({"r": 130}, -1, b"rotary_dim"), ({"r": 7}, -1, b"rotary_dim"), ({"r": 0}, -1, b"rotary_dim"),
                           ({"seq": 0}, -1, b"positive"), ({"sq": _i64(-8, 0, 0, 1)}, -1, b"non-negative"),
                           ({"so": _i64(0, 0, 0, 2)}, -1, b"contiguous")):
        assert call(**args) == rc and text in _err(), args


def test_append_entry_refusals():
    lib = _native.load_library()
    st, pool = _i64(512, 128, 1, 0), _i64(4096, 256, 128, 1)

    def call(cu=FAKE, n=2, t=8, kv=2, page=16, pages=9, kp=pool, sq=st, dtype=1, bt=6):
        return lib.tasft_rotary_append_paged(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, cu, None, 0, FAKE, None, n,
                                             t, 4, kv, 128, 128, page, pages, 6, sq, st, st, st, kp, pool, bt, 0, 0, 1.0,
                                             dtype, None)

    for args, rc, text in (({"cu": None}, -1, b"null"), ({"n": 0}, -1, b"positive"), ({"kv": 0}, -1, b"positive"),
                           ({"page": 24}, -2, b"page_size"), ({"pages": 0}, -1, b"positive"),
                           ({"kp": _i64(4096, -8, 128, 1)}, -1, b"non-negative"), ({"bt": -1}, -1, b"non-negative"),
                           ({"kp": _i64(4096, 256, 128, 2)}, -1, b"contiguous"), ({"dtype": 5}, -2, b"dtype"),
                           ({"sq": _i64(512, 128, 2, 0)}, -1, b"contiguous")):
        assert call(**args) == rc and text in _err(), args
    assert call(t=0) == 0


def test_chunk_entry_refusals():
    lib = _native.load_library()
    st, pool, mask = _i64(512, 128, 1, 0), _i64(4096, 256, 128, 1), _i64(0, 0, 0, 1)
    assert lib.tasft_chunk_workspace_bytes(8, 4, 128, 1) == 0
    assert lib.tasft_chunk_workspace_bytes(8, 4, 128, 3) == 8 * 4 * 3 * 130 * 4

    def call(q=FAKE, v=FAKE, m=None, ws=None, wb=0, n=2, t=8, hq=4, hkv=2, longest=5, d=128, bs=64, rows=1, page=16,
             pages=9, per=6, splits=1, sq=st, kp=pool, vp=pool, so=st, scale=1.0, dtype=0):
        return lib.tasft_chunk_paged_fwd(q, FAKE, v, FAKE, None, m, FAKE, FAKE, FAKE, ws, wb, n, t, hq, hkv, longest, d,
                                         bs, rows, page, pages, per, splits, sq, kp, vp, so, mask if m else None, 6,
                                         scale, 1, dtype, None)

    for args, rc, text in (({"q": None}, -1, b"null"), ({"v": None}, -1, b"null"), ({"dtype": -1}, -2, b"dtype"),
                           ({"t": 0}, -1, b"positive"), ({"longest": 0}, -1, b"positive"), ({"hq": 5}, -1, b"multiple"),
                           ({"d": 96}, -2, b"head_dim"), ({"m": FAKE, "bs": 48}, -2, b"block_size"),
                           ({"m": FAKE, "rows": 0}, -1, b"positive"), ({"page": 4}, -2, b"page_size"),
                           ({"page": 12}, -2, b"page_size"), ({"scale": 0.0}, -1, b"scale"),
                           ({"per": 1 << 28}, -2, b"32 bits"), ({"q": ODD}, -1, b"aligned"), ({"v": ODD}, -1, b"aligned"),
                           ({"sq": _i64(516, 128, 1, 0)}, -1, b"multiples of 8"),
                           ({"kp": _i64(4096, 1 << 27, 128, 1)}, -2, b"too large"),
                           ({"vp": _i64(4096, 256, -128, 1)}, -1, b"non-negative"),
                           ({"so": _i64(512, 128, 2, 0)}, -1, b"contiguous"), ({"splits": 0}, -1, b"num_splits"),
                           ({"splits": 2000}, -1, b"num_splits"), ({"splits": 2}, -4, b"workspace"),
                           ({"splits": 2, "ws": FAKE, "wb": 100}, -4, b"workspace")):
        assert call(**args) == rc and text in _err(), args


def test_key_weight_entry_refusals():
    lib = _native.load_library()
    st, pool = _i64(512, 128, 1, 0), _i64(4096, 256, 128, 1)

    def call(lse=FAKE, scores=None, ss=None, sl=_i64(4, 1), d=64):
        return lib.tasft_key_weights(FAKE, FAKE, None, FAKE, FAKE, FAKE, lse, scores, FAKE, 2, 8, 4, 2, 5, d, 64, 0, 16,
                                     9, 6, st, pool, sl, ss, None, 6, 1.0, 1, 0, None)

    for args, rc, text in (({"lse": None}, -1, b"null"), ({"scores": FAKE}, -1, b"null"), ({"d": 32}, -2, b"head_dim"),
                           ({"sl": _i64(-4, 1)}, -1, b"non-negative"),
                           ({"scores": FAKE, "ss": _i64(0, 0, -1)}, -1, b"non-negative")):
        assert call(**args) == rc and text in _err(), args


def test_evict_entry_refusals():
    lib = _native.load_library()
    pool, st = _i64(4096, 256, 128, 1), _i64(192, 96, 1, 0)
    assert lib.tasft_evict_workspace_bytes(2, 2, 64, 10) == 4 * 21 * 4
    assert lib.tasft_evict_workspace_bytes(2, 2, 8, 10) == 4 * 17 * 4
    assert lib.tasft_evict_workspace_bytes(0, 2, 64, 10) == 0 == lib.tasft_evict_workspace_bytes(2, 2, 0, 10)
    # In parts of 8192 slots: three words each, three digits of three, three times 2048 counts each.
    assert lib.tasft_evict_workspace_bytes(2, 3, 40000, 10) == 6 * 4 * (21 + 15 + 9 + 15 * 2048)
    # At most 64 parts, of whole runs.
    assert lib.tasft_evict_workspace_bytes(1, 1, 1 << 20, 10) == 4 * (21 + 192 + 9 + 192 * 2048)
    assert lib.tasft_evict_workspace_bytes(1, 1, (1 << 19) + 1, 10) == 4 * (21 + 99 + 9 + 99 * 2048)

    def call(k=FAKE, wb=1 << 20, n=2, d=128, page=16, budget=10, recent=2, sinks=1, kp=pool, ss=st, per=6):
        return lib.tasft_evict_paged(k, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, wb, n, 2, d, page, 9, per,
                                     budget, recent, sinks, kp, pool, ss, st, 6, None)

    for args, rc, text in (({"k": None}, -1, b"null"), ({"n": 0}, -1, b"positive"), ({"budget": 0}, -1, b"positive"),
                           ({"recent": 10}, -1, b"fit the budget"), ({"sinks": -1}, -1, b"non-negative"),
                           ({"page": 20}, -2, b"page_size"), ({"d": 12}, -2, b"head_dim"), ({"d": 264}, -2, b"head_dim"),
                           ({"n": 40000}, -2, b"range"), ({"kp": _i64(4096, 256, 124, 1)}, -1, b"multiples of 8"),
                           ({"kp": _i64(4096, 256, 128, 2)}, -1, b"contiguous"), ({"k": ODD}, -1, b"aligned"),
                           ({"ss": _i64(0, 0, -1, 0)}, -1, b"non-negative"), ({"wb": 100}, -4, b"workspace")):
        assert call(**args) == rc and text in _err(), args


def test_launches_of_too_many_threads_are_refused():
    """A launch holds fewer than 2^32 threads: refused before anything is launched."""
    lib = _native.load_library()
    st, pool = _i64(64, 64, 1, 0), _i64(4096, 256, 128, 1)

    def chunk(n, t, longest, splits, heads=1):
        size = lib.tasft_chunk_workspace_bytes(t, heads, 64, splits)
        return lib.tasft_chunk_paged_fwd(FAKE, FAKE, FAKE, FAKE, None, None, FAKE, FAKE, FAKE, FAKE, size, n, t, heads,
                                         heads, longest, 64, 64, 0, 16, 9, 6, splits, st, pool, pool, st, None, 6, 1.0,
                                         1, 0, None)

    assert chunk(1 << 14, 1 << 17, 1 << 17, 1) == -2 and b"launch too large" in _err()      # 2^24 row tiles
    assert chunk(1, 1 << 20, 1, 9, 16) == -2 and b"launch too large" in _err()              # joined, a workgroup a row
    assert chunk(1, 1 << 20, 1, 8, 2048) == -2 and b"launch too large" in _err()            # joined, 16 rows a workgroup

    def weights(n, per):
        return lib.tasft_key_weights(FAKE, FAKE, None, FAKE, FAKE, FAKE, FAKE, None, FAKE, n, 8, 1, 1, 5, 64, 64, 0, 256,
                                     9, per, st, pool, _i64(4, 1), None, None, 6, 1.0, 1, 0, None)

    assert weights(1 << 14, 1 << 10) == -2 and b"launch too large" in _err()                # 2^24 times 256 keys


def test_evict_entry_refuses_outputs_that_are_inputs():
    """Lengths cut in place would be read again, shorter, by the launches behind."""
    lib = _native.load_library()
    pool, st = _i64(4096, 256, 128, 1), _i64(192, 96, 1, 0)
    a = [ctypes.c_void_p(16 * (i + 1)) for i in range(10)]  # never dereferenced

    def call(kv, scores, pos, kv_out, scores_out, pos_out):
        return lib.tasft_evict_paged(a[0], a[1], a[2], kv, scores, pos, kv_out, scores_out, pos_out, a[9], 1 << 20, 2, 2,
                                     128, 16, 9, 6, 10, 2, 1, pool, pool, st, st, 6, None)

    for same in ((3, 4, 5, 3, 7, 8), (3, 4, 5, 6, 4, 8), (3, 4, 5, 6, 7, 5)):
        assert call(*(a[i] for i in same)) == -1 and b"outputs" in _err(), same
