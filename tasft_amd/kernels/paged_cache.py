"""A paged KV cache around the attention that reads it: writing new tokens, weighing the cached
keys, evicting the light ones.

The pools are those of ``BlockSparseFlashAttention.forward_decode_paged`` and
``forward_chunk_paged``: ``[num_pages, page_size, Hkv, D]``, slot s of sequence n in row
``s % page_size`` of page ``block_table[n, s // page_size]``. A serving step of a chunk is

    q = append_paged(q, k, v, k_pages, v_pages, table, kv_lens, cu, inv_freq, slot_positions=pos)
    out, lse = attn.forward_chunk_paged(q, k_pages, v_pages, table, kv_lens, cu, return_lse=True)
    scores = accumulate_key_weights(q, k_pages, table, kv_lens, cu, lse, scores)
    kv_lens, scores, pos = evict_paged(k_pages, v_pages, table, kv_lens, scores, pos, budget)

with the last two only where a cache is bounded. Scores and positions are kept per KV head, since
each head keeps its own keys. The reference has no cache of its own (its vLLM backend leaves it to
vLLM, ``tasft/inference/vllm_patch.py:172-196``).
"""
from __future__ import annotations

import functools
import math
from typing import NamedTuple

import torch

from tasft_amd import _native
from tasft_amd.exceptions import KernelError
from tasft_amd.kernels.rotary import _new_like, _unit_last, check_frequencies, check_positions

_VALID_HEAD_DIMS = frozenset({64, 128})


class PagedBatch(NamedTuple):
    """Sizes of a packed batch over a paged cache, and its index tensors as the kernels read them."""

    num_seqs: int
    tokens: int
    max_seqlen: int
    page_size: int
    max_pages: int
    cu: torch.Tensor
    kv_lens: torch.Tensor
    table: torch.Tensor
    slots: int   # max_pages * page_size
    dtype: int   # the C interface's code


def int32_on(t: torch.Tensor, device: torch.device) -> torch.Tensor:
    """``t`` as a contiguous int32 tensor on ``device``, itself if it is one."""
    if t.dtype == torch.int32 and t.device == device and t.is_contiguous():
        return t
    return t.to(device=device, dtype=torch.int32).contiguous()


def check_pools(k_pages: torch.Tensor, v_pages: torch.Tensor) -> None:
    if k_pages.ndim != 4 or k_pages.shape != v_pages.shape or k_pages.numel() == 0:
        raise KernelError("page pools must be two of [num_pages, page_size, Hkv, D]",
                          context={"k": list(k_pages.shape), "v": list(v_pages.shape)})
    if k_pages.dtype != v_pages.dtype:
        raise KernelError(f"v_pages is {v_pages.dtype} but k_pages is {k_pages.dtype}",
                          context={"k": str(k_pages.dtype), "v": str(v_pages.dtype)})


def check_batch(q: torch.Tensor, k_pages: torch.Tensor, block_table: torch.Tensor, kv_lens: torch.Tensor,
                cu_seqlens: torch.Tensor, max_seqlen: int | None, min_page: int = 8,
                need_max: bool = True) -> PagedBatch:
    """The checks shared by the calls on a packed chunk over page pools."""
    qs, ks, cs, bs = q.shape, k_pages.shape, cu_seqlens.shape, block_table.shape
    if len(qs) != 3:
        raise KernelError(f"Expected packed q of shape [T, H, D], got {tuple(qs)}", context={"q_shape": list(qs)})
    T, H, D = qs
    if k_pages.dtype != q.dtype:
        raise KernelError(f"page pools are {k_pages.dtype} but q is {q.dtype}",
                          context={"q": str(q.dtype), "pages": str(k_pages.dtype)})
    code = _native.dtype_code(q.dtype, "paged cache")
    _, page_size, Hkv, Dk = ks
    if Dk != D or H == 0 or H % Hkv != 0:
        raise KernelError("page pools must have q's head_dim and Hq % Hkv == 0",
                          context={"q": list(qs), "pages": list(ks)})
    if page_size < min_page or page_size & (page_size - 1):
        raise KernelError(f"page_size must be a power of two >= {min_page}, got {page_size}",
                          context={"page_size": page_size})
    if len(cs) != 1 or cs[0] < 2:
        raise KernelError("cu_seqlens must be a 1-D tensor of N + 1 >= 2 offsets",
                          context={"cu_seqlens_shape": list(cs)})
    n = cs[0] - 1
    if len(bs) != 2 or bs[0] != n or bs[1] == 0:
        raise KernelError(f"block_table must have shape [{n}, max_pages], got {tuple(bs)}",
                          context={"block_table": list(bs)})
    if kv_lens.shape != (n,):
        raise KernelError(f"kv_lens must have shape ({n},), got {tuple(kv_lens.shape)}",
                          context={"kv_lens": list(kv_lens.shape)})
    slots = bs[1] * page_size
    lens = None
    if cu_seqlens.is_cpu:
        cu = cu_seqlens.to(torch.int64)
        lens = cu[1:] - cu[:-1]
        if int(cu[0]) != 0 or bool((lens < 0).any()) or int(cu[-1]) > T:
            raise KernelError("cu_seqlens must start at 0, be non-decreasing and end at <= T",
                              context={"cu_seqlens": cu.tolist()[:16], "T": T})
        longest = int(lens.max())
        if max_seqlen is None:
            max_seqlen = max(longest, 1)
        elif longest > max_seqlen:
            raise KernelError(f"a sequence has {longest} tokens, more than max_seqlen={max_seqlen}",
                              context={"max_seqlen": max_seqlen, "longest": longest})
    elif max_seqlen is None and need_max:
        raise KernelError("max_seqlen is required when cu_seqlens is on the device",
                          context={"device": str(cu_seqlens.device)})
    if kv_lens.is_cpu:
        kv = kv_lens.to(torch.int64)
        if bool((kv < 0).any()) or int(kv.max()) > slots or (lens is not None and bool((kv < lens).any())):
            raise KernelError(f"kv_lens must hold the chunk and be at most max_pages * page_size = {slots}",
                              context={"kv_lens": kv.tolist()[:16], "slots": slots})
    if max_seqlen is not None and max_seqlen <= 0:
        raise KernelError(f"max_seqlen must be positive, got {max_seqlen}", context={"max_seqlen": max_seqlen})
    dev = q.device
    if not q.is_cuda or k_pages.device != dev:
        raise KernelError("Tensors must be on one CUDA device", context={"q": str(dev), "pages": str(k_pages.device)})
    return PagedBatch(n, T, max_seqlen or 0, page_size, bs[1], int32_on(cu_seqlens, dev), int32_on(kv_lens, dev),
                      int32_on(block_table, dev), slots, code)


def chunk_mask(block_mask: torch.Tensor, batch: PagedBatch, heads: int, block_size: int,
               device: torch.device) -> torch.Tensor:
    """A chunk's block mask as bytes: ``[N, Hq, R, NB]``, R the query blocks that ``max_seqlen``
    tokens can touch."""
    rows = (batch.max_seqlen + block_size - 2) // block_size + 1
    want = (batch.num_seqs, heads, rows, math.ceil(batch.slots / block_size))
    if tuple(block_mask.shape) != want:
        raise KernelError(f"block_mask shape mismatch: expected {want}, got {tuple(block_mask.shape)}",
                          context={"expected": list(want), "got": list(block_mask.shape)})
    mask = block_mask if block_mask.device == device else block_mask.to(device)
    if mask.dtype in (torch.bool, torch.int8):
        return mask.view(torch.uint8)
    return mask if mask.dtype == torch.uint8 else (mask != 0).view(torch.uint8)


def readable(t: torch.Tensor) -> torch.Tensor:
    """``t`` if its layout suits the attention kernels (16-byte rows), else a copy."""
    return t if _native.kernel_layout(t) else t.clone(memory_format=torch.contiguous_format)


@functools.lru_cache(maxsize=1024)
def _overlaps(shape: tuple[int, ...], strides: tuple[int, ...]) -> bool:
    expect = 1
    for size, stride in sorted(((n, s) for n, s in zip(shape, strides) if n > 1), key=lambda x: x[1]):
        if stride < expect:
            return True
        expect = stride * size
    return False


def writable_pool(t: torch.Tensor, what: str, rows16: bool) -> None:
    """Refuses pools that cannot be written in place: overlapping elements, or rows that the
    kernel does not address."""
    if _overlaps(t.shape, t.stride()):
        raise KernelError(f"{what} must not overlap itself (an expanded pool cannot be written)",
                          context={"strides": list(t.stride())})
    if t.stride(-1) != 1 or (rows16 and not _native.kernel_layout(t)):
        raise KernelError(f"{what} must have contiguous rows" + (", 16-byte aligned" if rows16 else ""),
                          context={"strides": list(t.stride())})


def _slot_state(t: torch.Tensor, shape: tuple[int, ...], dtype: torch.dtype, device: torch.device,
                what: str) -> None:
    if tuple(t.shape) != shape or t.dtype != dtype or t.device != device:
        raise KernelError(f"{what} must be {dtype} of shape {shape} on {device}, got {t.dtype} "
                          f"{tuple(t.shape)} on {t.device}", context={"shape": list(t.shape)})


def append_paged(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    block_table: torch.Tensor,
    kv_lens: torch.Tensor,
    cu_seqlens: torch.Tensor,
    inv_freq: torch.Tensor,
    *,
    positions: torch.Tensor | None = None,
    interleaved: bool = False,
    scale: float = 1.0,
    slot_positions: torch.Tensor | None = None,
) -> torch.Tensor:
    """New tokens rotated and written into the pages of their sequences, in one launch.

    Args:
        q, k, v: ``[T, Hq, D]`` and ``[T, Hkv, D]`` of the packed new tokens, before the rotation
            (bf16 or fp16, the pools' dtype).
        k_pages, v_pages: ``[num_pages, page_size, Hkv, D]`` pools, written in place, in any layout of
            contiguous rows. (The attention and the key weights copy, at every call, pools whose base
            is not 16-byte aligned or whose strides are not multiples of 8.)
        block_table: ``[N, max_pages]`` int32. A token whose page lies outside the pool (or whose
            slot outside the table) is rotated but not written.
        kv_lens: ``[N]`` lengths with the new tokens: token i of a sequence's ``len`` goes to slot
            ``kv_lens[n] - len + i``.
        cu_seqlens: ``[N + 1]`` offsets of the sequences' tokens, as in ``forward_varlen``.
        inv_freq, interleaved, scale: as in ``apply_rotary``.
        positions: ``[T]`` int32 or int64 positions (default: the tokens' slots, right as long as
            nothing was evicted).
        slot_positions: ``[N, Hkv, max_pages * page_size]`` int32 contiguous, receives each new
            token's position at its slot (what ``evict_paged`` reads; its low 32 bits).

    Returns:
        The rotated queries ``[T, Hq, D]`` (0 for tokens behind ``cu_seqlens[N]``, which are not
        written to the pages). No gradients.
    """
    check_pools(k_pages, v_pages)
    b = check_batch(q, k_pages, block_table, kv_lens, cu_seqlens, None, min_page=1, need_max=False)
    T, H, D = q.shape
    Hkv = k_pages.shape[2]
    dev = q.device
    for name, t in (("k", k), ("v", v)):
        if tuple(t.shape) != (T, Hkv, D) or t.dtype != q.dtype or t.device != dev:
            raise KernelError(f"{name} must be {q.dtype} of shape {(T, Hkv, D)} on {dev}, got {t.dtype} "
                              f"{tuple(t.shape)} on {t.device}", context={"shape": list(t.shape)})
    if v_pages.device != dev:
        raise KernelError("Tensors must be on one CUDA device", context={"v_pages": str(v_pages.device)})
    writable_pool(k_pages, "k_pages", False)
    writable_pool(v_pages, "v_pages", False)
    inv_freq = check_frequencies(inv_freq, D, dev)
    if positions is not None:
        if tuple(positions.shape) != (T,):
            raise KernelError(f"positions must have shape ({T},), got {tuple(positions.shape)}",
                              context={"positions": list(positions.shape)})
        positions = check_positions(positions, dev)
    if slot_positions is not None:
        _slot_state(slot_positions, (b.num_seqs, Hkv, b.slots), torch.int32, dev, "slot_positions")
        if not slot_positions.is_contiguous():
            raise KernelError("slot_positions must be contiguous", context={"strides": list(slot_positions.stride())})
    q, k, v = _unit_last(q), _unit_last(k), _unit_last(v)
    out = _new_like(q)
    if T == 0:
        return out
    lib = _native.load_library()
    with _native.on_device(dev):
        status = lib.tasft_rotary_append_paged(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(),
            b.table.data_ptr(), b.kv_lens.data_ptr(), b.cu.data_ptr(), _native.ptr(positions),
            1 if positions is not None and positions.dtype == torch.int64 else 0, inv_freq.data_ptr(),
            _native.ptr(slot_positions), b.num_seqs, T, H, Hkv, D, 2 * inv_freq.numel(), b.page_size,
            k_pages.shape[0], b.max_pages, _native.strides(q), _native.strides(k), _native.strides(v),
            _native.strides(out), _native.strides(k_pages), _native.strides(v_pages), b.table.stride(0),
            positions.stride(0) if positions is not None else 0, 1 if interleaved else 0, float(scale),
            b.dtype, _native.stream_handle(dev))
    _native.check(status, "tasft_rotary_append_paged", {"tokens": T, "sequences": b.num_seqs})
    return out


def accumulate_key_weights(
    q: torch.Tensor,
    k_pages: torch.Tensor,
    block_table: torch.Tensor,
    kv_lens: torch.Tensor,
    cu_seqlens: torch.Tensor,
    lse: torch.Tensor,
    scores: torch.Tensor | None = None,
    *,
    block_mask: torch.Tensor | None = None,
    block_size: int = 64,
    max_seqlen: int | None = None,
    causal: bool = True,
) -> torch.Tensor:
    """The attention weight every cached key received from a chunk, added to ``scores``.

    ``out[n, g, j] = scores[n, g, j] + sum of softmax weights`` over the chunk's tokens and the
    query heads of KV head g that see key j, from the attention's ``lse`` (one product instead of
    two, no values read). To weigh a window alone, pass its queries, offsets and ``lse``.

    Args:
        q, k_pages, block_table, kv_lens, cu_seqlens, block_mask, max_seqlen, causal: as given to
            ``forward_chunk_paged`` (``block_size``: that of the attention object).
        lse: ``[T, Hq]`` fp32, its second result (of plain scores: a cap, slopes and a tree are not known here).
        scores: ``[N, Hkv, max_pages * page_size]`` fp32, or None for zeros; not changed.

    Returns:
        ``[N, Hkv, max_pages * page_size]`` fp32; slots at or past ``kv_lens[n]`` keep their score.
    """
    if k_pages.ndim != 4 or k_pages.numel() == 0:
        raise KernelError("page pools must be [num_pages, page_size, Hkv, D]", context={"k": list(k_pages.shape)})
    b = check_batch(q, k_pages, block_table, kv_lens, cu_seqlens, max_seqlen)
    T, H, D = q.shape
    Hkv = k_pages.shape[2]
    dev = q.device
    if D not in _VALID_HEAD_DIMS:
        raise KernelError(f"HIP kernel supports head_dim in {sorted(_VALID_HEAD_DIMS)}, got {D}",
                          context={"head_dim": D})
    if block_size not in (32, 64, 128):
        raise ValueError(f"block_size must be one of [32, 64, 128], got {block_size}")
    _slot_state(lse, (T, H), torch.float32, dev, "lse")
    shape = (b.num_seqs, Hkv, b.slots)
    if scores is not None:
        _slot_state(scores, shape, torch.float32, dev, "scores")
    mask = None if block_mask is None else chunk_mask(block_mask, b, H, block_size, dev)
    if T == 0:
        return torch.zeros(shape, dtype=torch.float32, device=dev) if scores is None else scores.clone()
    q, k_pages = readable(q), readable(k_pages)
    out = (torch.empty_like(scores) if scores is not None and scores.is_contiguous()
           else torch.empty(shape, dtype=torch.float32, device=dev))
    lib = _native.load_library()
    with _native.on_device(dev):
        status = lib.tasft_key_weights(
            q.data_ptr(), k_pages.data_ptr(), _native.ptr(mask), b.table.data_ptr(), b.kv_lens.data_ptr(),
            b.cu.data_ptr(), lse.data_ptr(), _native.ptr(scores), out.data_ptr(), b.num_seqs, T, H, Hkv,
            b.max_seqlen, D, block_size, 0 if mask is None else mask.shape[2], b.page_size, k_pages.shape[0],
            b.max_pages, _native.strides(q), _native.strides(k_pages), _native.strides(lse),
            None if scores is None else _native.strides(scores), None if mask is None else _native.strides(mask),
            b.table.stride(0), 1.0 / math.sqrt(D), 1 if causal else 0, b.dtype, _native.stream_handle(dev))
    _native.check(status, "tasft_key_weights", {"tokens": T, "sequences": b.num_seqs})
    return out


def evict_paged(
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    block_table: torch.Tensor,
    kv_lens: torch.Tensor,
    scores: torch.Tensor,
    slot_positions: torch.Tensor,
    budget: int,
    *,
    recent: int = 0,
    sinks: int = 0,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Cuts every sequence's cache to ``budget`` keys per KV head, in place.

    Each head keeps the keys at positions below ``sinks``, those less than ``recent`` positions
    behind its newest, and then the heaviest by ``scores`` (NaN first, ties to the lowest slot).
    Kept keys behind the budget move into the slots it frees, so the keys of a head are no longer in
    order; every one of them is older than the tokens appended next, which is all that causal
    attention asks. Block masks, which select by slot, lose their meaning for such a cache.

    Args:
        k_pages, v_pages: the pools (bf16 or fp16, head_dim a multiple of 8), changed in place.
            No page may belong to two sequences, or twice to one.
        block_table: ``[N, max_pages]`` int32; kv_lens: ``[N]``.
        scores: ``[N, Hkv, max_pages * page_size]`` fp32 (``accumulate_key_weights``).
        slot_positions: the same shape, int32 (``append_paged``).
        budget: keys kept per head, at least ``recent + sinks``.

    Returns:
        ``(kv_lens, scores, slot_positions)`` of the smaller caches, new tensors: lengths
        ``min(kv_lens, budget)`` int32, and scores and positions at the keys' present slots, 0 and
        -1 behind them.
    """
    check_pools(k_pages, v_pages)
    _native.dtype_code(k_pages.dtype, "evict")
    P, page_size, Hkv, D = k_pages.shape
    dev = k_pages.device
    if page_size & (page_size - 1):
        raise KernelError(f"page_size must be a power of two, got {page_size}", context={"page_size": page_size})
    if D % 8 != 0 or D > 256:
        raise KernelError(f"HIP kernel supports head_dim a multiple of 8 up to 256, got {D}", context={"head_dim": D})
    if block_table.ndim != 2 or block_table.numel() == 0:
        raise KernelError(f"block_table must have shape [N, max_pages], got {tuple(block_table.shape)}",
                          context={"block_table": list(block_table.shape)})
    n, max_pages = block_table.shape
    if kv_lens.shape != (n,):
        raise KernelError(f"kv_lens must have shape ({n},), got {tuple(kv_lens.shape)}",
                          context={"kv_lens": list(kv_lens.shape)})
    if budget <= 0:
        raise ValueError(f"budget must be positive, got {budget}")
    if recent < 0 or sinks < 0 or recent + sinks > budget:
        raise ValueError(f"recent ({recent}) and sinks ({sinks}) must be non-negative and fit the budget ({budget})")
    shape = (n, Hkv, max_pages * page_size)
    _slot_state(scores, shape, torch.float32, dev, "scores")
    _slot_state(slot_positions, shape, torch.int32, dev, "slot_positions")
    writable_pool(k_pages, "k_pages", True)
    writable_pool(v_pages, "v_pages", True)
    if not k_pages.is_cuda or v_pages.device != dev:
        raise KernelError("Tensors must be on one CUDA device",
                          context={"k_pages": str(dev), "v_pages": str(v_pages.device)})
    table, lens = int32_on(block_table, dev), int32_on(kv_lens, dev)
    if budget >= shape[2]:  # nothing to evict
        budget, recent, sinks = shape[2], 0, 0
    lib = _native.load_library()
    ws_bytes = lib.tasft_evict_workspace_bytes(n, Hkv, shape[2], budget)
    workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
    lens_out = torch.empty((n,), dtype=torch.int32, device=dev)
    contiguous = scores.is_contiguous() and slot_positions.is_contiguous()
    scores_out = torch.empty_like(scores) if contiguous else torch.empty(shape, dtype=torch.float32, device=dev)
    pos_out = torch.empty_like(slot_positions) if contiguous else torch.empty(shape, dtype=torch.int32, device=dev)
    with _native.on_device(dev):
        status = lib.tasft_evict_paged(
            k_pages.data_ptr(), v_pages.data_ptr(), table.data_ptr(), lens.data_ptr(), scores.data_ptr(),
            slot_positions.data_ptr(), lens_out.data_ptr(), scores_out.data_ptr(), pos_out.data_ptr(),
            workspace.data_ptr(), ws_bytes, n, Hkv, D, page_size, P, max_pages, budget, recent, sinks,
            _native.strides(k_pages), _native.strides(v_pages), _native.strides(scores),
            _native.strides(slot_positions), table.stride(0), _native.stream_handle(dev))
    _native.check(status, "tasft_evict_paged", {"sequences": n, "slots": shape[2], "budget": budget})
    return lens_out, scores_out, pos_out


__all__ = ["accumulate_key_weights", "append_paged", "evict_paged"]
