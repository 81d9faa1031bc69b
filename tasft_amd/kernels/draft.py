"""Trees of drafted tokens over a paged cache: their plan, which tokens are kept, and the kept tokens'
keys and values.

A step of a server that drafts trees (the root is the last token that it produced):

    tree = draft_tree(parents, cu, kv_lens, max_nodes=most)
    q = append_paged(q, k, v, k_pages, v_pages, table, kv_lens, cu, inv_freq, positions=tree.positions)
    out = attn.forward_chunk_paged(q, k_pages, v_pages, table, kv_lens, cu, max_seqlen=most,
                                   ancestors=tree.ancestors)
    kept = accept_draft(parents, tokens, targets, cu, max_nodes=most)
    new_lens = commit_draft_paged(k_pages, v_pages, table, kv_lens, cu, kept.path, kept.counts)

with the appending, the attention and the commit in every layer (from the same ``kv_lens``: the new lengths are the
same for all of them). The reference drafts nothing (its vLLM
backend hands decoding back to vLLM, ``tasft/inference/vllm_patch.py:189-196``).
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from tasft_amd import _native
from tasft_amd.exceptions import KernelError
from tasft_amd.kernels.paged_cache import _slot_state, check_pools, int32_on, writable_pool

_MAX_NODES = 4096


class DraftTree(NamedTuple):
    """``ancestors`` ``[T, ceil(max_nodes / 64)]`` int64: bit a % 64 of word a // 64 is set for node a itself
    and its ancestors. ``positions`` ``[T]`` int32."""

    ancestors: torch.Tensor
    positions: torch.Tensor


class AcceptedDraft(NamedTuple):
    """``path`` ``[N, max_nodes]`` int32: the kept nodes from a root down, -1 behind them. ``counts`` ``[N]``
    int32. ``next_tokens`` ``[N]``: the target's token behind the last kept node."""

    path: torch.Tensor
    counts: torch.Tensor
    next_tokens: torch.Tensor


def _check_tree(parents: torch.Tensor, cu_seqlens: torch.Tensor, max_nodes: int | None) -> int:
    """Checks the tree's description; returns max_nodes."""
    if parents.ndim != 1 or parents.dtype not in (torch.int32, torch.int64):
        raise KernelError(f"parents must be int32 or int64 of shape [T], got {parents.dtype} {tuple(parents.shape)}",
                          context={"parents": list(parents.shape)})
    if cu_seqlens.ndim != 1 or cu_seqlens.numel() < 2:
        raise KernelError("cu_seqlens must be a 1-D tensor of N + 1 >= 2 offsets",
                          context={"cu_seqlens_shape": list(cu_seqlens.shape)})
    if cu_seqlens.is_cpu:
        cu = cu_seqlens.to(torch.int64)
        lens = cu[1:] - cu[:-1]
        if int(cu[0]) != 0 or bool((lens < 0).any()) or int(cu[-1]) > parents.numel():
            raise KernelError("cu_seqlens must start at 0, be non-decreasing and end at <= T",
                              context={"cu_seqlens": cu.tolist()[:16], "T": parents.numel()})
        longest = int(lens.max())
        if max_nodes is None:
            max_nodes = max(longest, 1)
        elif longest > max_nodes:
            raise KernelError(f"a tree has {longest} nodes, more than max_nodes={max_nodes}",
                              context={"max_nodes": max_nodes, "longest": longest})
        if parents.is_cpu:
            at = torch.cat([torch.arange(int(x)) for x in lens])
            p = parents[:int(cu[-1])].to(torch.int64)
            if bool((p < -1).any()) or bool((p >= at).any()):
                raise KernelError("a node's parent must be a node of its tree before it, or -1",
                                  context={"parents": p.tolist()[:16]})
    elif max_nodes is None:
        raise KernelError("max_nodes is required when cu_seqlens is on the device",
                          context={"device": str(cu_seqlens.device)})
    if not 0 < max_nodes <= _MAX_NODES:
        raise KernelError(f"max_nodes must be in [1, {_MAX_NODES}], got {max_nodes}", context={"max_nodes": max_nodes})
    return max_nodes


def _nodes_on(nodes: torch.Tensor, device: torch.device) -> torch.Tensor:
    """Indices of nodes (or how many there are) as the kernels read them; what 32 bits do not hold stays no node."""
    if nodes.dtype == torch.int64:
        nodes = nodes.clamp(-1, 0x7fffffff)
    return int32_on(nodes, device)


def draft_tree(parents: torch.Tensor, cu_seqlens: torch.Tensor, kv_lens: torch.Tensor, *,
               max_nodes: int | None = None) -> DraftTree:
    """Ancestors and positions of the nodes of drafted trees, in one launch for all layers of a step.

    Args:
        parents: ``[T]`` int32 or int64: the index within its own sequence's nodes of each packed node's
            parent, a node before it; -1 for a node that follows the cache directly. (On the device anything
            that is no earlier node counts as -1.)
        cu_seqlens: ``[N + 1]`` offsets of the sequences' nodes.
        kv_lens: ``[N]`` cached lengths, the nodes included: a root's position is ``kv_lens[n] - len_n``.
        max_nodes: the most nodes of a tree (at most 4096; default: from a CPU ``cu_seqlens``). A tree's nodes
            behind its first ``max_nodes`` have no bits.

    Returns:
        ``DraftTree`` for ``append_paged(positions=)`` and ``forward_chunk_paged(ancestors=)``; rows behind
        ``cu_seqlens[N]`` are 0.
    """
    most = _check_tree(parents, cu_seqlens, max_nodes)
    n, T = cu_seqlens.numel() - 1, parents.numel()
    if kv_lens.shape != (n,):
        raise KernelError(f"kv_lens must have shape ({n},), got {tuple(kv_lens.shape)}",
                          context={"kv_lens": list(kv_lens.shape)})
    dev = parents.device if parents.is_cuda else kv_lens.device
    if dev.type != "cuda":
        raise KernelError("parents or kv_lens must be on a CUDA device", context={"device": str(dev)})
    ancestors = torch.empty((T, (most + 63) // 64), dtype=torch.int64, device=dev)
    positions = torch.empty((T,), dtype=torch.int32, device=dev)
    if T == 0:
        return DraftTree(ancestors, positions)
    parents, cu, lens = _nodes_on(parents, dev), int32_on(cu_seqlens, dev), int32_on(kv_lens, dev)
    with _native.on_device(dev):
        status = _native.load_library().tasft_draft_tree(
            parents.data_ptr(), cu.data_ptr(), lens.data_ptr(), ancestors.data_ptr(), positions.data_ptr(), n, T, most,
            _native.stream_handle(dev))
    _native.check(status, "tasft_draft_tree", {"tokens": T, "sequences": n})
    return DraftTree(ancestors, positions)


def accept_draft(parents: torch.Tensor, tokens: torch.Tensor, targets: torch.Tensor, cu_seqlens: torch.Tensor, *,
                 first_targets: torch.Tensor | None = None, max_nodes: int | None = None) -> AcceptedDraft:
    """The longest path down each tree whose tokens are what the target would have chosen.

    A node is kept if its token is the target's choice behind its parent and its parent is kept; a root is
    kept, or with ``first_targets`` if its token is that. Of several deepest kept nodes the lowest ends the
    path.

    Args:
        parents, cu_seqlens, max_nodes: as in ``draft_tree``.
        tokens: ``[T]`` int32 or int64 drafted tokens on the device; targets: ``[T]`` of the same type, the
            target's choice behind each node.
        first_targets: ``[N]`` of the same type: the target's choice behind the cache, where the trees do not
            start with the last token.

    Returns:
        ``AcceptedDraft``; where nothing is kept the next token is ``first_targets[n]``, or -1 without.
    """
    most = _check_tree(parents, cu_seqlens, max_nodes)
    n, T, dev = cu_seqlens.numel() - 1, parents.numel(), tokens.device
    if tokens.dtype not in (torch.int32, torch.int64) or tuple(tokens.shape) != (T,):
        raise KernelError(f"tokens must be int32 or int64 of shape ({T},), got {tokens.dtype} {tuple(tokens.shape)}",
                          context={"tokens": list(tokens.shape)})
    _slot_state(targets, (T,), tokens.dtype, dev, "targets")
    if first_targets is not None:
        _slot_state(first_targets, (n,), tokens.dtype, dev, "first_targets")
        first_targets = first_targets.contiguous()
    if dev.type != "cuda":
        raise KernelError("Tensors must be on CUDA device", context={"device": str(dev)})
    path = torch.empty((n, most), dtype=torch.int32, device=dev)
    counts = torch.empty((n,), dtype=torch.int32, device=dev)
    following = torch.empty((n,), dtype=tokens.dtype, device=dev)
    if T == 0:
        following = following.fill_(-1) if first_targets is None else first_targets.clone()
        return AcceptedDraft(path.fill_(-1), counts.zero_(), following)
    parents, cu = _nodes_on(parents, dev), int32_on(cu_seqlens, dev)
    tokens, targets = tokens.contiguous(), targets.contiguous()
    with _native.on_device(dev):
        status = _native.load_library().tasft_draft_accept(
            parents.data_ptr(), tokens.data_ptr(), targets.data_ptr(), _native.ptr(first_targets), cu.data_ptr(),
            path.data_ptr(), counts.data_ptr(), following.data_ptr(), n, T, most,
            1 if tokens.dtype == torch.int64 else 0, _native.stream_handle(dev))
    _native.check(status, "tasft_draft_accept", {"tokens": T, "sequences": n})
    return AcceptedDraft(path, counts, following)


def commit_draft_paged(
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    block_table: torch.Tensor,
    kv_lens: torch.Tensor,
    cu_seqlens: torch.Tensor,
    path: torch.Tensor,
    counts: torch.Tensor,
    *,
    slot_positions: torch.Tensor | None = None,
) -> torch.Tensor:
    """Moves the keys and values of the kept nodes of each tree to the slots behind its cache, in place.

    Args:
        k_pages, v_pages: ``[num_pages, page_size, Hkv, D]`` pools (bf16 or fp16, D a multiple of 8 up to
            256), changed in place. No page may belong to two sequences, or twice to one.
        block_table: ``[N, max_pages]``; kv_lens: ``[N]``, all nodes included, cu_seqlens: ``[N + 1]``, as in the
            step's other calls.
        path: ``[N, W]`` rising node indices, counts: ``[N]`` how many of them (``accept_draft``). An index that
            is not past its own place in the path, or is no node, is not moved.
        slot_positions: ``[N, Hkv, max_pages * page_size]`` int32 contiguous, if kept: moved alike.

    Returns:
        ``[N]`` int32 lengths ``kv_lens - len + counts``, a new tensor. What lies in the slots behind them is
        not defined.
    """
    check_pools(k_pages, v_pages)
    _native.dtype_code(k_pages.dtype, "commit")
    P, page_size, Hkv, D = k_pages.shape
    dev = k_pages.device
    if page_size & (page_size - 1):
        raise KernelError(f"page_size must be a power of two, got {page_size}", context={"page_size": page_size})
    if D % 8 != 0 or D > 256:
        raise KernelError(f"HIP kernel supports head_dim a multiple of 8 up to 256, got {D}", context={"head_dim": D})
    if cu_seqlens.ndim != 1 or cu_seqlens.numel() < 2:
        raise KernelError("cu_seqlens must be a 1-D tensor of N + 1 >= 2 offsets",
                          context={"cu_seqlens_shape": list(cu_seqlens.shape)})
    n = cu_seqlens.numel() - 1
    if block_table.ndim != 2 or block_table.shape[0] != n or block_table.shape[1] == 0:
        raise KernelError(f"block_table must have shape [{n}, max_pages], got {tuple(block_table.shape)}",
                          context={"block_table": list(block_table.shape)})
    for name, t in (("kv_lens", kv_lens), ("counts", counts)):
        if t.shape != (n,):
            raise KernelError(f"{name} must have shape ({n},), got {tuple(t.shape)}", context={name: list(t.shape)})
    if path.ndim != 2 or path.shape[0] != n:
        raise KernelError(f"path must have shape [{n}, W], got {tuple(path.shape)}", context={"path": list(path.shape)})
    max_pages = block_table.shape[1]
    writable_pool(k_pages, "k_pages", True)
    writable_pool(v_pages, "v_pages", True)
    if slot_positions is not None:
        _slot_state(slot_positions, (n, Hkv, max_pages * page_size), torch.int32, dev, "slot_positions")
        if not slot_positions.is_contiguous():
            raise KernelError("slot_positions must be contiguous", context={"strides": list(slot_positions.stride())})
    if not k_pages.is_cuda or v_pages.device != dev:
        raise KernelError("Tensors must be on one CUDA device",
                          context={"k_pages": str(dev), "v_pages": str(v_pages.device)})
    table, lens, cu = int32_on(block_table, dev), int32_on(kv_lens, dev), int32_on(cu_seqlens, dev)
    path, counts = _nodes_on(path, dev), _nodes_on(counts, dev)
    out = torch.empty((n,), dtype=torch.int32, device=dev)
    with _native.on_device(dev):
        status = _native.load_library().tasft_draft_commit_paged(
            k_pages.data_ptr(), v_pages.data_ptr(), table.data_ptr(), lens.data_ptr(), cu.data_ptr(), path.data_ptr(),
            counts.data_ptr(), out.data_ptr(), _native.ptr(slot_positions), n, path.shape[1], Hkv, D,
            page_size, P, max_pages, _native.strides(k_pages), _native.strides(v_pages), table.stride(0),
            _native.stream_handle(dev))
    _native.check(status, "tasft_draft_commit_paged", {"sequences": n})
    return out


__all__ = ["AcceptedDraft", "DraftTree", "accept_draft", "commit_draft_paged", "draft_tree"]
