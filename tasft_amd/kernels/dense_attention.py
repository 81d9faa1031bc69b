"""Dense attention of a training step, forward and backward, with capped and biased scores, packed
documents and prefixes.

The reference trains its gates beside attention that it computes densely, storing the
``[B, H, S, S]`` scores (``tasft/modules/tasft_attention.py:426-466``); ``gate_target_from_qk`` takes
the gate's target from Q and K without them (of scores without a cap or slopes), and ``dense_attention``
the attention itself. Serving has the same scores in ``BlockSparseFlashAttention.forward_chunk_paged``.
"""
from __future__ import annotations

import functools
import math

import torch
from torch.autograd import forward_ad

from tasft_amd import _native
from tasft_amd._autograd import first_order_only
from tasft_amd.exceptions import KernelError
from tasft_amd.kernels.paged_cache import int32_on

_VALID_HEAD_DIMS = frozenset({64, 128})


def check_softcap(softcap: float | None) -> float:
    """The cap as the C interface takes it (0: none)."""
    if softcap is None:
        return 0.0
    softcap = float(softcap)
    if not 1e-30 <= softcap <= 1e30:
        raise ValueError(f"softcap must be positive and finite (1e-30 to 1e30), got {softcap}")
    return softcap


def check_slopes(alibi_slopes: torch.Tensor | None, heads: int, device: torch.device) -> torch.Tensor | None:
    """``alibi_slopes`` as the kernels read it (contiguous fp32 on ``device``)."""
    if alibi_slopes is None:
        return None
    if tuple(alibi_slopes.shape) != (heads,) or not alibi_slopes.is_floating_point():
        raise KernelError(f"alibi_slopes must be floating point of shape ({heads},), got {alibi_slopes.dtype} "
                          f"{tuple(alibi_slopes.shape)}", context={"alibi_slopes": list(alibi_slopes.shape)})
    if alibi_slopes.requires_grad:
        raise KernelError("alibi_slopes must not require grad: the bias has no gradient for it", context={})
    if alibi_slopes.dtype == torch.float32 and alibi_slopes.device == device and alibi_slopes.is_contiguous():
        return alibi_slopes
    return alibi_slopes.to(device=device, dtype=torch.float32).contiguous()


def _ready(t: torch.Tensor) -> torch.Tensor:
    return t if _native.kernel_layout(t) else t.clone(memory_format=torch.contiguous_format)


def _new_like(t: torch.Tensor) -> torch.Tensor:
    """A new tensor of t's layout where the kernels can write that, else contiguous."""
    out = torch.empty_like(t)
    return out if _native.kernel_layout(out) else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _strides4(st: tuple[int, ...]):
    """(b, h, s, d) strides of ``[B, H, S, D]``, or of packed ``[T, H, D]`` as one batch entry, from a tensor's."""
    return _native.kept_strides(st if len(st) == 4 else (0, st[1], st[0], st[2]))


def _strides3(st: tuple[int, ...]):
    """(b, h, s) strides of ``[B, H, S]``, or of ``[T, H]``, from a tensor's."""
    return _native.kept_strides(st if len(st) == 3 else (0, st[1], st[0]))


class _Call:
    """What a call's kernels take beside the tensors that they differentiate."""

    __slots__ = ("causal", "cu", "dtype", "layout", "lens", "longest", "num_seqs", "prefix", "scale", "sizes", "slopes",
                 "softcap", "strides", "tokens")


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(num_seqs: int, rows: int, *sizes: int) -> int:
    return _native.load_library().tasft_dense_bwd_workspace_bytes(num_seqs, rows, *sizes)


def _forward(q, k, v, c: _Call, want_lse: bool, want_kept: bool):
    """out, its log-sums (or None), and what the backward needs beside them (or None): what out's rounding left
    over, a byte an element, and behind it the log-sums if they are not wanted."""
    out = _new_like(q)
    dev = q.device
    lse, kept, lse_ptr, rest_ptr = None, None, None, None
    rows = q.numel() // q.shape[-1]
    if want_lse:
        # A head's sums lie together: that is how the kernels read them.
        lse = (torch.empty(q.shape[:3], dtype=torch.float32, device=dev) if q.ndim == 4
               else torch.empty((q.shape[1], q.shape[0]), dtype=torch.float32, device=dev).t())
        lse_ptr = lse.data_ptr()
    if want_kept:
        kept = torch.empty((q.numel() + (0 if want_lse else 4 * rows),), dtype=torch.int8, device=dev)
        rest_ptr = kept.data_ptr()
        if not want_lse:
            lse_ptr = rest_ptr + q.numel()
    if q.numel() == 0:
        return out, lse, kept
    # (b, h, s) strides of the log-sums, [B, H, S] or the transpose of [H, T].
    heads, tokens = q.shape[1], c.tokens
    # num_seqs, tokens, q heads, KV heads, max_seqlen, head_dim of the C interface.
    c.sizes = c.num_seqs, tokens, heads, k.shape[1], c.longest, q.shape[-1]
    c.layout = q.stride(), k.stride(), v.stride(), out.stride()
    c.strides = (*map(_strides4, c.layout), _native.kept_strides((heads * tokens if q.ndim == 4 else 0, tokens, 1)))
    lib = _native.load_library()
    with _native.on_device(dev):
        status = lib.tasft_dense_fwd(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse_ptr, rest_ptr, _native.ptr(c.cu),
            _native.ptr(c.lens), _native.ptr(c.prefix), _native.ptr(c.slopes), *c.sizes, *c.strides, c.scale,
            c.softcap, c.causal, c.dtype, _native.stream_handle(dev))
    _native.check(status, "tasft_dense_fwd", {"q": list(q.shape), "k": list(k.shape)})
    return out, lse, kept


class _Dense(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, c: _Call, return_lse: bool):
        out, lse, kept = _forward(q, k, v, c, return_lse, True)
        ctx.save_for_backward(q, k, v, out, lse, kept, c.cu, c.lens, c.prefix, c.slopes)
        ctx.call = c
        ctx.set_materialize_grads(False)
        return (out, lse) if return_lse else out

    @staticmethod
    @first_order_only
    def backward(ctx, go, glse=None):
        if go is None and glse is None:
            return None, None, None, None, None
        q, k, v, out, lse, kept, cu, lens, prefix, slopes = ctx.saved_tensors
        c = ctx.call
        gq, gk, gv = _new_like(q), _new_like(k), _new_like(v)
        if q.numel() == 0:
            return gq, gk, gv, None, None
        # Hooks on saved tensors (copies to host memory among them) give back values, not strides.
        strides, layout = c.strides, (q.stride(), k.stride(), v.stride(), out.stride())
        at = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()
        if layout != c.layout or (at[0] | at[1] | at[2] | at[3]) & 15 or kept.data_ptr() & 7:
            q, k, v, out, kept = _ready(q), _ready(k), _ready(v), _ready(out), kept.clone()
            cu, lens, prefix, slopes = (None if t is None else t.contiguous() for t in (cu, lens, prefix, slopes))
            strides = (*(_strides4(t.stride()) for t in (q, k, v, out)), strides[4])
            at = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()
        if lse is not None:
            strides = (*strides[:4], _strides3(lse.stride()))
        go = torch.zeros_like(out) if go is None else _ready(go)
        rest_ptr = kept.data_ptr()
        lib = _native.load_library()
        rows = c.tokens if cu is not None else c.num_seqs * c.tokens
        ws_bytes = _workspace_bytes(c.num_seqs, rows, *c.sizes[2:])
        workspace = torch.empty((ws_bytes,), dtype=torch.uint8, device=q.device)
        with _native.on_device(q.device):
            status = lib.tasft_dense_bwd(
                *at, rest_ptr + q.numel() if lse is None else lse.data_ptr(), rest_ptr, go.data_ptr(),
                _native.ptr(glse), gq.data_ptr(), gk.data_ptr(), gv.data_ptr(), workspace.data_ptr(), ws_bytes,
                _native.ptr(cu), _native.ptr(lens), _native.ptr(prefix), _native.ptr(slopes), *c.sizes, *strides,
                _strides4(go.stride()), None if glse is None else _strides3(glse.stride()), _strides4(gq.stride()),
                _strides4(gk.stride()), _strides4(gv.stride()), c.scale, c.softcap, c.causal, c.dtype,
                _native.stream_handle(q.device))
        _native.check(status, "tasft_dense_bwd", {"q": list(q.shape), "k": list(k.shape)})
        return gq, gk, gv, None, None


def _lengths(t: torch.Tensor, n: int, most: int, what: str, device: torch.device) -> torch.Tensor:
    """``[n]`` lengths of at most ``most`` as the kernels read them; on the CPU they are checked."""
    if tuple(t.shape) != (n,):
        raise KernelError(f"{what} must have shape ({n},), got {tuple(t.shape)}", context={what: list(t.shape)})
    if t.is_floating_point() or t.is_complex() or t.dtype == torch.bool:
        raise KernelError(f"{what} must be integers, got {t.dtype}", context={"dtype": str(t.dtype)})
    if t.is_cpu and n and (int(t.min()) < 0 or int(t.max()) > most):
        raise KernelError(f"{what} must be in [0, {most}]", context={what: t.tolist()[:16]})
    return int32_on(t, device)


def dense_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    *,
    causal: bool = True,
    softcap: float | None = None,
    alibi_slopes: torch.Tensor | None = None,
    prefix_lens: torch.Tensor | None = None,
    cu_seqlens: torch.Tensor | None = None,
    max_seqlen: int | None = None,
    seq_lens: torch.Tensor | None = None,
    scale: float | None = None,
    return_lse: bool = False,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """Attention of every token to the tokens of its sequence; differentiable in q, k and v.

    With ``s = scale q_i . k_j``: ``s = softcap * tanh(s / softcap)`` if there is a cap, then
    ``s -= alibi_slopes[h] * |i - j|`` if there are slopes; ``out_i = softmax_j(s) v`` over the keys that
    token i sees.

    Args:
        q: ``[B, Hq, S, D]``, or with ``cu_seqlens`` packed ``[T, Hq, D]``; bf16 or fp16, D 64 or 128. Any
            strides (a transposed view of a projection is read in place; layouts without 16-byte rows
            are copied).
        k, v: ``[B, Hkv, S, D]`` / ``[T, Hkv, D]``, ``Hq % Hkv == 0`` (query head h reads KV head
            ``h // (Hq // Hkv)``).
        causal: token i sees keys ``j <= i`` of its sequence; False: all of them.
        softcap: positive cap of the scores' magnitude (and ``scale / softcap`` between 1e-37 and 1e37).
        alibi_slopes: ``[Hq]`` (fp32 on the device is read as it is).
        prefix_lens: ``[B]`` / ``[N]`` integers: with ``causal`` the first ``prefix_lens[n]`` tokens of a
            sequence are seen by all of its tokens.
        cu_seqlens: ``[N + 1]`` offsets of packed documents, as in
            ``BlockSparseFlashAttention.forward_varlen``: a token sees its own document alone. On the CPU
            they are checked; on the device they are trusted and ``max_seqlen`` must be given (tokens
            behind a document's first ``max_seqlen`` are left out: their rows are 0, nothing sees them).
            A batch of rows of several documents each is such a packed one, ``x.flatten(0, 1)``.
        seq_lens: ``[B]`` integers, batched form: tokens at or behind ``seq_lens[b]`` are padding.
        scale: default ``1 / sqrt(D)``.
        return_lse: also return the log-sum-exp of every token's scores.

    Lengths on the CPU are checked; on the device they are trusted (and clamped to what is there).

    Returns:
        ``[B, Hq, S, D]`` / ``[T, Hq, D]`` in q's layout; rows of padding and of tokens behind the last
        document are 0, and so are their gradients. With ``return_lse`` also ``[B, Hq, S]`` / ``[T, Hq]``
        fp32 (differentiable too), -inf for those rows. Equal calls give equal bits, gradients included; in
        another batch a sequence's gradients may differ in their last bits (how dS is rounded and heads are
        shared out goes by the tokens of the whole call). What is kept for the backward: q, k, v, the output
        with a byte more an element, and the log-sums. In fp16 the weights' gradients are rounded to fp16
        for their products: scale the loss, as for every fp16 gradient, so that they stay above 2^-14 where
        they matter.
        A row all of whose scores are -inf is 0, with log-sum -inf (its gradients are NaN); an infinity of v
        whose weight rounds to 0 gives NaN in the rows that see it. A second derivative and forward mode are
        refused. As for every operator of a graph of gradients: to capture a backward pass into a HIP graph,
        drop eager results of the same leaves first (torch ends the process otherwise).
    """
    qs, dev = tuple(q.shape), q.device
    packed = cu_seqlens is not None
    if len(qs) != (3 if packed else 4):
        raise KernelError(f"Expected q of shape {'[T, H, D] with' if packed else '[B, H, S, D] without'} cu_seqlens, "
                          f"got {qs}", context={"q_shape": list(qs)})
    ks = tuple(k.shape)
    if len(ks) != len(qs) or tuple(v.shape) != ks or ks[0] != qs[0] or ks[2:] != qs[2:] or ks[1] == 0 or \
            qs[1] == 0 or qs[1] % ks[1] != 0:
        raise KernelError("k and v must be alike and have q's shape but for the heads, with Hq % Hkv == 0",
                          context={"q": list(qs), "k": list(ks), "v": list(v.shape)})
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise KernelError("q, k and v must have one dtype",
                          context={"q": str(q.dtype), "k": str(k.dtype), "v": str(v.dtype)})
    c = _Call()
    c.dtype = _native.dtype_code(q.dtype, "dense attention")
    if qs[-1] not in _VALID_HEAD_DIMS:
        raise KernelError(f"HIP kernel supports head_dim in {sorted(_VALID_HEAD_DIMS)}, got {qs[-1]}",
                          context={"head_dim": qs[-1], "supported": sorted(_VALID_HEAD_DIMS)})
    c.softcap = check_softcap(softcap)
    c.scale = 1.0 / math.sqrt(qs[-1]) if scale is None else float(scale)
    if not 1e-30 <= c.scale <= 1e30:
        raise ValueError(f"scale must be positive and finite (1e-30 to 1e30), got {scale}")
    if prefix_lens is not None and not causal:
        raise ValueError("prefix_lens needs causal=True: without it every key is seen")
    if packed:
        if seq_lens is not None:
            raise ValueError("seq_lens is for a batch without cu_seqlens")
        if cu_seqlens.ndim != 1 or cu_seqlens.numel() < 2:
            raise KernelError("cu_seqlens must be a 1-D tensor of N + 1 >= 2 offsets",
                              context={"cu_seqlens_shape": list(cu_seqlens.shape)})
        if cu_seqlens.is_cpu:
            cu = cu_seqlens.to(torch.int64)
            lens = cu[1:] - cu[:-1]
            if int(cu[0]) != 0 or bool((lens < 0).any()) or int(cu[-1]) > qs[0]:
                raise KernelError("cu_seqlens must start at 0, be non-decreasing and end at <= T",
                                  context={"cu_seqlens": cu.tolist()[:16], "T": qs[0]})
            longest = int(lens.max())
            if max_seqlen is None:
                max_seqlen = max(longest, 1)
            elif longest > max_seqlen:
                raise KernelError(f"a sequence has {longest} tokens, more than max_seqlen={max_seqlen}",
                                  context={"max_seqlen": max_seqlen, "longest": longest})
        elif max_seqlen is None:
            raise KernelError("max_seqlen is required when cu_seqlens is on the device",
                              context={"device": str(cu_seqlens.device)})
        if max_seqlen <= 0:
            raise KernelError(f"max_seqlen must be positive, got {max_seqlen}", context={"max_seqlen": max_seqlen})
        c.num_seqs, c.tokens, c.longest = cu_seqlens.numel() - 1, qs[0], min(int(max_seqlen), max(qs[0], 1))
    else:
        if max_seqlen is not None:
            raise ValueError("max_seqlen goes with cu_seqlens")
        c.num_seqs, c.tokens, c.longest = qs[0], qs[2], max(qs[2], 1)
    c.causal = 1 if causal else 0
    # (A dual tensor does not require grad.)
    if forward_ad._current_level >= 0 and any(
            t is not None and forward_ad.unpack_dual(t).tangent is not None for t in (q, k, v, alibi_slopes)):
        raise KernelError("q, k, v and alibi_slopes must not carry tangents: dense attention has no forward-mode "
                          "derivative", context={})
    if not q.is_cuda or k.device != dev or v.device != dev:
        raise KernelError("Tensors must be on one CUDA device",
                          context={"q": str(dev), "k": str(k.device), "v": str(v.device)})
    c.cu = int32_on(cu_seqlens, dev) if packed else None
    c.lens = None if seq_lens is None else _lengths(seq_lens, c.num_seqs, c.tokens, "seq_lens", dev)
    c.prefix = None if prefix_lens is None else _lengths(prefix_lens, c.num_seqs, c.longest, "prefix_lens", dev)
    c.slopes = check_slopes(alibi_slopes, qs[1], dev)
    q, k, v = _ready(q), _ready(k), _ready(v)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _Dense.apply(q, k, v, c, return_lse)
    out, lse, _ = _forward(q, k, v, c, return_lse, False)
    return (out, lse) if return_lse else out


__all__ = ["dense_attention"]
