"""Rotary position embedding of queries and keys, for training and for the attention calls.

The attention, gate and cache entry points of this package take Q and K after the rotation, as
the reference does (``tasft/modules/tasft_attention.py:426``, which gets them from its model's own
rotary module). ``rotary_frequencies`` gives the inverse frequencies of a model's configuration,
``apply_rotary`` rotates a batch (with gradients), and ``append_paged`` (in
``tasft_amd.kernels.paged_cache``) rotates new tokens on their way into a paged cache.
"""
from __future__ import annotations

import math

import torch
from torch.autograd import forward_ad

from tasft_amd import _native
from tasft_amd.exceptions import KernelError

_MAX_HEAD_DIM = 256


def rotary_frequencies(
    rotary_dim: int,
    base: float = 10000.0,
    scaling: dict | None = None,
    device: torch.device | str | None = None,
) -> tuple[torch.Tensor, float]:
    """Inverse frequencies ``[rotary_dim / 2]`` in 64 bits, and the factor on cosine and sine.

    Args:
        rotary_dim: rotated dims of a head (even).
        base: the frequencies are ``base ** (-2 j / rotary_dim)``.
        scaling: a model configuration's ``rope_scaling``: ``None`` or ``{"rope_type": "default"}``;
            ``"linear"`` (``factor``): positions divided by the factor; ``"llama3"`` (``factor``,
            ``low_freq_factor``, ``high_freq_factor``, ``original_max_position_embeddings``):
            frequencies of fewer than ``low_freq_factor`` turns over the original length divided by
            the factor, of more than ``high_freq_factor`` kept, those between blended; ``"yarn"``
            (``factor``, ``original_max_position_embeddings``, optional ``beta_fast`` 32,
            ``beta_slow`` 1, ``truncate``, ``attention_factor``, ``mscale`` with
            ``mscale_all_dim``): blended by dimension between the dims that make ``beta_fast`` and
            ``beta_slow`` turns (whole dims unless ``truncate`` is false), with a factor on the
            result: ``attention_factor``, or ``0.1 mscale ln(factor) + 1`` over the same of
            ``mscale_all_dim`` (without them ``0.1 ln(factor) + 1``; what such a model multiplies
            its softmax by is the caller's). Types whose frequencies follow the running length, and
            entries that none of these types has, are refused.
        device: of the returned tensor.
    """
    if rotary_dim <= 0 or rotary_dim % 2 != 0:
        raise ValueError(f"rotary_dim must be even and positive, got {rotary_dim}")
    if not base > 0.0 or not math.isfinite(base):
        raise ValueError(f"base must be positive and finite, got {base}")
    inv = torch.tensor([base ** (-2.0 * j / rotary_dim) for j in range(rotary_dim // 2)], dtype=torch.float64)
    kind = "default" if scaling is None else scaling.get("rope_type", scaling.get("type", "default"))
    attention = 1.0
    if kind not in ("default", "linear", "llama3", "yarn"):
        raise ValueError(f"rope_type must be default, linear, llama3 or yarn, got {kind!r}")
    unknown = sorted(name for name, value in (scaling or {}).items() if name not in _ENTRIES and value is not None)
    if unknown:
        raise ValueError(f"rope_type {kind!r}: no such entries: {', '.join(map(str, unknown))}")
    theta = (scaling or {}).get("rope_theta")
    if theta is not None and float(theta) != float(base):
        raise ValueError(f"rope_theta is {theta} but base is {base}")
    if kind != "default":
        factor = _entry(scaling, "factor", kind)
        if not 0.0 < factor < math.inf:
            raise ValueError(f"factor must be positive and finite, got {factor}")
        if kind == "linear":
            inv = inv / factor
        else:
            original = _entry(scaling, "original_max_position_embeddings", kind)
            if not 0.0 < original < math.inf:
                raise ValueError(f"original_max_position_embeddings must be positive and finite, got {original}")
            if kind == "llama3":
                low, high = _entry(scaling, "low_freq_factor", kind), _entry(scaling, "high_freq_factor", kind)
                if not 0.0 < low < high:
                    raise ValueError(f"need 0 < low_freq_factor < high_freq_factor, got {low} and {high}")
                keep = ((original * inv / (2.0 * math.pi) - low) / (high - low)).clamp(0.0, 1.0)
            else:
                keep = 1.0 - _yarn_ramp(rotary_dim, base, original, scaling)
                attention = _yarn_factor(factor, scaling)
            inv = inv / factor * (1.0 - keep) + inv * keep
    return inv.to(device) if device is not None else inv, attention


# What the configurations of these types hold. Of no effect here: "finetuned" (describes the weights),
# "partial_rotary_factor" (the caller's rotary_dim), "mrope_section" (one position a token, so that its
# sections turn alike).
_ENTRIES = frozenset({
    "rope_type", "type", "rope_theta", "factor", "original_max_position_embeddings", "low_freq_factor",
    "high_freq_factor", "beta_fast", "beta_slow", "attention_factor", "mscale", "mscale_all_dim", "truncate",
    "finetuned", "partial_rotary_factor", "mrope_section"})


def _entry(scaling: dict, name: str, kind: str) -> float:
    if scaling.get(name) is None:
        raise ValueError(f"rope_type {kind!r} needs {name!r}")
    return float(scaling[name])


def _yarn_factor(factor: float, scaling: dict) -> float:
    """The factor on cosine and sine."""
    if scaling.get("attention_factor") is not None:
        return float(scaling["attention_factor"])
    over, under = scaling.get("mscale"), scaling.get("mscale_all_dim")
    # Alone, and not at the value that leaving it out means, an entry is read in two ways.
    if (under is None and over not in (None, 1)) or (over is None and under not in (None, 0)):
        raise ValueError("mscale and mscale_all_dim are given together or not at all")
    over, under = 1.0 if over is None else float(over), 0.0 if under is None else float(under)
    growth = 0.1 * math.log(factor) if factor > 1.0 else 0.0
    return (growth * over + 1.0) / (growth * under + 1.0)


def _yarn_ramp(dim: int, base: float, original: float, scaling: dict) -> torch.Tensor:
    """0 for the pairs that keep their frequency, 1 for those divided by the factor."""
    if not base > 1.0:
        raise ValueError(f"rope_type 'yarn' needs a base above 1, got {base}")
    fast, slow = float(scaling.get("beta_fast") or 32.0), float(scaling.get("beta_slow") or 1.0)
    if not (0.0 < fast < math.inf and 0.0 < slow < math.inf):
        raise ValueError(f"beta_fast and beta_slow must be positive and finite, got {fast} and {slow}")

    def pair_with_turns(turns: float) -> float:
        return dim * math.log(original / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))

    low, high = pair_with_turns(fast), pair_with_turns(slow)
    if scaling.get("truncate") is None or scaling["truncate"]:
        low, high = math.floor(low), math.ceil(high)
    low, high = max(low, 0), min(high, dim - 1)
    at = torch.arange(dim // 2, dtype=torch.float64)
    return ((at - low) / (high - low if high != low else 0.001)).clamp(0.0, 1.0)


def check_frequencies(inv_freq: torch.Tensor, head_dim: int, device: torch.device) -> torch.Tensor:
    """``inv_freq`` as the kernels read it (contiguous doubles on ``device``)."""
    if head_dim > _MAX_HEAD_DIM:
        raise KernelError(f"rotary kernels take head_dim up to {_MAX_HEAD_DIM}, got {head_dim}",
                          context={"head_dim": head_dim})
    if inv_freq.ndim != 1 or not 1 <= inv_freq.numel() <= head_dim // 2:
        raise KernelError(f"inv_freq must be 1-D with 1 to head_dim / 2 = {head_dim // 2} entries, "
                          f"got shape {tuple(inv_freq.shape)}", context={"inv_freq": list(inv_freq.shape)})
    if not inv_freq.is_floating_point():
        raise KernelError(f"inv_freq must be floating point, got {inv_freq.dtype}",
                          context={"dtype": str(inv_freq.dtype)})
    if inv_freq.requires_grad:
        raise KernelError("inv_freq must not require grad: the rotation has no gradient for it", context={})
    if inv_freq.dtype == torch.float64 and inv_freq.device == device and inv_freq.is_contiguous():
        return inv_freq
    return inv_freq.to(device=device, dtype=torch.float64).contiguous()


def check_positions(positions: torch.Tensor, device: torch.device) -> torch.Tensor:
    if positions.dtype not in (torch.int32, torch.int64):
        raise KernelError(f"positions must be int32 or int64, got {positions.dtype}",
                          context={"dtype": str(positions.dtype)})
    return positions if positions.device == device else positions.to(device)


def _unit_last(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(-1) == 1 else t.contiguous()


def _new_like(t: torch.Tensor) -> torch.Tensor:
    """A new tensor of t's layout, of contiguous rows in any case (rows that overlap can make torch put
    another dim innermost)."""
    out = torch.empty_like(t)
    return out if out.stride(-1) == 1 else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _strides4(st: tuple[int, ...]):
    """(b, h, s, d) strides of ``[B, H, S, D]``, or of packed ``[T, H, D]`` as one batch entry."""
    return _native.kept_strides(st if len(st) == 4 else (0, st[1], st[0], st[2]))


def _rows_and_new(t: torch.Tensor):
    """``t`` with contiguous rows and a new tensor like it (``_unit_last``, ``_new_like``), each with its
    strides for the library: looked up once."""
    st = t.stride()
    if st[-1] != 1:
        t = t.contiguous()
        st = t.stride()
    out = torch.empty_like(t)
    so = out.stride()
    if so[-1] != 1:
        out = _new_like(t)
        so = out.stride()
    return t, _strides4(st), out, _strides4(so)


def _rotate(q, k, positions, inv_freq, interleaved, scale, inverse):
    """``tasft_rotary`` on checked tensors; ``k`` may be None."""
    q, qs, q_out, qos = _rows_and_new(q)
    k, ks, k_out, kos = (None,) * 4 if k is None else _rows_and_new(k)
    ps = positions.stride()
    if q.ndim == 4:
        B, Hq, S, D = q.shape
        pos_strides = (0 if len(ps) == 1 or positions.shape[0] == 1 else ps[0], ps[-1])
    else:
        S, Hq, D = q.shape
        B, pos_strides = 1, (0, ps[0])
    if q.numel() == 0:
        return q_out, k_out
    lib = _native.load_library()
    with _native.on_device(q.device):
        status = lib.tasft_rotary(
            q.data_ptr(), _native.ptr(k), q_out.data_ptr(), _native.ptr(k_out), positions.data_ptr(),
            1 if positions.dtype == torch.int64 else 0, inv_freq.data_ptr(), B, Hq,
            0 if k is None else k.shape[1], S, D, 2 * inv_freq.numel(), qs, ks, qos, kos,
            _native.kept_strides(pos_strides), 1 if interleaved else 0, 1 if inverse else 0, scale,
            _native.dtype_code(q.dtype, "rotary"), _native.stream_handle(q.device))
    _native.check(status, "tasft_rotary", {"shape": list(q.shape)})
    return q_out, k_out


class _Rotary(torch.autograd.Function):
    """The rotation is linear: its gradient is the inverse rotation of the outputs' gradients (with the
    same factor), its forward derivative the rotation of the tangents; both are this function again,
    so derivatives of any order."""

    @staticmethod
    def forward(ctx, q, k, positions, inv_freq, interleaved, scale, inverse):
        ctx.save_for_backward(positions, inv_freq)
        ctx.cfg = (interleaved, scale, inverse)
        if forward_ad._current_level >= 0:
            ctx.save_for_forward(positions, inv_freq)
            ctx.heads = (q.shape[1], None if k is None else k.shape[1])
        ctx.set_materialize_grads(False)
        return _rotate(q, k, positions, inv_freq, interleaved, scale, inverse)

    @staticmethod
    def backward(ctx, gq, gk):
        want_q, want_k = ctx.needs_input_grad[:2]
        gq, gk = _turn_given(ctx, gq if want_q else None, gk if want_k else None, not ctx.cfg[2])
        return gq, gk, None, None, None, None, None

    @staticmethod
    def jvp(ctx, tq, tk, positions, inv_freq, *_):
        if inv_freq is not None:
            raise KernelError("inv_freq must not carry a tangent: the rotation has no derivative for it", context={})
        out = _turn_given(ctx, tq, tk, ctx.cfg[2])
        there = tq if tq is not None else tk
        # torch takes no None for the tangent of a tensor.
        return tuple(there.new_zeros((there.shape[0], h, *there.shape[2:])) if t is None and h is not None else t
                     for t, h in zip(out, ctx.heads))


def _turn_given(ctx, a, b, inverse):
    """Those of the two that are there, rotated as ``ctx``'s operator or its inverse does."""
    given = [x for x in (a, b) if x is not None]
    if not given:
        return None, None
    positions, inv_freq = ctx.saved_tensors
    interleaved, scale, _ = ctx.cfg
    out = list(_turn(given[0], given[1] if len(given) > 1 else None, positions, inv_freq, interleaved, scale, inverse))
    return out.pop(0) if a is not None else None, out.pop(0) if b is not None else None


def _turn(q, k, *args):
    """Through the function only where a graph is being built or tangents are carried along (a dual
    tensor does not require grad)."""
    if forward_ad._current_level >= 0 or (torch.is_grad_enabled() and
                                          (q.requires_grad or (k is not None and k.requires_grad))):
        return _Rotary.apply(q, k, *args)
    return _rotate(q, k, *args)


def apply_rotary(
    q: torch.Tensor,
    k: torch.Tensor | None,
    positions: torch.Tensor,
    inv_freq: torch.Tensor,
    *,
    interleaved: bool = False,
    scale: float = 1.0,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Queries and keys rotated by their positions, in one launch; differentiable in q and k, also in
    forward mode.

    Args:
        q: ``[B, Hq, S, D]`` or packed ``[T, Hq, D]``, bf16 or fp16, any strides (a transposed view
            of a projection is read in place).
        k: ``[B, Hkv, S, D]`` / ``[T, Hkv, D]`` of q's dtype, or None.
        positions: int32 or int64 ``[S]``, ``[B, S]`` (or ``[1, S]``), packed ``[T]``.
        inv_freq: ``[R / 2]`` inverse frequencies (``rotary_frequencies``; float64 on the device is
            read as it is, other types are converted at each call). ``R <= D``: the dims behind the
            first R are copied.
        interleaved: pairs ``(2j, 2j + 1)`` instead of ``(j, j + R / 2)``.
        scale: factor on the rotated dims (the second value of ``rotary_frequencies``).

    Returns:
        The rotated q and k (None without k), new tensors of q's and k's layout. As for every
        operator of a graph of gradients: to capture a backward pass into a HIP graph, drop eager
        results of the same leaves first (torch ends the process otherwise).
    """
    qs, dev = tuple(q.shape), q.device
    if len(qs) not in (3, 4):
        raise KernelError(f"Expected q of shape [B, H, S, D] or [T, H, D], got {qs}", context={"q_shape": list(qs)})
    if qs[1] == 0:
        raise KernelError("q must have at least one head", context={"q_shape": list(qs)})
    _native.dtype_code(q.dtype, "rotary")
    if k is not None:
        ks = tuple(k.shape)  # all but the head count as q's
        if len(ks) != len(qs) or ks[1] == 0 or ks[0] != qs[0] or ks[2:] != qs[2:]:
            raise KernelError("q and k shapes are incompatible", context={"q": list(qs), "k": list(ks)})
        if k.dtype != q.dtype or k.device != dev:
            raise KernelError("q and k must have one dtype and device",
                              context={"q": [str(q.dtype), str(dev)], "k": [str(k.dtype), str(k.device)]})
    at = tuple(positions.shape)
    if at != ((qs[0],) if len(qs) == 3 else (qs[2],)) and (len(qs) == 3 or at not in ((1, qs[2]), (qs[0], qs[2]))):
        raise KernelError(f"positions of shape {at} do not fit q {qs}", context={"positions": list(at), "q": list(qs)})
    positions = check_positions(positions, dev)
    inv_freq = check_frequencies(inv_freq, qs[-1], dev)
    if not q.is_cuda:
        raise KernelError("Tensors must be on CUDA device", context={"device": str(dev)})
    return _turn(q, k, positions, inv_freq, bool(interleaved), float(scale), False)


__all__ = ["apply_rotary", "rotary_frequencies"]
