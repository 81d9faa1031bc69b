"""Dense attention without a GPU, continued: the ends of its ranges, and what reaches the kernels."""
from __future__ import annotations

import ctypes
import sys

import pytest
import torch
from torch.autograd import forward_ad

from tasft_amd import _native
from tasft_amd.exceptions import KernelError
from tasft_amd.kernels import dense_attention

module = sys.modules["tasft_amd.kernels.dense_attention"]

FAKE = ctypes.c_void_p(16)  # never dereferenced


@pytest.mark.parametrize(("scale", "cap"), [(1e-16, 1e30), (1e-30, 1e10), (1.0, 9e37)])
def test_quotients_that_fp32_does_not_hold(scale, cap):
    """scale / cap as 0 or with fewer bits: no scores could be made of it."""
    lib = _native.load_library()
    st, sl = _native.kept_strides((64 * 10 * 4, 640, 64, 1)), _native.kept_strides((40, 10, 1))
    rc = lib.tasft_dense_fwd(FAKE, FAKE, FAKE, FAKE, FAKE, None, None, None, None, None, 2, 10, 4, 2, 10, 64, st, st, st, st,
                             sl, scale, cap, 1, 0, None)
    assert rc == -1 and b"out of range" in lib.tasft_last_error()
    rc = lib.tasft_chunk_scored_fwd(
        FAKE, FAKE, FAKE, FAKE, None, None, FAKE, FAKE, FAKE, None, None, 0, None, 0, 2, 200, 4, 2, 100, 64, 64, 3, 8, 4,
        3, 1, st, st, st, st, st, 3, scale, cap, 1, 0, None)
    assert rc == -1 and b"out of range" in lib.tasft_last_error()


class Recorder:
    """Stands for the library: notes the addresses and strides that a backward call is given."""

    def __init__(self):
        self.seen = None
        self.tasft_dense_bwd_workspace_bytes = _native.load_library().tasft_dense_bwd_workspace_bytes

    def tasft_dense_fwd(self, *args):
        return 0

    def tasft_dense_bwd(self, *args):
        self.seen = args
        return 0


def fused(b, s, heads, d):
    """Heads of a projection as views of it, [B, H, S, D]."""
    wide = torch.zeros((b, s, sum(heads), d), dtype=torch.bfloat16)
    return [x.transpose(1, 2) for x in wide.split(heads, 2)]


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("return_lse", [False, True])
@pytest.mark.parametrize("odd", [False, True])
def test_backward_reads_saved_tensors_as_they_come_back(monkeypatch, packed, return_lse, odd):
    """Hooks on saved tensors give back values, not strides (torch's own copies to host memory do not keep those
    of a slice): each address goes to the kernels with the strides of the tensor that lies there."""
    lib = Recorder()
    monkeypatch.setattr(_native, "load_library", lambda: lib)
    monkeypatch.setattr(_native, "stream_handle", lambda device: 0)
    q, k, v = fused(2, 10, (4, 2, 2), 64)
    if packed:
        q, k, v = (x[0].transpose(0, 1) for x in (q, k, v))
    q, k, v = (x.detach().requires_grad_(True) for x in (q, k, v))
    assert not q.is_contiguous() and not k.is_contiguous()
    c = module._Call()
    c.causal, c.dtype, c.scale, c.softcap, c.longest = 1, 0, 0.125, 0.0, 10
    c.num_seqs, c.tokens = (1 if packed else 2), 10
    c.cu = torch.tensor([0, 10], dtype=torch.int32) if packed else None
    c.lens = c.prefix = c.slopes = None
    back = {}

    def unpack(t):
        # Dense, as from a buffer of many tensors, at a place that the kernels read or (odd) do not.
        room = torch.empty(t.numel() * t.element_size() + 64, dtype=torch.uint8)
        shift = (2 if t.dtype == torch.bfloat16 else 4) if odd else 0
        off = -room.data_ptr() % 16 + shift
        t = room[off:off + t.numel() * t.element_size()].view(t.dtype).view(t.shape).copy_(t)
        back[t.data_ptr()] = t
        return t

    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().contiguous().clone(), unpack):
        got = module._Dense.apply(q, k, v, c, return_lse)
    out = got[0] if return_lse else got
    copies = []
    ready = module._ready
    monkeypatch.setattr(module, "_ready", lambda t: copies.append(ready(t)) or copies[-1])
    torch.autograd.grad(out.float().sum(), (q, k, v))
    args = lib.seen
    for t in copies:
        back[t.data_ptr()] = t
    sizes_at = next(i for i, a in enumerate(args) if not isinstance(a, (int, type(None))))  # the first strides
    strides = args[sizes_at:sizes_at + 6]
    for at, (name, like) in enumerate((("q", q), ("k", k), ("v", v), ("out", q))):
        t = back[args[at]]
        assert tuple(t.shape) == tuple(like.shape) and args[at] % 16 == 0, name
        assert list(strides[at]) == list(module._strides4(t.stride())), name
    if return_lse:
        t = back[args[4]]
        assert list(strides[4]) == list(module._strides3(t.stride()))
    else:
        assert list(strides[4]) == [0 if packed else 40, 10, 1]
    assert args[5] % 8 == 0  # what out's rounding left over


@pytest.mark.parametrize("which", range(4))
@pytest.mark.parametrize("grad", [False, True])
def test_tangents_are_refused(which, grad):
    """A tangent would be lost: a dual tensor does not require grad."""
    args = [torch.zeros((2, h, 10, 64), dtype=torch.bfloat16) for h in (4, 2, 2)] + [torch.ones(4)]
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        with pytest.raises(KernelError, match="one CUDA device"):  # what a level alone leaves as it is
            dense_attention(*args[:3], alibi_slopes=args[3])
        args[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(KernelError, match="forward-mode"):
            dense_attention(*args[:3], alibi_slopes=args[3])
    args = [torch.zeros((2, h, 10, 64), dtype=torch.bfloat16) for h in (4, 2, 2)]
    with pytest.raises(KernelError, match="forward-mode"):
        torch.func.jvp(lambda q: dense_attention(q, *args[1:]), (args[0],), (args[0],))


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("most", [5000, 6144, 8192, 100000])
def test_backward_workspace_is_what_its_size_was_asked_for(packed, most):
    """Whatever max_seqlen is given: the size function and the backward go by the same number."""
    lib = _native.load_library()
    tokens, hq, hkv, d = 8192, 32, 8, 64
    size = lib.tasft_dense_bwd_workspace_bytes(1, tokens, hq, hkv, most, d)
    st = _native.kept_strides((hq * tokens * d, tokens * d, d, 1))
    sl = _native.kept_strides((hq * tokens, tokens, 1))
    unaligned = ctypes.c_void_p(8)

    def call(given):
        return lib.tasft_dense_bwd(FAKE, FAKE, FAKE, FAKE, FAKE, None, FAKE, None, FAKE, FAKE, FAKE, unaligned, given,
                                   FAKE if packed else None, None, None, None, 1, tokens, hq, hkv, most, d, st, st, st, st,
                                   sl, st, None, st, st, st, 0.1, 0.0, 1, 0, None)

    assert call(size) == -1 and b"aligned" in lib.tasft_last_error()  # enough: what is refused next is its address
    assert call(size - 1) == -4 and b"workspace" in lib.tasft_last_error()
