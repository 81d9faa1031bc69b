"""Dense attention without a GPU: what it refuses, and the reference's own gradients by differences."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

import dense_ref as ref
from tasft_amd import _native
from tasft_amd.exceptions import KernelError
from tasft_amd.kernels import dense_attention


def make(b=2, hq=4, hkv=2, s=10, d=64, dtype=torch.bfloat16):
    return [torch.zeros((b, h, s, d), dtype=dtype) for h in (hq, hkv, hkv)]


def test_cpu_tensors_are_refused_after_their_shapes():
    q, k, v = make()
    with pytest.raises(KernelError, match="one CUDA device"):
        dense_attention(q, k, v)
    with pytest.raises(KernelError, match="one CUDA device"):
        dense_attention(q[0].transpose(0, 1), k[0].transpose(0, 1), v[0].transpose(0, 1), cu_seqlens=torch.tensor([0, 10]))


@pytest.mark.parametrize(("change", "match"), [
    (lambda q, k, v: (q[0], k[0], v[0]), "Expected q"),
    (lambda q, k, v: (q, k, v[:, :1]), "alike"),
    (lambda q, k, v: (q[:, :3], k, v), "alike"),
    (lambda q, k, v: (q[:, :, :9], k, v), "alike"),
    (lambda q, k, v: (q, k[:, :0], v[:, :0]), "alike"),
    (lambda q, k, v: (q[:, :0], k, v), "alike"),
    (lambda q, k, v: (q, k.half(), v), "one dtype"),
    (lambda q, k, v: (q.float(), k.float(), v.float()), "bf16 or fp16"),
    (lambda q, k, v: (q[..., :32], k[..., :32], v[..., :32]), "head_dim"),
])
def test_shapes_and_types(change, match):
    with pytest.raises(KernelError, match=match):
        dense_attention(*change(*make()))


@pytest.mark.parametrize(("options", "error", "match"), [
    ({"softcap": 0.0}, ValueError, "softcap"),
    ({"softcap": -1.0}, ValueError, "softcap"),
    ({"softcap": math.inf}, ValueError, "softcap"),
    ({"softcap": math.nan}, ValueError, "softcap"),
    ({"softcap": 1e-50}, ValueError, "softcap"),  # 0 in 32 bits
    ({"softcap": 1e39}, ValueError, "softcap"),
    ({"scale": 1e-50}, ValueError, "scale"),
    ({"scale": 1e39}, ValueError, "scale"),
    ({"scale": 0.0}, ValueError, "scale"),
    ({"scale": math.nan}, ValueError, "scale"),
    ({"causal": False, "prefix_lens": torch.tensor([1, 1])}, ValueError, "prefix_lens"),
    ({"max_seqlen": 10}, ValueError, "max_seqlen"),
])
def test_options(options, error, match):
    with pytest.raises(error, match=match):
        dense_attention(*make(), **options)


@pytest.mark.parametrize(("options", "error", "match"), [
    ({"cu_seqlens": torch.tensor([0])}, KernelError, "offsets"),
    ({"cu_seqlens": torch.tensor([1, 10])}, KernelError, "start at 0"),
    ({"cu_seqlens": torch.tensor([0, 7, 5])}, KernelError, "start at 0"),
    ({"cu_seqlens": torch.tensor([0, 11])}, KernelError, "start at 0"),
    ({"cu_seqlens": torch.tensor([0, 9]), "max_seqlen": 8}, KernelError, "more than max_seqlen"),
    ({"cu_seqlens": torch.tensor([0, 0]), "max_seqlen": 0}, KernelError, "max_seqlen"),
    ({"cu_seqlens": torch.tensor([0, 9]), "seq_lens": torch.tensor([9])}, ValueError, "seq_lens"),
])
def test_packed_options(options, error, match):
    q, k, v = (x[0].transpose(0, 1) for x in make())
    with pytest.raises(error, match=match):
        dense_attention(q, k, v, **options)


def test_c_entries_refuse_before_any_launch():
    lib = _native.load_library()
    fake = ctypes.c_void_p(16)  # never dereferenced
    st = _native.kept_strides((64 * 10 * 4, 640, 64, 1))
    sl = _native.kept_strides((40, 10, 1))

    def fwd(q=fake, sizes=(2, 10, 4, 2, 10, 64), qs=st, scale=0.1, cap=0.0, dtype=0, cu=None, lens=None, lse_strides=sl, rest=None):
        return lib.tasft_dense_fwd(q, fake, fake, fake, fake, rest, cu, lens, None, None, *sizes, qs, st, st, st, lse_strides,
                                   scale, cap, 1, dtype, None)

    def refused(rc, code, text):
        assert rc == code and text in lib.tasft_last_error(), (rc, lib.tasft_last_error())

    refused(fwd(q=None), -1, b"null")
    refused(fwd(dtype=7), -2, b"dtype")
    refused(fwd(sizes=(2, 10, 4, 3, 10, 64)), -1, b"multiple")
    refused(fwd(sizes=(2, 0, 4, 2, 10, 64)), -1, b"positive")
    refused(fwd(sizes=(2, 10, 4, 2, 10, 96)), -2, b"head_dim")
    refused(fwd(sizes=(1 << 20, 1 << 20, 4, 2, 10, 64)), -2, b"launch too large")
    refused(fwd(scale=0.0), -1, b"scale")
    refused(fwd(cap=-1.0), -1, b"softcap")
    refused(fwd(cap=float("nan")), -1, b"softcap")
    refused(fwd(cap=float("inf")), -1, b"softcap")
    refused(fwd(scale=float("inf")), -1, b"scale")
    refused(fwd(scale=1e30, cap=1e-30), -1, b"out of range")  # their quotient
    refused(fwd(scale=1e-39), -1, b"out of range")
    refused(fwd(cu=fake, lens=fake), -1, b"not both")
    refused(fwd(qs=_native.kept_strides((2560, 640, 64, 2))), -1, b"contiguous")
    refused(fwd(qs=_native.kept_strides((2560, 640, 68, 1))), -1, b"multiples of 8")
    refused(fwd(qs=_native.kept_strides((2560, -640, 64, 1))), -1, b"non-negative")
    refused(fwd(qs=_native.kept_strides((2560, 640, 1 << 23, 1))), -2, b"token stride")
    refused(fwd(q=ctypes.c_void_p(18)), -1, b"16-byte")
    refused(fwd(lse_strides=None), -1, b"lse")
    size = lib.tasft_dense_bwd_workspace_bytes(2, 20, 4, 2, 10, 64)
    assert size == 20 * 4 * 8 + 2 * 20 * 2 * 64 * 8  # statistics, two partial sums of dk and dv
    assert lib.tasft_dense_bwd_workspace_bytes(2, 20, 4, 3, 10, 64) == 0
    assert lib.tasft_dense_bwd_workspace_bytes(1024, 70000, 4, 2, 100, 64) == 70000 * 4 * 8  # no partial sums

    def bwd(ws=fake, size=size, glse=None, rest=None):
        return lib.tasft_dense_bwd(fake, fake, fake, fake, fake, rest, fake, glse, fake, fake, fake, ws, size, None, None,
                                   None, None, 2, 10, 4, 2, 10, 64, st, st, st, st, sl, st, None, st, st, st, 0.1,
                                   0.0, 1, 0, None)

    refused(bwd(size=size - 1), -4, b"workspace")
    refused(bwd(ws=None), -4, b"workspace")
    refused(bwd(ws=ctypes.c_void_p(8)), -1, b"aligned")
    refused(bwd(glse=fake), -1, b"null")
    refused(bwd(rest=ctypes.c_void_p(4)), -1, b"out_rest")
    refused(fwd(rest=ctypes.c_void_p(4)), -1, b"out_rest")


@pytest.mark.parametrize("cap", [0.0, 5.0])
@pytest.mark.parametrize("prefix", [0, 4])
def test_reference_gradients_by_differences(cap, prefix):
    """The oracle's gradients against differences of its own forward in 64 bits."""
    n, h, d = 7, 2, 64
    rows = ref.inputs([n], h, 1, d, torch.float64, seed=1)[0]
    slopes = torch.tensor([0.5, 0.25])
    got = ref.reference(*rows, causal=True, scale=0.2, cap=cap, slopes=slopes, prefix=prefix, dtype=torch.bfloat16)
    ok = ref.seen(n, True, prefix)

    def loss(q, k, v):
        total = 0.0
        for j in range(h):
            out, lse = ref.forward(q[:, j], k[:, 0], v[:, 0], 0.2, cap, float(slopes[j]), ok)
            total += float((out * rows[3][:, j]).sum() + (lse * rows[4][:, j]).sum())
        return total

    g = torch.Generator().manual_seed(2)
    for i, name in enumerate(("gq", "gk", "gv")):
        way = torch.randn(rows[i].shape, generator=g, dtype=torch.float64)
        step = 1e-5
        plus, minus = list(rows[:3]), list(rows[:3])
        plus[i], minus[i] = rows[i] + step * way, rows[i] - step * way
        slope = (loss(*plus) - loss(*minus)) / (2 * step)
        # Central differences: step^2 of the third derivative, and 64-bit rounding over the step.
        assert abs(slope - float((got[name] * way).sum())) < 1e-6 * (1 + abs(slope))
