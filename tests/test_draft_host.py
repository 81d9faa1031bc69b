"""Drafted trees and scored chunks without a GPU: what is refused."""
from __future__ import annotations

import ctypes

import pytest
import torch

from tasft_amd import _native
from tasft_amd.exceptions import KernelError
from tasft_amd.kernels import accept_draft, commit_draft_paged, draft_tree

PARENTS, CU, LENS = torch.tensor([-1, 0, 0, -1, 0]), torch.tensor([0, 3, 5]), torch.tensor([10, 20])


@pytest.mark.parametrize(("parents", "cu", "options", "match"), [
    (PARENTS[None], CU, {}, "parents"),
    (PARENTS.float(), CU, {}, "parents"),
    (PARENTS, CU[:1], {}, "offsets"),
    (PARENTS, torch.tensor([1, 5]), {}, "start at 0"),
    (PARENTS, torch.tensor([0, 4, 3]), {}, "start at 0"),
    (PARENTS, torch.tensor([0, 3, 6]), {}, "start at 0"),
    (PARENTS, CU, {"max_nodes": 2}, "more than max_nodes"),
    (PARENTS, CU, {"max_nodes": 5000}, "max_nodes"),
    (torch.tensor([-1, 1, 0, -1, 0]), CU, {}, "before it"),
    (torch.tensor([-1, 0, 0, -2, 0]), CU, {}, "before it"),
    (torch.tensor([-1, 0, 0, 2, 0]), CU, {}, "before it"),
])
def test_trees(parents, cu, options, match):
    with pytest.raises(KernelError, match=match):
        draft_tree(parents, cu, LENS, **options)
    with pytest.raises(KernelError, match=match):
        accept_draft(parents, torch.zeros(5, dtype=torch.int64), torch.zeros(5, dtype=torch.int64), cu, **options)


def test_devices_and_types():
    with pytest.raises(KernelError, match="kv_lens must have shape"):
        draft_tree(PARENTS, CU, LENS[:1])
    with pytest.raises(KernelError, match="CUDA device"):
        draft_tree(PARENTS, CU, LENS)
    tok = torch.zeros(5, dtype=torch.int64)
    with pytest.raises(KernelError, match="CUDA device"):
        accept_draft(PARENTS, tok, tok, CU)
    for tokens, targets, first, match in ((tok.float(), tok, None, "tokens"), (tok[:4], tok, None, "tokens"),
                                          (tok, tok.int(), None, "targets"), (tok, tok[:4], None, "targets"),
                                          (tok, tok, tok, "first_targets"), (tok, tok, tok[:2].int(), "first_targets")):
        with pytest.raises(KernelError, match=match):
            accept_draft(PARENTS, tokens, targets, CU, first_targets=first)


@pytest.mark.parametrize(("change", "match"), [
    ({}, "one CUDA device"),
    ({"k_pages": torch.zeros(4, 8, 2, 32)}, "pools"),
    ({"k_pages": torch.zeros(4, 8, 2, 64), "v_pages": torch.zeros(4, 8, 2, 64)}, "bf16 or fp16"),
    ({"k_pages": torch.zeros(4, 6, 2, 64).half(), "v_pages": torch.zeros(4, 6, 2, 64).half()}, "page_size"),
    ({"k_pages": torch.zeros(4, 8, 2, 20).half(), "v_pages": torch.zeros(4, 8, 2, 20).half()}, "head_dim"),
    ({"k_pages": torch.zeros(4, 1, 2, 64).half().expand(4, 8, 2, 64)}, "overlap"),
    ({"block_table": torch.zeros(3, 2).int()}, "block_table"),
    ({"block_table": torch.zeros(2, 0).int()}, "block_table"),
    ({"kv_lens": torch.zeros(3).int()}, "kv_lens"),
    ({"counts": torch.zeros(1).int()}, "counts"),
    ({"cu_seqlens": torch.zeros(1).int()}, "offsets"),
    ({"path": torch.zeros(2).int()}, "path"),
    ({"path": torch.zeros(3, 4).int()}, "path"),
    ({"slot_positions": torch.zeros(2, 2, 15).int()}, "slot_positions"),
    ({"slot_positions": torch.zeros(2, 2, 16)}, "slot_positions"),
    ({"slot_positions": torch.zeros(2, 2, 32).int()[..., ::2]}, "slot_positions"),
])
def test_commit(change, match):
    args = {"k_pages": torch.zeros(4, 8, 2, 64).half(), "v_pages": torch.zeros(4, 8, 2, 64).half(),
            "block_table": torch.zeros(2, 2).int(), "kv_lens": LENS.int(), "cu_seqlens": CU.int(),
            "path": torch.zeros(2, 3).int(), "counts": torch.zeros(2).int(), **change}
    with pytest.raises(KernelError, match=match):
        commit_draft_paged(**args)


def test_c_entries_refuse_before_any_launch():
    lib = _native.load_library()
    fake = ctypes.c_void_p(16)  # never dereferenced

    def refused(rc, code, text):
        assert rc == code and text in lib.tasft_last_error(), (rc, lib.tasft_last_error())

    refused(lib.tasft_draft_tree(None, fake, fake, fake, fake, 1, 5, 5, None), -1, b"null")
    refused(lib.tasft_draft_tree(fake, fake, fake, fake, fake, 0, 5, 5, None), -1, b"positive")
    refused(lib.tasft_draft_tree(fake, fake, fake, fake, fake, 1, 5, 4097, None), -2, b"4096")
    refused(lib.tasft_draft_tree(fake, fake, fake, ctypes.c_void_p(12), fake, 1, 5, 5, None), -1, b"aligned")
    refused(lib.tasft_draft_accept(fake, fake, None, None, fake, fake, fake, fake, 1, 5, 5, 1, None), -1, b"null")
    refused(lib.tasft_draft_accept(fake, fake, fake, None, fake, fake, fake, fake, 1, 5, 9999, 1, None), -2, b"4096")
    st = _native.kept_strides((1024, 128, 64, 1))

    def commit(out=ctypes.c_void_p(32), d=64, page=8, pages=4, ks=st, heads=2):
        return lib.tasft_draft_commit_paged(fake, fake, fake, fake, fake, fake, fake, out, None, 2, 5, heads, d, page, pages,
                                            3, ks, st, 3, None)

    refused(commit(out=None), -1, b"null")
    refused(commit(out=fake), -1, b"kv_lens_out")
    refused(commit(d=20), -2, b"head_dim")
    refused(commit(page=6), -2, b"page_size")
    refused(commit(pages=0), -1, b"positive")
    refused(commit(ks=_native.kept_strides((1024, 128, 60, 1))), -1, b"multiples of 8")
    refused(commit(ks=_native.kept_strides((1024, 128, 64, 2))), -1, b"contiguous")
    refused(commit(ks=_native.kept_strides((1024, -128, 64, 1))), -1, b"non-negative")

    sq, so = _native.kept_strides((256, 64, 1)), _native.kept_strides((256, 64, 1))

    def chunk(mask=None, ancestors=None, words=0, scale=0.1, cap=0.0, causal=1, longest=100):
        return lib.tasft_chunk_scored_fwd(
            fake, fake, fake, fake, None, mask, fake, fake, fake, None, ancestors, words, None, 0, 2, 200, 4, 2, longest,
            64, 64, 3, 8, 4, 3, 1, sq, st, st, so, st, 3, scale, cap, causal, 0, None)

    refused(chunk(scale=0.0), -1, b"scale")
    refused(chunk(cap=-1.0), -1, b"softcap")
    refused(chunk(cap=float("nan")), -1, b"softcap")
    refused(chunk(ancestors=fake, words=0), -1, b"words")
    refused(chunk(ancestors=ctypes.c_void_p(20), words=2), -1, b"aligned")
    refused(chunk(ancestors=fake, words=1), -1, b"a bit a token")
    refused(chunk(ancestors=fake, words=2, causal=0), -1, b"causal")
    refused(chunk(ancestors=fake, words=2, mask=fake), -1, b"mask")
