"""Block-sparse attention kernels (reference package ``tasft/kernels/__init__.py``)."""
from tasft_amd.kernels.block_sparse_fa import (
    BlockSparseFlashAttention,
    KernelBackend,
    SparsityStats,
    default_chunk_splits,
    default_decode_splits,
    detect_kernels,
    executed_blocks,
    indices_to_mask,
    mask_to_csr,
)
from tasft_amd.kernels.kernel_config import KernelConfig, LayerKernelConfig
from tasft_amd.kernels.paged_cache import accumulate_key_weights, append_paged, evict_paged
from tasft_amd.kernels.rotary import apply_rotary, rotary_frequencies

__all__ = [
    "BlockSparseFlashAttention",
    "KernelBackend",
    "KernelConfig",
    "LayerKernelConfig",
    "SparsityStats",
    "accumulate_key_weights",
    "append_paged",
    "apply_rotary",
    "default_chunk_splits",
    "default_decode_splits",
    "detect_kernels",
    "evict_paged",
    "executed_blocks",
    "indices_to_mask",
    "mask_to_csr",
    "rotary_frequencies",
]
