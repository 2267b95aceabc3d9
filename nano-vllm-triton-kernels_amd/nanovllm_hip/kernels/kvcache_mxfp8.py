"""The paged KV cache in 8 bits: writing it and reading it back (kernels: csrc/kvcache_mxfp8.hip).

Not in the reference, whose cache holds the model's type (nanovllm/engine/model_runner.py:262-267). The format is the MX
format of the OCP specification with e4m3 elements: 32 consecutive elements of a head row share a power-of-two scale.
  k_cache, v_cache    [num_blocks, Hkv, block_size, D] float8_e4m3fn codes
  k_scales, v_scales  [num_blocks, Hkv, block_size, D / 32] uint8, a scale 2^(byte - 127)
An element is code * scale, exactly a bf16 number; it takes 8.25 bits. Slots are those of the bf16 cache: page
slot // block_size, row slot % block_size -- but the rows of one head in one page are contiguous here. The cache is read
by kernels.attention.flash_attn_with_kvcache_mxfp8 (decode) and tree_attention_with_kvcache; a prompt chunk over a cached
prefix reads it back with load_kvcache_mxfp8 and attends with flash_attn_varlen_func.

Rounding: a block is divided by the least power of two that brings its largest finite magnitude to 448 (the largest code)
or below, and rounded to the nearest code: an element is off by at most 1/16 of itself, or by 2^-10 of the scale where it
is tiny beside the block's largest. An infinity or a NaN becomes NaN and leaves the others of its block as they are.
"""
import torch

import nanovllm_hip.ops  # noqa: F401  (registers torch.ops.nvhip)

MX_BLOCK = 32  # elements that share a scale
_TYPES = (torch.bfloat16, torch.float16, torch.float32)


def allocate_kvcache_mxfp8(num_blocks: int, block_size: int, num_kv_heads: int, head_dim: int,
                           device=None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """An empty cache (all zeros): (k_cache, v_cache, k_scales, v_scales)."""
    assert head_dim in (64, 128, 256), head_dim
    shape = (num_blocks, num_kv_heads, block_size)
    codes = [torch.zeros(*shape, head_dim, dtype=torch.float8_e4m3fn, device=device) for _ in range(2)]
    scales = [torch.zeros(*shape, head_dim // MX_BLOCK, dtype=torch.uint8, device=device) for _ in range(2)]
    return codes[0], codes[1], scales[0], scales[1]


def check_caches(k_cache, v_cache, k_scales, v_scales):
    """Asserts the layout above; the codes' shape."""
    shape = k_cache.shape
    assert len(shape) == 4 and shape == v_cache.shape and shape[3] in (64, 128, 256), (shape, v_cache.shape)
    assert k_cache.dtype == v_cache.dtype == torch.float8_e4m3fn, (k_cache.dtype, v_cache.dtype)
    assert k_scales.dtype == v_scales.dtype == torch.uint8, (k_scales.dtype, v_scales.dtype)
    assert k_scales.shape == v_scales.shape == (shape[0], shape[1], shape[2], shape[3] // MX_BLOCK), k_scales.shape
    assert (k_cache.is_contiguous() and v_cache.is_contiguous() and k_scales.is_contiguous()
            and v_scales.is_contiguous())
    return shape


def store_kvcache_mxfp8(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                        k_scales: torch.Tensor, v_scales: torch.Tensor, slot_mapping: torch.Tensor) -> None:
    """Quantises key, value [N, Hkv, D] (bf16, fp16 or fp32; heads contiguous, rows may be strided views of the qkv
    projection) into the slots slot_mapping [N] int32 (-1, or any slot outside the cache: skipped). A slot may be given
    once in a call: of two tokens in one slot, either may be what parts of the row hold."""
    shape, dtype = key.shape, key.dtype
    N, Hkv, D = shape
    cache = check_caches(k_cache, v_cache, k_scales, v_scales)
    assert value.shape == shape and value.dtype == dtype and dtype in _TYPES, (dtype, value.dtype)
    assert cache[1] == Hkv and cache[3] == D, (shape, cache)
    assert key.stride()[1:] == value.stride()[1:] == (D, 1), (key.stride(), value.stride())
    assert slot_mapping.dtype == torch.int32 and slot_mapping.shape == (N,)
    torch.ops.nvhip.store_kvcache_mxfp8(key, value, k_cache, v_cache, k_scales, v_scales, slot_mapping.contiguous())


def load_kvcache_mxfp8(k_cache: torch.Tensor, v_cache: torch.Tensor, k_scales: torch.Tensor, v_scales: torch.Tensor,
                       block_table: torch.Tensor, cu_seqlens_k: torch.Tensor,
                       total_k: int) -> tuple[torch.Tensor, torch.Tensor]:
    """The sequences' tokens in bf16, one sequence behind the other: (k, v) [total_k, Hkv, D], the layout of
    flash_attn_varlen_func's k and v. block_table [B, max_blocks] int32; cu_seqlens_k [B + 1] int32: sequence b's tokens
    0 .. cu[b + 1] - cu[b] - 1 become rows cu[b] .. Rows behind the last sequence (total_k may be more than cu[B], for
    calls of a fixed size) and tokens without a valid page are zeros."""
    check_caches(k_cache, v_cache, k_scales, v_scales)
    assert block_table.dtype == cu_seqlens_k.dtype == torch.int32 and block_table.dim() == 2
    assert cu_seqlens_k.shape == (block_table.shape[0] + 1,), (cu_seqlens_k.shape, block_table.shape)
    assert total_k >= 0, total_k
    return torch.ops.nvhip.load_kvcache_mxfp8(k_cache, v_cache, k_scales, v_scales, block_table.contiguous(),
                                              cu_seqlens_k.contiguous(), total_k)
