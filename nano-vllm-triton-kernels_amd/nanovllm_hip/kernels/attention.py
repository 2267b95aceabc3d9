"""Attention over the paged KV cache: the HIP replacements of the two flash-attn calls in nano-vllm's layers.

flash_attn_varlen_func (prefill, nanovllm/layers/attention.py:77-83): variable-length causal attention over the
new tokens' own k, v, or -- with a block table (the prefix cache, a mixed prefill + decode step) -- over the paged
caches. Kernel: csrc/prefill_attention.hip; with a block table, the sequences that bring at most 16 / (Hq / Hkv)
queries (a mixed step's decode requests) run inside the same call in the paged decode kernel.

flash_attn_with_kvcache (decode):

nanovllm/layers/attention.py:84-90 reshapes q to [num_seqs, q_len, Hq, D] and calls
    flash_attn_with_kvcache(q, k_cache, v_cache, cache_seqlens=context_lens, block_table=block_tables,
                            softmax_scale=scale, causal=True)
on the paged cache [num_blocks, block_size, Hkv, D] that the fused qk_norm_rope_kv kernel writes. The function
below takes the same arguments and returns the same [num_seqs, q_len, Hq, D] output (query i of a sequence sees the
cache up to context_len - q_len + i with causal=True; a sequence with context_len 0 gets zeros). The kernel is
csrc/paged_attention.hip.

Not in the reference, both csrc/tree_attention.hip: flash_attn_with_kvcache_mxfp8, the decode call over the 8-bit cache,
and tree_attention_with_kvcache, the verification of a tree of drafted tokens over either cache.
"""
import torch

import nanovllm_hip.ops  # noqa: F401  (registers torch.ops.nvhip)
from nanovllm_hip.kernels.kvcache_mxfp8 import check_caches


def flash_attn_with_kvcache(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                            cache_seqlens: torch.Tensor, block_table: torch.Tensor, softmax_scale: float | None = None,
                            causal: bool = False) -> torch.Tensor:
    """q [num_seqs, q_len, Hq, D] bf16 -> o [num_seqs, q_len, Hq, D] bf16, attending over the paged caches."""
    assert q.dim() == 4 and q.dtype == torch.bfloat16, (q.shape, q.dtype)
    num_seqs, q_len, Hq, D = q.shape
    assert k_cache.dim() == 4 and k_cache.shape == v_cache.shape and k_cache.shape[3] == D, (k_cache.shape, D)
    assert k_cache.dtype == v_cache.dtype == torch.bfloat16
    assert k_cache.is_contiguous() and v_cache.is_contiguous()
    assert Hq % k_cache.shape[2] == 0, (Hq, k_cache.shape[2])
    assert block_table.dtype == torch.int32 and block_table.dim() == 2 and block_table.shape[0] == num_seqs
    assert cache_seqlens.dtype == torch.int32 and cache_seqlens.shape == (num_seqs,)
    block_table = block_table.contiguous()
    cache_seqlens = cache_seqlens.contiguous()
    if q.stride(-1) != 1 or q.stride(1) != Hq * q.stride(2) or q.stride(0) != q_len * q.stride(1):
        q = q.contiguous()
    scale = D ** -0.5 if softmax_scale is None else float(softmax_scale)
    o = torch.ops.nvhip.paged_decode_attention(q.view(num_seqs * q_len, Hq, D), k_cache, v_cache, block_table,
                                               cache_seqlens, q_len, scale, causal)
    return o.view(num_seqs, q_len, Hq, D)


paged_decode_attention = flash_attn_with_kvcache


def _packed_heads(t, D):
    st = t.stride()
    return (st[2] == 1 and st[1] == D and st[0] % 8 == 0 and t.dtype == torch.bfloat16
            and t.data_ptr() % 16 == 0)


def qk_norm_rope_kv_decode_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor,
                                     q_weight: torch.Tensor, k_weight: torch.Tensor, eps: float,
                                     cos_sin_cache: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                                     slot_mapping: torch.Tensor, cache_seqlens: torch.Tensor,
                                     block_table: torch.Tensor, softmax_scale: float | None = None) -> torch.Tensor:
    """One decode token per sequence: qk_norm_rope_kv(q, k, v, ...) (writing the new k / v into the caches)
    followed by flash_attn_with_kvcache(q_out, k_cache, v_cache, cache_seqlens, block_table, causal=True), in one
    launch -> o [B, Hq, D]. q [B, Hq, D], k / v [B, Hkv, D] the raw (strided) views of the qkv projection, the other
    arguments those of the two calls. The normed and rotated q / k are bitwise those of qk_norm_rope_kv and the
    output that of the two-step sequence; q_out is not written. Falls back to the two calls for layouts the fused
    kernel does not take (head_dim other than 64 / 128, unaligned rows, more than 16 q heads per kv head)."""
    from nanovllm_hip.kernels.qk_norm_rope_kv import qk_norm_rope_kv
    B, Hq, D = q.shape
    Hkv = k.shape[1]
    scale = D ** -0.5 if softmax_scale is None else float(softmax_scale)
    cs = cos_sin_cache.reshape(cos_sin_cache.shape[0], -1)
    assert block_table.dtype == torch.int32 and block_table.dim() == 2 and block_table.shape[0] == B
    assert cache_seqlens.dtype == torch.int32 and cache_seqlens.shape == (B,)
    assert k_cache.dim() == 4 and k_cache.shape == v_cache.shape and k_cache.shape[3] == D
    assert k_cache.dtype == v_cache.dtype == torch.bfloat16
    ok = (D in (64, 128) and Hq % Hkv == 0 and Hq // Hkv <= 16 and k.shape == v.shape == (B, Hkv, D)
          and _packed_heads(q, D) and _packed_heads(k, D) and _packed_heads(v, D)
          and q_weight.is_contiguous() and k_weight.is_contiguous() and q_weight.data_ptr() % 16 == 0
          and k_weight.data_ptr() % 16 == 0 and cs.dtype == torch.float32 and cs.stride(1) == 1
          and cs.shape[1] == D and cs.stride(0) % 4 == 0 and cs.data_ptr() % 16 == 0
          and k_cache.is_contiguous() and v_cache.is_contiguous() and k_cache.shape[2:] == (Hkv, D)
          and positions.dtype == torch.int64 and positions.shape == (B,) and slot_mapping.dtype == torch.int32
          and slot_mapping.shape == (B,) and cache_seqlens.dtype == torch.int32 and block_table.dtype == torch.int32)
    if not ok:
        q_out, _ = qk_norm_rope_kv(q, k, v, positions, q_weight, k_weight, eps, cos_sin_cache, k_cache, v_cache,
                                   slot_mapping, False)
        return flash_attn_with_kvcache(q_out.view(B, 1, Hq, D), k_cache, v_cache, cache_seqlens, block_table, scale,
                                       causal=True).view(B, Hq, D)
    return torch.ops.nvhip.qk_norm_rope_kv_decode_attention(
        q, k, v, positions.contiguous(), q_weight, k_weight, float(eps), cs, k_cache, v_cache,
        slot_mapping.contiguous(), cache_seqlens.contiguous(), block_table.contiguous(), scale)


def flash_attn_varlen_func(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, max_seqlen_q: int,
                           cu_seqlens_q: torch.Tensor, max_seqlen_k: int, cu_seqlens_k: torch.Tensor,
                           softmax_scale: float | None = None, causal: bool = False,
                           block_table: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """q [Tq, Hq, D] bf16 -> o [Tq, Hq, D]. Without block_table k, v are [Tk, Hkv, D] (the new tokens' own keys);
    with it they are the paged caches [num_blocks, block_size, Hkv, D]. Query i of a sequence with lq queries and
    lk keys sees keys j <= lk - lq + i when causal. out: an optional [Tq, Hq, D] bf16 tensor (dims contiguous,
    8-byte aligned rows) the result is written into and returned -- an addition of this package, so that a caller
    with a fixed output buffer (piecewise graphs) needs no copy."""
    assert q.dim() == 3 and q.dtype == torch.bfloat16 and q.stride(-1) == 1, (q.shape, q.dtype)
    Tq, Hq, D = q.shape
    assert k.dtype == v.dtype == torch.bfloat16 and k.shape == v.shape and k.shape[-1] == D
    assert cu_seqlens_q.dtype == cu_seqlens_k.dtype == torch.int32 and cu_seqlens_q.shape == cu_seqlens_k.shape
    if block_table is None:
        assert k.dim() == 3 and k.stride(-1) == 1 and v.stride(-1) == 1
        assert k.stride(1) == D and v.stride(1) == D, "heads of a k/v row must be contiguous"
        Hkv = k.shape[1]
    else:
        assert k.dim() == 4 and k.is_contiguous() and v.is_contiguous()
        assert block_table.dtype == torch.int32 and block_table.dim() == 2
        assert block_table.shape[0] == cu_seqlens_q.shape[0] - 1
        block_table = block_table.contiguous()
        Hkv = k.shape[2]
    assert Hq % Hkv == 0, (Hq, Hkv)
    if q.stride(1) % 8 or q.stride(0) % 8:
        q = q.contiguous()
    scale = D ** -0.5 if softmax_scale is None else float(softmax_scale)
    if out is not None:
        assert out.shape == q.shape and out.dtype == torch.bfloat16 and out.stride(2) == 1, (out.shape, out.stride())
        assert out.stride(1) % 4 == 0 and out.stride(0) % 4 == 0 and out.data_ptr() % 8 == 0
        torch.ops.nvhip.prefill_attention_out(q, k, v, cu_seqlens_q.contiguous(), cu_seqlens_k.contiguous(),
                                              int(max_seqlen_q), int(max_seqlen_k), scale, causal, block_table, out)
        return out
    return torch.ops.nvhip.prefill_attention(q, k, v, cu_seqlens_q.contiguous(), cu_seqlens_k.contiguous(),
                                             int(max_seqlen_q), int(max_seqlen_k), scale, causal, block_table)


def _few_queries(q, k_cache, v_cache, k_scales, v_scales, cache_seqlens, block_table, mask, softmax_scale, causal):
    assert q.dim() == 4 and q.dtype == torch.bfloat16, (q.shape, q.dtype)
    B, n, Hq, D = q.shape
    assert 1 <= n <= 64, n
    if k_scales is None:
        assert k_cache.dim() == 4 and k_cache.shape == v_cache.shape, (k_cache.shape, v_cache.shape)
        assert k_cache.dtype == v_cache.dtype == torch.bfloat16
        assert k_cache.is_contiguous() and v_cache.is_contiguous()
        Hkv = k_cache.shape[2]
    else:
        Hkv = check_caches(k_cache, v_cache, k_scales, v_scales)[1]
    assert k_cache.shape[3] == D and D in (64, 128, 256), (k_cache.shape, D)
    assert Hq % Hkv == 0, (Hq, Hkv)
    assert block_table.dtype == torch.int32 and block_table.dim() == 2 and block_table.shape[0] == B
    assert cache_seqlens.dtype == torch.int32 and cache_seqlens.shape == (B,)
    st = q.stride()
    if (st[3] != 1 or st[2] % 8 or st[1] % 8 or st[2] < D or st[1] < Hq * st[2] or (B > 1 and st[0] != n * st[1])
            or q.data_ptr() % 16):
        q = q.clone(memory_format=torch.contiguous_format)
    scale = D ** -0.5 if softmax_scale is None else float(softmax_scale)
    return torch.ops.nvhip.tree_attention(q, k_cache, v_cache, k_scales, v_scales, block_table.contiguous(),
                                          cache_seqlens.contiguous(), mask, scale, causal)


def flash_attn_with_kvcache_mxfp8(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scales: torch.Tensor,
                                  v_scales: torch.Tensor, cache_seqlens: torch.Tensor, block_table: torch.Tensor,
                                  softmax_scale: float | None = None, causal: bool = False) -> torch.Tensor:
    """flash_attn_with_kvcache over the 8-bit cache (layout and format: kernels.kvcache_mxfp8): q [num_seqs, q_len, Hq, D]
    bf16, q_len <= 64 -> o, the same shape. The codes are read as what they stand for, exactly; the arithmetic is that of
    the bf16 cache's attention. Query i sees the cache up to cache_seqlens - q_len + i with causal=True, all of it
    without; a query that sees nothing gets zeros. Kernel: csrc/tree_attention.hip."""
    assert k_scales is not None and v_scales is not None, "the 8-bit cache has scales"
    return _few_queries(q, k_cache, v_cache, k_scales, v_scales, cache_seqlens, block_table, None, softmax_scale, causal)


def tree_attention_with_kvcache(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                                cache_seqlens: torch.Tensor, block_table: torch.Tensor, tree_mask: torch.Tensor,
                                softmax_scale: float | None = None, k_scales: torch.Tensor | None = None,
                                v_scales: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of a tree of n <= 64 drafted tokens per sequence, the step that verifies them: q [num_seqs, n, Hq, D] bf16
    -> o, the same shape. The nodes' keys and values are stored first, as the sequence's last n cached tokens
    (cache_seqlens counts them). Node i sees the tokens before the tree and, of the tree, node j where bit j of
    tree_mask[b, i] is set: its ancestors and itself (tree_mask() makes the row of a tree from its nodes' parents).
    tree_mask [num_seqs, n] int64; bits from n on are ignored. A node that sees nothing gets zeros; a batch of smaller trees
    is padded with nodes that no mask names.
    k_cache, v_cache: bf16 [num_blocks, block_size, Hkv, D], or, with k_scales and v_scales, the 8-bit caches of
    kernels.kvcache_mxfp8. Kernel: csrc/tree_attention.hip."""
    assert (k_scales is None) == (v_scales is None), "k_scales and v_scales are given together"
    assert tree_mask.dtype == torch.int64 and tree_mask.shape == q.shape[:2], (tree_mask.dtype, tree_mask.shape)
    return _few_queries(q, k_cache, v_cache, k_scales, v_scales, cache_seqlens, block_table, tree_mask.contiguous(),
                        softmax_scale, False)


def tree_mask(parents: list[int]) -> list[int]:
    """The masks of a tree's nodes, as tree_attention_with_kvcache takes them, from each node's parent (an earlier node, or
    -1 for a child of the last accepted token): bit j of entry i says that node i sees node j."""
    assert len(parents) <= 64, len(parents)
    masks = []
    for i, p in enumerate(parents):
        assert -1 <= p < i, f"node {i}: parent {p} is no earlier node"
        masks.append((masks[p] if p >= 0 else 0) | 1 << i)
    return [m - (1 << 64) if m >> 63 else m for m in masks]  # as int64
