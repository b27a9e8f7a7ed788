"""Packed tree attention over the 8-bit paged cache (``fp8_cache``).

``packed_tree_attention_gqa``'s operands and metadata (tree_gqa.py), with each layer's K / V
pools held as e4m3 codes and power-of-two row scales: half the bytes of a 16-bit cache to hold
and to read.  An ordinary decode step is the same call on trees of one node.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _launch, _lib
from .fp8_cache import check_layer
from .tree_gqa import _check_metadata

MAX_HEAD_DIM = 128
MAX_GROUPS = 128
_WORKSPACE_SIZES: dict = {}


def packed_tree_attention_fp8(q, k_pool, v_pool, k_scale, v_scale, metadata, scale,
                              num_queries_per_kv, *, output_dtype=None):
    """Attention of every packed tree node over its request's prefix and its ancestors.

    ``q`` [Q, q_heads, dim] in BF16 or FP16; ``k_pool`` / ``v_pool`` [pages, block_size,
    kv_heads, dim] e4m3 with ``k_scale`` / ``v_scale`` [pages, kv_heads, block_size];
    ``metadata`` a ``PackedTreeMetadata``.  fp32 scores, softmax and sums; returns the output
    in ``q``'s dtype, or FP32 on request.  A row that sees no key gives zeros; one that sees a
    NaN row of the cache gives NaN.  A key whose page or slot lies outside the pool is left out;
    requests that cannot be taken (trees above 1024 nodes, rows outside the packed ones, device
    counts that the host's rule out) give zeros.  Both set a device error bit
    (``read_device_errors``).
    """
    shape, pool_shape, dtype = q.shape, k_pool.shape, q.dtype
    if len(shape) != 3 or shape[0] != metadata.total_queries:
        raise ValueError("packed queries do not match the metadata")
    if (len(pool_shape) != 4 or v_pool.shape != pool_shape
            or pool_shape[1] != metadata.block_size):
        raise ValueError("packed K/V page geometry does not match metadata")
    check_layer(k_pool, v_pool, k_scale, v_scale)
    total, q_heads, dim = shape
    kv_heads = pool_shape[2]
    if dim != pool_shape[3] or dim % 16 or not 16 <= dim <= MAX_HEAD_DIM:
        raise ValueError("head dim must be the pool's, a multiple of 16 up to 128")
    groups = num_queries_per_kv
    if (isinstance(groups, bool) or not isinstance(groups, int) or not 1 <= groups <= MAX_GROUPS
            or q_heads != kv_heads * groups):
        raise ValueError("invalid packed GQA head grouping")
    if dtype != torch.bfloat16 and dtype != torch.float16:
        raise ValueError("8-bit cache attention takes BF16 or FP16 queries")
    if output_dtype not in (None, dtype, torch.float32):
        raise ValueError("output dtype must match the queries or be FP32")
    if not 0 < scale < math.inf:
        raise ValueError("the softmax scale must be positive and finite")
    device = q.device
    if (not q.is_cuda or k_pool.device != device or v_pool.device != device
            or metadata.tree_slots.device != device):
        raise ValueError("packed attention requires CUDA queries, KV and metadata on one device")
    if q.stride(2) != 1 or k_pool.stride(3) != 1 or v_pool.stride(3) != 1:
        raise ValueError("queries and pools need a contiguous head dimension")
    _check_metadata(metadata)
    out = torch.empty(shape, dtype=output_dtype or dtype, device=device)
    if total == 0:
        return out
    from . import ops

    if ops.compiling():
        m = metadata
        torch.ops.jetspec_b200.tree_attention_fp8_(
            out, q, k_pool, v_pool, k_scale, v_scale, m.cu_seqlens_q, m.query_to_request,
            m.query_local_row, m.prefix_lens, m.node_counts, m.block_tables, m.tree_slots,
            m.qq_bias, m.qq_bias_offsets, float(scale), groups)
    else:
        _launch_attention(out, q, k_pool, v_pool, k_scale, v_scale, metadata, scale, groups)
    return out


def _node_range(metadata) -> tuple[int, int]:
    """Least (above zero) and largest node count, (0, 0) when the host does not know them."""
    counts = getattr(metadata, "node_counts_host", None)
    if not counts:
        return 0, 0
    low, high = min(counts), max(counts)
    return low or min((c for c in counts if c), default=0), high


def _launch_attention(out, q, k_pool, v_pool, k_scale, v_scale, m, scale, groups) -> None:
    """jt_tree_attn_fp8_launch on the current stream (validated arguments)."""
    lib = _lib.load_library()
    codes = _launch.DTYPE_CODES
    device = q.device
    total, _, dim = q.shape
    blocks, block_size, kv_heads, _ = k_pool.shape
    requests = m.prefix_lens.shape[0]
    shape = (requests, total, kv_heads, groups, dim)
    nbytes = _WORKSPACE_SIZES.get(shape)
    if nbytes is None:
        nbytes = lib.jt_tree_attn_fp8_workspace_size(*shape)
        if nbytes < 0:
            raise ValueError("8-bit cache attention: invalid geometry")
        _launch.remember(_WORKSPACE_SIZES, shape, nbytes)
    stream = _launch.raw_stream(device)
    qs, os_, ks, vs = q.stride(), out.stride(), k_pool.stride(), v_pool.stride()
    kss, vss = k_scale.stride(), v_scale.stride()
    p = _lib.JtTreeAttnFp8Params(
        out.data_ptr(), q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), k_scale.data_ptr(),
        v_scale.data_ptr(), m.cu_seqlens_q.data_ptr(), m.query_to_request.data_ptr(),
        m.query_local_row.data_ptr(), m.prefix_lens.data_ptr(), m.node_counts.data_ptr(),
        m.block_tables.data_ptr(), m.tree_slots.data_ptr(), m.qq_bias.data_ptr(),
        m.qq_bias_offsets.data_ptr(), None, nbytes,
        blocks, qs[0], qs[1], os_[0], os_[1], m.block_tables.stride(0), ks[0], ks[1], ks[2],
        vs[0], vs[1], vs[2], kss[0], kss[1], vss[0], vss[1], scale, requests, total, kv_heads,
        groups, dim, block_size, m.block_tables.shape[1], codes[q.dtype], codes[out.dtype],
        *_node_range(m))

    def launch(scratch):
        p.workspace = scratch
        return lib.jt_tree_attn_fp8_launch(ctypes.byref(p), stream)

    _lib.check(_launch.with_workspace(device, nbytes, stream, launch))
