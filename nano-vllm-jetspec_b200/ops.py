"""torch.library registration of the launchers (the custom-op half of the boundary).

The Python wrappers call the C ABI through ctypes, which a tracing compiler cannot see
into: a ``torch.compile``d caller (the reference compiles its norms and rotary embedding,
nanovllm/layers/layernorm.py, rotary_embedding.py) would break its graph at every kernel.
Each launcher is therefore also a custom operator in the ``jetspec_b200`` namespace, with
a fake (shape-only) implementation, and the public wrappers route through it while
``torch.compiler.is_compiling()``; eager calls keep the direct launch (no dispatcher
overhead).  The operators mutate their output arguments in place and return nothing, so
functionalisation sees exactly which buffers they write.

* ``jetspec_b200::tree_attention_`` - out[Q, Hq, D] <- packed tree attention
* ``jetspec_b200::kv_store_``       - k_cache / v_cache rows <- key / value
* ``jetspec_b200::kv_commit_``      - kv_pool accepted rows moved to their destinations
* ``jetspec_b200::rope_scatter_``   - out <- rope(q); k_pool / v_pool <- rope(k) / v
* ``jetspec_b200::request_maps_``   - block tables, slots, positions <- request lengths
* ``jetspec_b200::qk_norm_rope_``   - q_out / k_out <- rotated normed heads
* ``jetspec_b200::qk_norm_rope_store_`` - q_out and the cache rows <- rotated normed heads
* ``jetspec_b200::kv_fp8_commit_``  - kv_pool / kv_scale accepted rows moved
* ``jetspec_b200::tree_attention_fp8_`` - out <- tree attention over the 8-bit cache
"""
from __future__ import annotations

from types import SimpleNamespace
from typing import Optional

import torch

NAMESPACE = "jetspec_b200"


@torch.library.custom_op(f"{NAMESPACE}::tree_attention_", mutates_args=("out",))
def tree_attention_(out: torch.Tensor, q: torch.Tensor, k_pool: torch.Tensor,
                    v_pool: torch.Tensor, cu_seqlens_q: torch.Tensor,
                    query_to_request: torch.Tensor, query_local_row: torch.Tensor,
                    prefix_lens: torch.Tensor, node_counts: torch.Tensor,
                    block_tables: torch.Tensor, tree_slots: torch.Tensor, qq_bias: torch.Tensor,
                    qq_bias_offsets: torch.Tensor, block_size: int, scale: float, groups: int,
                    fp32_probability: bool, split_keys: int, portable_core: bool) -> None:
    from .tree_gqa import launch_tree_attention_eager

    metadata = SimpleNamespace(
        cu_seqlens_q=cu_seqlens_q, query_to_request=query_to_request,
        query_local_row=query_local_row, prefix_lens=prefix_lens, node_counts=node_counts,
        block_tables=block_tables, tree_slots=tree_slots, qq_bias=qq_bias,
        qq_bias_offsets=qq_bias_offsets, block_size=block_size,
        num_requests=int(prefix_lens.numel()), total_queries=int(q.shape[0]),
        node_counts_host=None)
    launch_tree_attention_eager(out, q, k_pool, v_pool, metadata, scale, groups,
                                fp32_probability=fp32_probability, split_keys=split_keys,
                                portable_core=portable_core)


@tree_attention_.register_fake
def _(out, q, k_pool, v_pool, cu_seqlens_q, query_to_request, query_local_row, prefix_lens,
      node_counts, block_tables, tree_slots, qq_bias, qq_bias_offsets, block_size, scale,
      groups, fp32_probability, split_keys, portable_core):
    return None


@torch.library.custom_op(f"{NAMESPACE}::kv_store_", mutates_args=("k_cache", "v_cache"))
def kv_store_(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor,
              v_cache: torch.Tensor, slot_mapping: torch.Tensor) -> None:
    from .attention import _store

    _store(key, value, k_cache, v_cache, slot_mapping)


@kv_store_.register_fake
def _(key, value, k_cache, v_cache, slot_mapping):
    return None


@torch.library.custom_op(f"{NAMESPACE}::kv_commit_", mutates_args=("kv_pool",))
def kv_commit_(kv_pool: torch.Tensor, source_slots: torch.Tensor,
               destination_slots: torch.Tensor, block_size: int) -> None:
    from .state import _commit

    _commit(kv_pool, source_slots, destination_slots, block_size)


@kv_commit_.register_fake
def _(kv_pool, source_slots, destination_slots, block_size):
    return None


@torch.library.custom_op(f"{NAMESPACE}::rope_scatter_",
                         mutates_args=("k_pool", "v_pool", "out"))
def rope_scatter_(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor,
                  cos_sin_cache: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                  node_slots: torch.Tensor, out: torch.Tensor) -> None:
    from .tree_fusion import _rope_scatter_launch

    _rope_scatter_launch(q, k, v, positions, cos_sin_cache, k_pool, v_pool, node_slots, out)


@rope_scatter_.register_fake
def _(q, k, v, positions, cos_sin_cache, k_pool, v_pool, node_slots, out):
    return None


@torch.library.custom_op(f"{NAMESPACE}::request_maps_",
                         mutates_args=("block_tables", "slots", "positions", "owners", "cu",
                                       "lens", "taken"))
def request_maps_(block_tables: torch.Tensor, cached_lens: torch.Tensor, new_lens: torch.Tensor,
                  free_pages: torch.Tensor, block_size: int, slots: torch.Tensor,
                  positions: torch.Tensor, owners: torch.Tensor, cu: torch.Tensor,
                  lens: torch.Tensor, taken: torch.Tensor) -> None:
    from .request_maps import _launch_maps

    _launch_maps(block_tables, cached_lens, new_lens, free_pages, block_size, slots, positions,
                 owners, cu, lens, taken)


@request_maps_.register_fake
def _(block_tables, cached_lens, new_lens, free_pages, block_size, slots, positions, owners, cu,
      lens, taken):
    return None


@torch.library.custom_op(f"{NAMESPACE}::qk_norm_rope_", mutates_args=("q_out", "k_out"))
def qk_norm_rope_(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor,
                  k_weight: torch.Tensor, positions: torch.Tensor, cos_sin_cache: torch.Tensor,
                  eps: float, q_out: torch.Tensor, k_out: torch.Tensor) -> None:
    from .qk_norm_rope import _launch_norm

    _launch_norm(q, k, q_weight, k_weight, positions, cos_sin_cache, eps, q_out, k_out)


@qk_norm_rope_.register_fake
def _(q, k, q_weight, k_weight, positions, cos_sin_cache, eps, q_out, k_out):
    return None


@torch.library.custom_op(f"{NAMESPACE}::qk_norm_rope_store_",
                         mutates_args=("k_pool", "v_pool", "k_scale", "v_scale", "q_out"))
def qk_norm_rope_store_(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                        q_weight: torch.Tensor, k_weight: torch.Tensor, positions: torch.Tensor,
                        cos_sin_cache: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                        slots: torch.Tensor, eps: float, k_scale: Optional[torch.Tensor],
                        v_scale: Optional[torch.Tensor], q_out: torch.Tensor) -> None:
    from .qk_norm_rope import _launch_norm

    _launch_norm(q, k, q_weight, k_weight, positions, cos_sin_cache, eps, q_out, None, v, k_pool,
                 v_pool, slots, k_scale, v_scale)


@qk_norm_rope_store_.register_fake
def _(q, k, v, q_weight, k_weight, positions, cos_sin_cache, k_pool, v_pool, slots, eps, k_scale,
      v_scale, q_out):
    return None


@torch.library.custom_op(f"{NAMESPACE}::kv_fp8_commit_", mutates_args=("kv_pool", "kv_scale"))
def kv_fp8_commit_(kv_pool: torch.Tensor, kv_scale: torch.Tensor, source_slots: torch.Tensor,
                   destination_slots: torch.Tensor) -> None:
    from .fp8_cache import _launch_commit

    _launch_commit(kv_pool, kv_scale, source_slots, destination_slots)


@kv_fp8_commit_.register_fake
def _(kv_pool, kv_scale, source_slots, destination_slots):
    return None


@torch.library.custom_op(f"{NAMESPACE}::tree_attention_fp8_", mutates_args=("out",))
def tree_attention_fp8_(out: torch.Tensor, q: torch.Tensor, k_pool: torch.Tensor,
                        v_pool: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                        cu_seqlens_q: torch.Tensor, query_to_request: torch.Tensor,
                        query_local_row: torch.Tensor, prefix_lens: torch.Tensor,
                        node_counts: torch.Tensor, block_tables: torch.Tensor,
                        tree_slots: torch.Tensor, qq_bias: torch.Tensor,
                        qq_bias_offsets: torch.Tensor, scale: float, groups: int) -> None:
    # Without the host's node counts (which would be guards of the graph): the launch covers
    # small and large trees.
    from .tree_fp8 import _launch_attention

    metadata = SimpleNamespace(
        cu_seqlens_q=cu_seqlens_q, query_to_request=query_to_request,
        query_local_row=query_local_row, prefix_lens=prefix_lens, node_counts=node_counts,
        block_tables=block_tables, tree_slots=tree_slots, qq_bias=qq_bias,
        qq_bias_offsets=qq_bias_offsets, node_counts_host=None)
    _launch_attention(out, q, k_pool, v_pool, k_scale, v_scale, metadata, scale, groups)


@tree_attention_fp8_.register_fake
def _(out, q, k_pool, v_pool, k_scale, v_scale, cu_seqlens_q, query_to_request, query_local_row,
      prefix_lens, node_counts, block_tables, tree_slots, qq_bias, qq_bias_offsets, scale,
      groups):
    return None


def compiling() -> bool:
    """True while torch.compile traces the caller (route through the operators)."""
    return torch.compiler.is_compiling()
