"""Block tables, slot maps and positions of a round, built on the GPU from request lengths.

The reference builds them on the host (BlockManager's page lists and the runner's
prepare_prefill / prepare_decode loops, nanovllm/engine/block_manager.py,
nanovllm/engine/model_runner.py) and uploads them every round.  ``build_request_maps`` takes
the lengths and a free list that already live on the GPU, so the maps of a round whose lengths
come out of the device-side acceptance walk need no host in between.  What is left to the host:
the free list has no cursor on the device (the next round's list begins ``pages_taken`` further
on), and ``PackedTreeMetadata``'s builders take page tables of the host.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass

import torch

from . import _launch, _lib


@dataclass(frozen=True)
class RequestMaps:
    """One round's maps.  Entries from the round's total to ``max_tokens`` are padding: slot
    -1 (the cache writes skip it), position 0, request -1."""
    block_tables: torch.Tensor      # i32 [requests, width], the caller's, extended in place
    slot_mapping: torch.Tensor      # i64 [max_tokens]
    positions: torch.Tensor         # i64 [max_tokens]
    token_to_request: torch.Tensor  # i32 [max_tokens]
    cu_seqlens: torch.Tensor        # i32 [requests + 1]
    context_lens: torch.Tensor      # i32 [requests]: cached + new
    pages_taken: torch.Tensor       # i32 [1]: pages the round needs of the free list


def build_request_maps(block_tables: torch.Tensor, cached_lens: torch.Tensor,
                       new_lens: torch.Tensor, free_pages: torch.Tensor, block_size: int, *,
                       max_tokens: int) -> RequestMaps:
    """Maps of a round in which request r, with ``cached_lens[r]`` tokens in its pages, writes
    ``new_lens[r]`` more (0 is allowed).

    Pages beyond ``ceil(cached / block_size)`` are the next entries of ``free_pages``, in
    request order, and are written into ``block_tables`` ([requests, width] int32) in place.
    ``max_tokens`` sizes the per-token outputs (a captured graph's padded length); tokens past
    it are dropped.  When ``pages_taken`` exceeds the free list, the pages past its end are -1
    and so are the slots of their tokens; the same holds for tokens past the table's width.
    One launch on the current stream, no synchronisation.
    """
    requests = cached_lens.shape[0] if cached_lens.ndim == 1 else 0
    if requests < 1 or new_lens.shape != cached_lens.shape:
        raise ValueError("cached and new lengths must be equally sized nonempty vectors")
    if block_tables.ndim != 2 or block_tables.shape[0] != requests or block_tables.shape[1] < 1:
        raise ValueError("block tables must be [requests, width]")
    if free_pages.ndim != 1:
        raise ValueError("free pages must be a vector")
    block_size, max_tokens = int(block_size), int(max_tokens)
    if block_size < 1 or not 0 <= max_tokens < 1 << 31:
        raise ValueError("invalid block size or token capacity")
    i32 = torch.int32
    if (block_tables.dtype != i32 or cached_lens.dtype != i32 or new_lens.dtype != i32
            or free_pages.dtype != i32):
        raise ValueError("block tables, lengths and free pages must be int32")
    device = block_tables.device
    if (not block_tables.is_cuda or cached_lens.device != device or new_lens.device != device
            or free_pages.device != device):
        raise ValueError("request maps require CUDA tensors on one device")
    if (not cached_lens.is_contiguous() or not new_lens.is_contiguous()
            or not free_pages.is_contiguous() or block_tables.stride(1) != 1
            or block_tables.stride(0) < block_tables.shape[1]):
        raise ValueError("lengths, free pages and table rows must be contiguous")
    slots, positions = torch.empty((2, max_tokens), dtype=torch.int64, device=device).unbind(0)
    owners, cu, lens, taken = torch.empty(
        max_tokens + 2 * requests + 2, dtype=i32, device=device).split_with_sizes(
            (max_tokens, requests + 1, requests, 1))
    maps = RequestMaps(block_tables, slots, positions, owners, cu, lens, taken)
    from . import ops

    if ops.compiling():
        torch.ops.jetspec_b200.request_maps_(block_tables, cached_lens, new_lens, free_pages,
                                             block_size, slots, positions, owners, cu, lens, taken)
    else:
        _launch_maps(block_tables, cached_lens, new_lens, free_pages, block_size, slots,
                     positions, owners, cu, lens, taken)
    return maps


def _launch_maps(block_tables, cached_lens, new_lens, free_pages, block_size, slots, positions,
                 owners, cu, lens, taken) -> None:
    """jt_request_maps_launch on the current stream (validated arguments)."""
    lib = _lib.load_library()
    p = _lib.JtRequestMapsParams(
        block_tables.data_ptr(), cached_lens.data_ptr(), new_lens.data_ptr(),
        free_pages.data_ptr(), slots.data_ptr(), positions.data_ptr(), owners.data_ptr(),
        cu.data_ptr(), lens.data_ptr(), taken.data_ptr(), block_tables.stride(0),
        cached_lens.shape[0], block_tables.shape[1], block_size, free_pages.shape[0],
        slots.shape[0])
    _lib.check(lib.jt_request_maps_launch(ctypes.byref(p),
                                          _launch.raw_stream(block_tables.device)))
