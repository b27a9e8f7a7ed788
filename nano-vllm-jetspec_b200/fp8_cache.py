"""The 8-bit paged KV cache: its layout, and the accepted-only commit over it.

Codes live in a pool of the usual shape, ``[2, layers, blocks, block_size, kv_heads,
head_dim]`` (K and V, float8_e4m3fn); each (slot, KV head) row has one power-of-two scale
(float8_e8m0fnu) in ``[2, layers, blocks, kv_heads, block_size]``.  A row's value is
``code * scale``: exact in bf16 and fp32, since the scale only moves the exponent.  The scale's
last two dimensions are swapped against the pool's so that the attention reads the scales of
128 consecutive keys of one head as 128 contiguous bytes.  A row that had a non-finite
element has the NaN scale and reads back as NaN.
"""
from __future__ import annotations

import ctypes

import torch

from . import _launch, _lib

CODE_DTYPE = torch.float8_e4m3fn
SCALE_DTYPE = torch.float8_e8m0fnu


def alloc_fp8_kv_cache(layers: int, blocks: int, block_size: int, kv_heads: int, head_dim: int,
                       device) -> tuple[torch.Tensor, torch.Tensor]:
    """(kv_pool, kv_scale) of zeros.  Layer l's views for the other calls: ``kv_pool[0, l]``,
    ``kv_pool[1, l]``, ``kv_scale[0, l]``, ``kv_scale[1, l]``."""
    shape = (2, int(layers), int(blocks), int(block_size), int(kv_heads), int(head_dim))
    if min(shape) < 1:
        raise ValueError("cache dimensions must be positive")
    pool = torch.zeros(shape, dtype=torch.uint8, device=device)
    scale = torch.full(shape[:3] + (shape[4], shape[3]), 127, dtype=torch.uint8, device=device)
    return pool.view(CODE_DTYPE), scale.view(SCALE_DTYPE)


def check_layer(k_pool, v_pool, k_scale, v_scale) -> None:
    """Checks of one layer's 8-bit pools and scales (ValueError)."""
    if k_scale is None or v_scale is None:
        raise ValueError("8-bit pools need k_scale and v_scale")
    if k_pool.dtype != CODE_DTYPE or v_pool.dtype != CODE_DTYPE:
        raise ValueError("8-bit pools must both hold float8_e4m3fn codes")
    if k_scale.dtype != SCALE_DTYPE or v_scale.dtype != SCALE_DTYPE:
        raise ValueError("scales must be float8_e8m0fnu")
    blocks, block_size, heads, _ = k_pool.shape
    shape, device = (blocks, heads, block_size), k_pool.device
    if k_scale.shape != shape or v_scale.shape != shape:
        raise ValueError("scales must be [pages, kv_heads, page_size]")
    if k_scale.stride(2) != 1 or v_scale.stride(2) != 1:
        raise ValueError("scales need a contiguous last dimension")
    if k_scale.device != device or v_scale.device != device:
        raise ValueError("pools and scales must share one device")


def dequantize_kv(pool: torch.Tensor, scale: torch.Tensor, dtype=torch.bfloat16) -> torch.Tensor:
    """The values a pool holds, [..., blocks, block_size, kv_heads, head_dim] in ``dtype`` (a
    plain conversion for inspection and for handing pages to a 16-bit cache)."""
    if pool.dtype != CODE_DTYPE or scale.dtype != SCALE_DTYPE:
        raise ValueError("dequantize_kv takes e4m3 codes and e8m0 scales")
    if pool.ndim < 4 or scale.shape != pool.shape[:-3] + (pool.shape[-2], pool.shape[-3]):
        raise ValueError("scales must be [..., pages, kv_heads, page_size]")
    return (pool.float() * scale.float().transpose(-1, -2).unsqueeze(-1)).to(dtype)


def copy_accepted_kv_fp8(kv_pool: torch.Tensor, kv_scale: torch.Tensor,
                         source_slots: torch.Tensor, destination_slots: torch.Tensor,
                         block_size: int) -> int:
    """Copy accepted rows and their scales across both KV axes and all layers (gather before
    scatter, one launch).

    ``copy_accepted_kv`` (nanovllm/speculative/jetspec/state.py:64-86) for the 8-bit cache:
    same slot maps, same checks; returns the payload in bytes (rows and scales).  One call
    takes at most ``jt_kv_fp8_commit_max_slots()`` slots (12047).
    """
    if source_slots.ndim != 1 or destination_slots.ndim != 1:
        raise ValueError("KV copy requires one-dimensional slot maps")
    n = source_slots.shape[0]
    if destination_slots.shape[0] != n:
        raise ValueError("KV copy source and destination lengths differ")
    shape = kv_pool.shape
    if kv_pool.ndim != 6 or shape[0] != 2 or shape[3] != int(block_size):
        raise ValueError("KV pool must be [2, layers, blocks, block_size, kv_heads, head_dim]")
    if kv_pool.dtype != CODE_DTYPE or kv_scale.dtype != SCALE_DTYPE:
        raise ValueError("an 8-bit commit takes e4m3 codes and e8m0 scales")
    if kv_scale.shape != shape[:3] + (shape[4], shape[3]):
        raise ValueError("KV scales must be [2, layers, blocks, kv_heads, block_size]")
    if n == 0:
        return 0
    device = kv_pool.device
    if (not kv_pool.is_cuda or kv_scale.device != device or source_slots.device != device
            or destination_slots.device != device):
        raise ValueError("KV commit requires the pool, scales and slot maps on one CUDA device")
    if source_slots.dtype not in (torch.int32, torch.int64):
        raise ValueError("slot maps must be int32 or int64")
    if kv_pool.stride(5) != 1 or kv_scale.stride(4) != 1:
        raise ValueError("KV pool rows and scales need a contiguous last dimension")
    if destination_slots.dtype != source_slots.dtype:
        destination_slots = destination_slots.to(source_slots.dtype)
    destination_slots, source_slots = destination_slots.contiguous(), source_slots.contiguous()
    from . import ops

    if ops.compiling():
        torch.ops.jetspec_b200.kv_fp8_commit_(kv_pool, kv_scale, source_slots, destination_slots)
    else:
        _launch_commit(kv_pool, kv_scale, source_slots, destination_slots)
    return n * 2 * shape[1] * shape[4] * (shape[5] + 1)


def _launch_commit(kv_pool, kv_scale, source_slots, destination_slots) -> None:
    """jt_kv_fp8_commit_launch on the current stream (validated arguments)."""
    lib = _lib.load_library()
    _, layers, blocks, block_size, heads, dim = kv_pool.shape
    p = _lib.JtKvFp8CommitParams(
        kv_pool.data_ptr(), kv_scale.data_ptr(), source_slots.data_ptr(),
        destination_slots.data_ptr(), blocks, *kv_pool.stride()[:5], *kv_scale.stride()[:4],
        int(source_slots.dtype == torch.int64), source_slots.shape[0], layers, heads, dim,
        block_size)
    _lib.check(lib.jt_kv_fp8_commit_launch(ctypes.byref(p), _launch.raw_stream(kv_pool.device)))
