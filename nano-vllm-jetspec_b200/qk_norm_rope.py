"""RMS norm of every query and key head with the position rotation in the same pass.

The reference's attention layer norms Q and K (nanovllm/models/qwen3.py:223-225), rotates
them and writes K / V into the cache as separate kernels, rounding to bf16 between the steps.
``qk_norm_rope`` does norm and rotation in one pass over fp32 values with one rounding at the
end; ``qk_norm_rope_store`` also writes the rotated K and the V rows into the paged cache, of
the operand type or in 8 bits (``fp8_cache``).  For a verifier that has to match eager
PyTorch bit for bit, ``rope_scatter`` keeps its rounding points.
"""
from __future__ import annotations

import ctypes

import torch

from . import _launch, _lib
from .fp8_cache import CODE_DTYPE, check_layer

_INDEX = (torch.int32, torch.int64)
_STORE_NONE, _STORE_SAME, _STORE_FP8 = 0, 1, 2


def _check(q, k, q_weight, k_weight, positions, cache, eps):
    # Every attribute of a tensor is a call of 50 to 200 ns: each is read once.
    q_shape, k_shape, cache_shape = q.shape, k.shape, cache.shape
    if (len(q_shape) != 3 or len(k_shape) != 3 or k_shape[0] != q_shape[0]
            or k_shape[2] != q_shape[2]):
        raise ValueError("Q and K must be [rows, heads, dim] with equal rows and dim")
    rows, q_heads, dim = q_shape
    if q_heads < 1 or k_shape[1] < 1 or dim < 2 or dim % 2 or dim > 512:
        raise ValueError("heads must be positive and head dim even, at most 512")
    codes = _launch.DTYPE_CODES
    dtype, weight_dtype = q.dtype, q_weight.dtype
    if dtype not in codes or k.dtype != dtype:
        raise ValueError("Q and K must share one of BF16, FP16 and FP32")
    if (q_weight.shape != (dim,) or k_weight.shape != (dim,) or weight_dtype not in codes
            or k_weight.dtype != weight_dtype):
        raise ValueError("norm weights must be [dim] vectors of one floating dtype")
    if positions.shape != (rows,) or positions.dtype not in _INDEX:
        raise ValueError("positions must be an integer [rows] vector")
    if (len(cache_shape) not in (2, 3) or cache_shape[-1] != dim or cache_shape[0] < 1
            or (len(cache_shape) == 3 and cache_shape[1] != 1) or cache.dtype not in codes):
        raise ValueError("cos/sin cache must be floating [positions, dim] or [positions, 1, dim]")
    if q.stride(2) != 1 or k.stride(2) != 1 or cache.stride(-1) != 1 \
            or q_weight.stride(0) != 1 or k_weight.stride(0) != 1:
        raise ValueError("head dimensions, weights and cache rows must be contiguous")
    if not eps >= 0:
        raise ValueError("eps must not be negative")
    device = q.device
    if (not q.is_cuda or k.device != device or q_weight.device != device
            or k_weight.device != device or positions.device != device
            or cache.device != device):
        raise ValueError("head norm and rotation require CUDA tensors on one device")


def _output(out, like, name):
    if out is None:
        return torch.empty(like.shape, dtype=like.dtype, device=like.device)
    if out is like and like.stride(2) == 1:
        return out
    if (out.shape != like.shape or out.dtype != like.dtype or out.device != like.device
            or out.stride(2) != 1):
        raise ValueError(f"{name} must match its input's shape, dtype and device")
    return out


def qk_norm_rope(q, k, q_weight, k_weight, positions, cos_sin_cache, eps=1e-6, *, q_out=None,
                 k_out=None):
    """Normed and rotated (Q, K), both [rows, heads, dim] in the operand type.

    ``out = rotate(x * rsqrt(mean(x^2) + eps) * weight)`` per head, in fp32 with one rounding;
    the rotation pairs element d with d + dim/2, cache rows hold ``[cos | sin]`` halves.
    ``q_out`` / ``k_out`` may be the inputs themselves (in place) but not overlap them otherwise.
    """
    _check(q, k, q_weight, k_weight, positions, cos_sin_cache, eps)
    q_out = _output(q_out, q, "q_out")
    k_out = _output(k_out, k, "k_out")
    from . import ops

    if ops.compiling():
        torch.ops.jetspec_b200.qk_norm_rope_(q, k, q_weight, k_weight, positions, cos_sin_cache,
                                             float(eps), q_out, k_out)
    else:
        _launch_norm(q, k, q_weight, k_weight, positions, cos_sin_cache, eps, q_out, k_out)
    return q_out, k_out


def qk_norm_rope_store(q, k, v, q_weight, k_weight, positions, cos_sin_cache, k_pool, v_pool,
                       slot_mapping, eps=1e-6, *, k_scale=None, v_scale=None, q_out=None):
    """Normed and rotated Q; rotated K and V written to their cache slots in the same launch.

    Pools are [pages, page_size, kv_heads, dim] of the operand type, or e4m3 with the layer's
    ``k_scale`` / ``v_scale`` (see ``fp8_cache``).  Rows with slot -1 are not written; the
    caller guarantees unique slots.  ``q_out`` may be ``q`` (in place).
    """
    _check(q, k, q_weight, k_weight, positions, cos_sin_cache, eps)
    k_shape, dtype, pool_shape = k.shape, q.dtype, k_pool.shape
    if v.shape != k_shape or v.dtype != dtype or v.stride(2) != 1:
        raise ValueError("V must match K's shape and dtype with a contiguous head dimension")
    if slot_mapping.shape != positions.shape or slot_mapping.dtype not in _INDEX:
        raise ValueError("slots must be an integer [rows] vector")
    if (len(pool_shape) != 4 or v_pool.shape != pool_shape or pool_shape[2:] != k_shape[1:]
            or pool_shape[0] < 1 or pool_shape[1] < 1):
        raise ValueError("KV pools must be [pages, page_size, kv_heads, dim]")
    if k_pool.stride(3) != 1 or v_pool.stride(3) != 1:
        raise ValueError("KV pools need a contiguous head dimension")
    if k_pool.dtype == CODE_DTYPE:
        check_layer(k_pool, v_pool, k_scale, v_scale)
    elif k_pool.dtype != dtype or v_pool.dtype != dtype:
        raise ValueError("KV pools must have the operand dtype, or hold e4m3 codes with scales")
    elif k_scale is not None or v_scale is not None:
        raise ValueError("scales belong to 8-bit pools")
    device = q.device
    if (v.device != device or slot_mapping.device != device or k_pool.device != device
            or v_pool.device != device):
        raise ValueError("the cache write requires CUDA tensors on one device")
    q_out = _output(q_out, q, "q_out")
    from . import ops

    if ops.compiling():
        torch.ops.jetspec_b200.qk_norm_rope_store_(
            q, k, v, q_weight, k_weight, positions, cos_sin_cache, k_pool, v_pool, slot_mapping,
            float(eps), k_scale, v_scale, q_out)
    else:
        _launch_norm(q, k, q_weight, k_weight, positions, cos_sin_cache, eps, q_out, None, v,
                     k_pool, v_pool, slot_mapping, k_scale, v_scale)
    return q_out


def _launch_norm(q, k, q_weight, k_weight, positions, cache, eps, q_out, k_out, v=None,
                 k_pool=None, v_pool=None, slots=None, k_scale=None, v_scale=None) -> None:
    """jt_qk_norm_rope_launch on the current stream (validated arguments)."""
    lib = _lib.load_library()
    codes = _launch.DTYPE_CODES
    rows, q_heads, dim = q.shape
    qs, ks, qo = q.stride(), k.stride(), q_out.stride()
    if k_pool is None:
        store, ko = _STORE_NONE, k_out.stride()
        ptrs = (None,) * 5
        out_k, pages, page_size = k_out.data_ptr(), 0, 0
        vs = kp = vp = kss = vss = (0, 0, 0)
        slot_ptr, slot_stride, slot64 = None, 0, 0
    else:
        ko, out_k = (0, 0), None
        pages, page_size = k_pool.shape[0], k_pool.shape[1]
        vs, kp, vp = v.stride(), k_pool.stride(), v_pool.stride()
        if k_scale is None:
            store, kss, vss = _STORE_SAME, (0, 0), (0, 0)
            scale_ptrs = (None, None)
        else:
            store, kss, vss = _STORE_FP8, k_scale.stride(), v_scale.stride()
            scale_ptrs = (k_scale.data_ptr(), v_scale.data_ptr())
        ptrs = (v.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr()) + scale_ptrs
        slot_ptr, slot_stride = slots.data_ptr(), slots.stride(0)
        slot64 = int(slots.dtype == torch.int64)
    p = _lib.JtQkNormRopeParams(
        q.data_ptr(), k.data_ptr(), ptrs[0], q_weight.data_ptr(), k_weight.data_ptr(),
        positions.data_ptr(), cache.data_ptr(), slot_ptr, q_out.data_ptr(), out_k, ptrs[1],
        ptrs[2], ptrs[3], ptrs[4], pages, cache.shape[0], qs[0], qs[1], ks[0], ks[1], vs[0],
        vs[1], qo[0], qo[1], ko[0], ko[1], kp[0], kp[1], kp[2], vp[0], vp[1], vp[2], kss[0],
        kss[1], vss[0], vss[1], positions.stride(0), slot_stride, cache.stride(0), eps, rows,
        q_heads, k.shape[1], dim, page_size, codes[q.dtype], codes[q_weight.dtype],
        codes[cache.dtype], store, int(positions.dtype == torch.int64), slot64)
    _lib.check(lib.jt_qk_norm_rope_launch(ctypes.byref(p), _launch.raw_stream(q.device)))
