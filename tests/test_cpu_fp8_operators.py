"""Refusals of the 8-bit cache operators, and the C ABI's own checks, without a GPU."""
from __future__ import annotations

import ctypes

import pytest
import torch

import jetspec_b200 as jb
from jetspec_b200 import _lib


@pytest.fixture(scope="module")
def lib():
    return _lib.load_library()


def _maps_args(**over):
    a = dict(block_tables=torch.zeros((2, 4), dtype=torch.int32),
             cached_lens=torch.zeros(2, dtype=torch.int32),
             new_lens=torch.ones(2, dtype=torch.int32),
             free_pages=torch.arange(8, dtype=torch.int32), block_size=16, max_tokens=8)
    a.update(over)
    return a


@pytest.mark.parametrize("over,match", [
    (dict(new_lens=torch.ones(3, dtype=torch.int32)), "equally sized"),
    (dict(block_tables=torch.zeros(4, dtype=torch.int32)), "requests, width"),
    (dict(free_pages=torch.zeros((2, 2), dtype=torch.int32)), "vector"),
    (dict(block_size=0), "block size"),
    (dict(max_tokens=-1), "capacity"),
    (dict(cached_lens=torch.zeros(2, dtype=torch.int64)), "int32"),
    ({}, "CUDA"),
])
def test_request_maps_refusals(over, match):
    with pytest.raises(ValueError, match=match):
        jb.build_request_maps(**_maps_args(**over))


def _norm_args(**over):
    a = dict(q=torch.zeros(3, 4, 64), k=torch.zeros(3, 2, 64), q_weight=torch.ones(64),
             k_weight=torch.ones(64), positions=torch.zeros(3, dtype=torch.int64),
             cos_sin_cache=torch.zeros(10, 64))
    a.update(over)
    return a


@pytest.mark.parametrize("over,match", [
    (dict(k=torch.zeros(2, 2, 64)), "equal rows"),
    (dict(q=torch.zeros(3, 4, 63), k=torch.zeros(3, 2, 63)), "even"),
    (dict(q=torch.zeros(3, 4, 64).bfloat16()), "share"),
    (dict(q_weight=torch.ones(32)), "weights"),
    (dict(positions=torch.zeros(3)), "positions"),
    (dict(cos_sin_cache=torch.zeros(10, 32)), "cos/sin"),
    (dict(q=torch.zeros(3, 64, 4).transpose(1, 2)), "contiguous"),
    (dict(eps=-1.0), "eps"),
    ({}, "CUDA"),
])
def test_norm_refusals(over, match):
    with pytest.raises(ValueError, match=match):
        jb.qk_norm_rope(**_norm_args(**over))


def test_commit_refusals():
    pool, scale = jb.alloc_fp8_kv_cache(1, 2, 16, 2, 64, "cpu")
    one = torch.zeros(1, dtype=torch.int64)
    with pytest.raises(ValueError, match="lengths differ"):
        jb.copy_accepted_kv_fp8(pool, scale, one, torch.zeros(2, dtype=torch.int64), 16)
    with pytest.raises(ValueError, match="one-dimensional"):
        jb.copy_accepted_kv_fp8(pool, scale, one[None], one, 16)
    with pytest.raises(ValueError, match="KV pool must be"):
        jb.copy_accepted_kv_fp8(pool, scale, one, one, 32)
    with pytest.raises(ValueError, match="e4m3"):
        jb.copy_accepted_kv_fp8(pool.view(torch.uint8), scale, one, one, 16)
    with pytest.raises(ValueError, match="KV scales"):
        jb.copy_accepted_kv_fp8(pool, scale[..., :8], one, one, 16)
    with pytest.raises(ValueError, match="CUDA"):
        jb.copy_accepted_kv_fp8(pool, scale, one, one, 16)
    assert jb.copy_accepted_kv_fp8(pool, scale, one[:0], one[:0], 16) == 0


def test_dequantize_and_layout():
    pool, scale = jb.alloc_fp8_kv_cache(2, 3, 16, 2, 64, "cpu")
    assert pool.shape == (2, 2, 3, 16, 2, 64) and scale.shape == (2, 2, 3, 2, 16)
    pool[0, 1, 2, 5, 1] = torch.full((64,), 3.0).to(pool.dtype)
    scale.view(torch.uint8)[0, 1, 2, 1, 5] = 129
    scale.view(torch.uint8)[0, 1, 2, 0, 5] = 255
    values = jb.dequantize_kv(pool, scale)
    assert values.dtype == torch.bfloat16
    assert (values[0, 1, 2, 5, 1] == 12).all() and torch.isnan(values[0, 1, 2, 5, 0]).all()
    with pytest.raises(ValueError):
        jb.alloc_fp8_kv_cache(0, 3, 16, 2, 64, "cpu")
    with pytest.raises(ValueError):
        jb.dequantize_kv(pool[0], scale)


def test_c_abi_checks_precede_the_device(lib):
    for launch in (lib.jt_request_maps_launch, lib.jt_qk_norm_rope_launch,
                   lib.jt_kv_fp8_commit_launch):
        assert launch(None, None) == _lib.JT_ERR_INVALID
    maps = _lib.JtRequestMapsParams()
    maps.num_requests, maps.block_size, maps.table_width, maps.table_stride0 = 1, 16, 4, 3
    assert lib.jt_request_maps_launch(ctypes.byref(maps), None) == _lib.JT_ERR_INVALID
    maps.table_stride0 = 4
    assert lib.jt_request_maps_launch(ctypes.byref(maps), None) == _lib.JT_ERR_INVALID
    assert b"null" in lib.jt_last_error()
    norm = _lib.JtQkNormRopeParams()
    norm.rows, norm.q_heads, norm.kv_heads, norm.head_dim, norm.max_position = 1, 4, 2, 63, 9
    assert lib.jt_qk_norm_rope_launch(ctypes.byref(norm), None) == _lib.JT_ERR_INVALID
    norm.head_dim, norm.dtype = 64, 9
    assert lib.jt_qk_norm_rope_launch(ctypes.byref(norm), None) == _lib.JT_ERR_UNSUPPORTED
    norm.dtype = 0
    assert lib.jt_qk_norm_rope_launch(ctypes.byref(norm), None) == _lib.JT_ERR_INVALID
    assert b"null" in lib.jt_last_error()
    move = _lib.JtKvFp8CommitParams()
    move.num_slots, move.num_layers, move.num_kv_heads, move.head_dim = 1, 1, 1, 24
    move.block_size, move.num_blocks = 16, 4
    assert lib.jt_kv_fp8_commit_launch(ctypes.byref(move), None) == _lib.JT_ERR_INVALID
    move.head_dim, move.num_slots = 32, 10 ** 6
    assert lib.jt_kv_fp8_commit_launch(ctypes.byref(move), None) == _lib.JT_ERR_UNSUPPORTED
    assert lib.jt_kv_fp8_commit_max_slots() == 200 * 1024 // 17
