"""The C entry of the attention over the 8-bit cache refuses bad arguments before any CUDA call."""
from __future__ import annotations

import ctypes

import pytest

from jetspec_b200 import _lib


@pytest.fixture(scope="module")
def lib():
    return _lib.load_library()


def params(**over):
    p = _lib.JtTreeAttnFp8Params()
    values = dict(num_requests=2, total_queries=5, num_kv_heads=2, groups=4, head_dim=64,
                  block_size=16, num_blocks=8, table_width=3, dtype=_lib.JT_BF16,
                  out_dtype=_lib.JT_BF16, scale=0.125)
    for name in ("out q k_pool v_pool k_scale v_scale cu_seqlens_q query_to_request "
                 "query_local_row prefix_lens node_counts block_tables tree_slots qq_bias "
                 "qq_bias_offsets workspace").split():
        values[name] = 4096
    for name in ("q_stride0 q_stride1 out_stride0 out_stride1 k_stride0 k_stride1 k_stride2 "
                 "v_stride0 v_stride1 v_stride2 ks_stride0 ks_stride1 vs_stride0 "
                 "vs_stride1").split():
        values[name] = 64
    for name, value in {**values, **over}.items():
        setattr(p, name, value)
    return p


@pytest.mark.parametrize("over,status,words", [
    (dict(num_requests=0), "JT_ERR_INVALID", "geometry"),
    (dict(groups=129), "JT_ERR_INVALID", "geometry"),
    (dict(num_blocks=1 << 31), "JT_ERR_INVALID", "geometry"),
    (dict(table_width=0), "JT_ERR_INVALID", "geometry"),
    (dict(head_dim=72), "JT_ERR_UNSUPPORTED", "head_dim 72"),
    (dict(head_dim=144), "JT_ERR_UNSUPPORTED", "head_dim 144"),
    (dict(dtype=_lib.JT_F32), "JT_ERR_UNSUPPORTED", "bf16 or f16"),
    (dict(out_dtype=_lib.JT_F16), "JT_ERR_INVALID", "output dtype"),
    (dict(scale=0.0), "JT_ERR_INVALID", "scale"),
    (dict(scale=float("nan")), "JT_ERR_INVALID", "scale"),
    (dict(v_scale=None), "JT_ERR_INVALID", "null"),
    (dict(q=4100), "JT_ERR_INVALID", "16 bytes"),
    (dict(k_stride1=72), "JT_ERR_INVALID", "16 bytes"),
    (dict(q_stride1=4), "JT_ERR_INVALID", "16 bytes"),
    (dict(workspace_bytes=100), "JT_ERR_WORKSPACE", "workspace"),
    (dict(workspace=None, workspace_bytes=1 << 40), "JT_ERR_WORKSPACE", "workspace"),
    (dict(workspace=4104, workspace_bytes=1 << 40), "JT_ERR_WORKSPACE", "workspace"),
])
def test_refusals(lib, over, status, words):
    p = params(**over)
    assert lib.jt_tree_attn_fp8_launch(ctypes.byref(p), None) == getattr(_lib, status)
    assert words in lib.jt_last_error().decode()


def test_null_params(lib):
    assert lib.jt_tree_attn_fp8_launch(None, None) == _lib.JT_ERR_INVALID


def test_workspace_size(lib):
    size = lib.jt_tree_attn_fp8_workspace_size
    assert size(0, 5, 2, 4, 64) == -1 and size(1, 5, 2, 0, 64) == -1
    assert 0 < size(1, 1, 1, 1, 64) < size(4, 4096, 8, 4, 128)
