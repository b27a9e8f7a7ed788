"""packed_tree_attention_fp8 on requests of few query rows (nodes x query heads of a KV head up
to 16), which take a kernel of their own, and on batches that mix them with larger trees.

The tolerance is test_gpu_tree_fp8's: queries kept to 2^-22 of the row's largest and weights to
f16 (2^-12; 2^-22 for FP16 and FP32 outputs) lie within its terms.
"""
from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

import jetspec_b200 as jb

from helpers import bits_equal
from test_gpu_tree_fp8 import DEVICE, Case

pytestmark = pytest.mark.gpu

EDGES = [0, 1, 15, 16, 17, 127, 128, 129, 255, 256, 257, 1000]
FIELDS = ("cu_seqlens_q", "query_to_request", "query_local_row", "prefix_lens", "node_counts",
          "block_tables", "tree_slots", "qq_bias", "qq_bias_offsets", "block_size",
          "total_queries", "num_requests", "node_counts_host")


def namespace(meta, **over):
    return SimpleNamespace(**{name: over.get(name, getattr(meta, name)) for name in FIELDS})


@pytest.mark.parametrize("groups,nodes", [(1, 1), (1, 16), (2, 8), (3, 5), (4, 1), (4, 2), (4, 4),
                                          (5, 3), (7, 1), (7, 2), (8, 1), (8, 2), (16, 1), (1, 9),
                                          (1, 17), (4, 5), (9, 2)])
def test_rows_at_tile_and_page_edges(groups, nodes):
    Case(EDGES, [nodes] * len(EDGES), kv_heads=2, groups=groups, seed=groups + nodes).check()


@pytest.mark.parametrize("dim", [16, 48, 64, 80, 128])
@pytest.mark.parametrize("block", [1, 7, 16, 32, 100, 128, 256, 512])
def test_head_dims_and_page_sizes(dim, block):
    Case([333, 0, 1, 640], [3, 2, 1, 4], dim=dim, block=block, seed=dim + block).check()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("out", [None, torch.float32])
@pytest.mark.parametrize("nodes", [1, 3])
def test_types(dtype, out, nodes):
    case = Case([1000, 129], [nodes, nodes], dtype=dtype, seed=11)
    assert case.check(output_dtype=out).dtype == (out or dtype)


@pytest.mark.parametrize("nodes", [1, 2, 4])
def test_requests_cut_over_many_multiprocessors(nodes):
    Case([30011, 20], [nodes, 1], kv_heads=3, seed=nodes).check()


def test_large_and_small_magnitudes():
    Case([700], [2], q_std=20.0, v_std=1e-20, seed=3).check()
    Case([700], [2], q_std=1e-3, v_std=1e20, seed=4).check(output_dtype=torch.float32)
    Case([700], [1], q_std=30.0, seed=5, dtype=torch.float16).check(output_dtype=torch.float32)


def test_values_of_very_different_scales():
    """Value rows 2^-90 to 2^90 of each other: the exponents P carries."""
    case = Case([500], [2], seed=6)
    byte = case.vs.view(torch.uint8)
    byte[:] = torch.where(byte == 255, byte, (byte.int() + 30 * (byte.int() % 7 - 3)).clamp(1, 250)
                          .to(torch.uint8))
    case.check(output_dtype=torch.float32)


@pytest.mark.parametrize("counts", [[1, 64, 2, 130, 4, 5], [4, 5], [16, 1, 1, 1]])
def test_mixed_batches_and_unknown_counts(counts):
    case = Case([300 * i + 7 for i in range(len(counts))], counts, seed=len(counts))
    want = case.check()
    case.meta = namespace(case.meta, node_counts_host=None)
    assert bits_equal(case.check(), want)


def test_off_branch_rows_never_arrive():
    case = Case([130], [16], groups=1, seed=9)
    want = case.check()
    block = case.batch.block_size
    seen = case.meta.qq_bias.view(16, 16) == 0
    for node, byte in ((3, 255), (6, 254)):
        slot = int(case.meta.tree_slots[node])
        for scale in (case.ks, case.vs):
            scale.view(torch.uint8)[slot // block, :, slot % block] = byte
    for pool, code in ((case.k, 0x7F), (case.v, 0xFF)):
        slot = int(case.meta.tree_slots[3])
        pool.view(torch.uint8)[slot // block, slot % block] = code
    got = case.run()
    apart = ~(seen[:, 3] | seen[:, 6])
    assert apart.any()
    assert bits_equal(got[apart], want[apart])
    assert torch.isnan(got[seen[:, 3]]).all()


def test_a_nan_row_in_the_prefix_reaches_every_row():
    case = Case([300, 200], [2, 4], seed=10)
    page = case.batch.block_tables[0][1]
    case.ks.view(torch.uint8)[page, 0, 3] = 255
    got = case.check()
    groups = case.batch.groups
    assert torch.isnan(got[:2, :groups]).all()
    assert torch.isfinite(got[:2, groups:]).all() and torch.isfinite(got[2:]).all()


def test_non_finite_queries_stay_in_their_rows():
    case = Case([300], [2], seed=19)
    want = case.run()
    q = case.q.clone()
    q[0, 1, 5] = float("inf")
    q[1, 3, 0] = float("nan")
    case.q = q
    got = case.run()
    assert torch.isnan(got[0, 1]).all() and torch.isnan(got[1, 3]).all()
    got[0, 1], got[1, 3] = want[0, 1], want[1, 3]
    assert bits_equal(got, want)


def test_rows_that_see_nothing_give_zeros():
    case = Case([0, 0], [4, 2], seed=12)
    case.meta.qq_bias.view(-1)[:16].view(4, 4)[2] = -torch.inf
    got = case.check()
    assert (got[2] == 0).all() and (got[3] != 0).any()


def test_repeats_are_identical_and_streams_are_respected():
    case = Case([9000, 300, 20], [1, 3, 4], seed=15)
    want = case.run()
    for _ in range(3):
        assert bits_equal(case.run(), want)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = case.run()
    torch.cuda.current_stream().wait_stream(stream)
    assert bits_equal(got, want)


def test_a_captured_decode_replays_with_larger_trees():
    """The node counts of the capture bind no replay."""
    small, large = Case([200, 900], [4, 4], seed=16), Case([150, 800], [1, 7], seed=17)
    # One set of buffers: the small batch's, then the large one's in the same places.
    bias = torch.zeros(64, dtype=torch.float32, device=DEVICE)
    width = max(small.meta.block_tables.shape[1], large.meta.block_tables.shape[1])
    table = torch.full((2, width), -1, dtype=torch.int32, device=DEVICE)
    buffers = {name: getattr(small.meta, name).clone()
               for name in FIELDS[:9] if name not in ("block_tables", "qq_bias")}
    meta = namespace(small.meta, **buffers, block_tables=table, qq_bias=bias)

    def fill(case):
        for name, buffer in buffers.items():
            buffer.copy_(getattr(case.meta, name))
        bias[:case.meta.qq_bias.numel()] = case.meta.qq_bias.view(-1)
        table[:, :case.meta.block_tables.shape[1]] = case.meta.block_tables

    def run():
        return jb.packed_tree_attention_fp8(q, large.k, large.v, large.ks, large.vs, meta,
                                            large.scale, large.batch.groups)

    q = large.q.clone()
    fill(small)
    table.clamp_(max=large.k.shape[0] - 1)
    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    fill(large)
    jb.read_device_errors()
    graph.replay()
    assert bits_equal(out, large.check())


def test_index_errors_are_flagged_and_skipped():
    case = Case([300], [1], seed=17)
    jb.read_device_errors()
    case.meta.block_tables[0, 1] = 10 ** 6
    case.run()
    assert jb.read_device_errors() & 1
