"""A round of the 8-bit cache's operators (maps, norm and store, tree attention, commit) under
torch.compile (no graph break) and in a CUDA graph: bit for bit the eager results."""
from __future__ import annotations

import pytest
import torch

import jetspec_b200 as jb

from helpers import bits_equal
from test_gpu_tree_fp8 import DEVICE, Case

pytestmark = pytest.mark.gpu


class Round:
    def __init__(self, counts):
        case = self.case = Case([200, 700], counts, seed=sum(counts))
        gen = torch.Generator(device=DEVICE).manual_seed(1)
        total, kv_heads, dim = sum(counts), case.batch.num_kv_heads, case.batch.head_dim
        heads = kv_heads * (case.batch.groups + 2)
        self.qkv = torch.randn((total, heads, dim), generator=gen, device=DEVICE).bfloat16()
        self.weights = [torch.randn(dim, generator=gen, device=DEVICE).bfloat16() for _ in "qk"]
        self.cos_sin = torch.randn((1024, dim), generator=gen, device=DEVICE)
        self.cached = torch.tensor([200, 700], dtype=torch.int32, device=DEVICE)
        self.fresh = torch.tensor([2, 1], dtype=torch.int32, device=DEVICE)
        self.positions = case.meta.query_local_row + self.cached[case.meta.query_to_request.long()]
        self.free = torch.arange(2, dtype=torch.int32, device=DEVICE)
        self.source = case.meta.tree_slots[torch.tensor([0, 1, counts[0]], device=DEVICE)]
        page = torch.tensor([case.batch.block_tables[0][-1], case.batch.block_tables[0][-1],
                             case.batch.block_tables[1][-1]], device=DEVICE)
        self.target = page * 256 + torch.tensor([200, 201, 700 % 256], device=DEVICE)

    def state(self):
        return tuple(x.view(torch.uint8).clone().view(x.dtype) for x in self.case.cache)

    def step(self, qkv, pool, scale):
        case, m = self.case, self.case.meta
        kv_heads, groups = case.batch.num_kv_heads, case.batch.groups
        maps = jb.build_request_maps(m.block_tables, self.cached, self.fresh, self.free, 256,
                                     max_tokens=3)
        q, k, v = qkv.split((kv_heads * groups, kv_heads, kv_heads), dim=1)
        q = jb.qk_norm_rope_store(q, k, v, *self.weights, self.positions, self.cos_sin, pool[0, 1],
                                  pool[1, 1], m.tree_slots, k_scale=scale[0, 1],
                                  v_scale=scale[1, 1])
        out = jb.packed_tree_attention_fp8(q, pool[0, 1], pool[1, 1], scale[0, 1], scale[1, 1], m,
                                           case.scale, groups)
        jb.copy_accepted_kv_fp8(pool, scale, self.source, self.target, 256)
        return out, maps.slot_mapping, maps.positions


@pytest.mark.parametrize("counts", [[4, 3], [4, 20], [64, 33]])
def test_compiled_round_matches_eager(counts):
    r = Round(counts)
    pool, scale = r.state()
    want = r.step(r.qkv, pool, scale)
    got_pool, got_scale = r.state()
    got = torch.compile(r.step, fullgraph=True, backend="aot_eager")(r.qkv, got_pool, got_scale)
    for a, b in zip(got, want):
        assert bits_equal(a, b)
    assert bits_equal(got_pool.view(torch.uint8), pool.view(torch.uint8))
    assert bits_equal(got_scale.view(torch.uint8), scale.view(torch.uint8))


@pytest.mark.parametrize("counts", [[4, 3], [4, 20], [64, 33]])
def test_captured_round_matches_eager(counts):
    r = Round(counts)
    pool, scale = r.state()
    want = r.step(r.qkv, pool, scale)
    got_pool, got_scale = r.state()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = r.step(r.qkv, got_pool, got_scale)
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert bits_equal(a, b)
    assert bits_equal(got_pool.view(torch.uint8), pool.view(torch.uint8))
    assert bits_equal(got_scale.view(torch.uint8), scale.view(torch.uint8))
    assert jb.read_device_errors() == 0
