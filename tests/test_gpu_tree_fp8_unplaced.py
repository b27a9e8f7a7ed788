"""Keys without a place in the pool (a page or slot out of range, as build_request_maps leaves them
when the free list is short) are left out of the attention: its value is that of the keys that
have one, whatever lies in page 0.  Tolerance as in test_gpu_tree_fp8, over the keys left.
"""
from __future__ import annotations

import pytest
import torch

import jetspec_b200 as jb

from test_gpu_tree_fp8 import DEVICE, Case

pytestmark = pytest.mark.gpu


class Holes(Case):
    """A case with entries of its page tables and node slots put out of range."""

    def __init__(self, prefixes, counts, *, bad_pages=(), bad_nodes=(), value=-1, **kwargs):
        super().__init__(prefixes, counts, num_blocks=256, **kwargs)
        block = self.batch.block_size
        self.bad_pages, self.bad_nodes = set(bad_pages), set(bad_nodes)
        live = {p for table in self.batch.block_tables for p in table}
        live |= {int(s) // block for s in self.meta.tree_slots}
        if 0 in live:  # page 0 changes places with a free one
            free = next(p for p in range(self.k.shape[0]) if p not in live)
            for pool in (self.k, self.v, self.ks, self.vs):
                raw = pool.view(torch.uint8)
                raw[free] = raw[0]
            self.batch.block_tables = [[free if p == 0 else p for p in t]
                                       for t in self.batch.block_tables]
            table = self.meta.block_tables
            table[table == 0] = free
            slots = self.meta.tree_slots
            slots[slots < block] += free * block
        # Page 0: the largest codes, NaN scales.
        for pool, byte in ((self.k, 0x7E), (self.v, 0x7E), (self.ks, 255), (self.vs, 255)):
            pool.view(torch.uint8)[0] = byte
        for r, column in self.bad_pages:
            self.meta.block_tables[r, column] = value
        offsets = self.meta.cu_seqlens_q.tolist()
        self.true_slots = self.meta.tree_slots.clone()
        for r, node in self.bad_nodes:
            self.meta.tree_slots[offsets[r] + node] = value * block

    def exact(self, requests=None):
        b, m = self.batch, self.meta
        out = torch.zeros(self.q.shape, dtype=torch.float64, device=DEVICE)
        spread, shift = torch.zeros_like(out), torch.zeros_like(out[..., :1])
        offsets, biases = m.cu_seqlens_q.tolist(), m.qq_bias_offsets.tolist()
        for r in range(b.num_requests):
            lo, hi, p = offsets[r], offsets[r + 1], b.prefix_lens[r]
            t = hi - lo
            pos = torch.arange(p, device=DEVICE)
            table = torch.tensor(b.block_tables[r] or [0], device=DEVICE)
            slots = torch.cat([table[pos // b.block_size] * b.block_size + pos % b.block_size,
                               self.true_slots[lo:hi]])
            placed = torch.tensor([(r, int(x) // b.block_size) not in self.bad_pages
                                   for x in range(p)]
                                  + [(r, n) not in self.bad_nodes for n in range(t)], device=DEVICE)
            seen = torch.ones((t, p + t), dtype=torch.bool, device=DEVICE)
            seen[:, p:] = (m.qq_bias[biases[r]:biases[r + 1]].view(t, t) == 0).tril()
            seen &= placed
            k, v = self.rows(self.k, self.ks, slots), self.rows(self.v, self.vs, slots)
            q = self.q[lo:hi].double().unflatten(1, (-1, b.groups))
            for h in range(k.shape[1]):
                s = torch.einsum("tgd,kd->tgk", q[:, h], k[:, h]) * self.scale
                s = torch.where(seen[:, None], s, -torch.inf)
                top = s.amax(-1, keepdim=True)
                w = torch.exp(s - torch.where(torch.isinf(top), 0.0, top))
                w = torch.where(seen[:, None], w, 0.0)
                w = w / torch.where(w.sum(-1, keepdim=True) == 0, 1.0, w.sum(-1, keepdim=True))
                rows = slice(h * b.groups, (h + 1) * b.groups)
                out[lo:hi, rows] = torch.einsum("tgk,kd->tgd", w, v[:, h])
                spread[lo:hi, rows] = torch.einsum("tgk,kd->tgd", w, v[:, h].abs())
                kk = torch.where(seen[:, None], k[:, h].abs().sum(-1), 0.0).amax(-1)
                shift[lo:hi, rows] = (self.scale * 2.0 ** -17 * q[:, h].abs().amax(-1)
                                      * kk)[..., None]
        return out, spread, shift

    def check(self, requests=None, **kwargs):
        jb.read_device_errors()
        got = self.run(**kwargs)
        assert jb.read_device_errors() == 1
        run, self.run = self.run, lambda **kw: got
        try:
            return super().check()
        finally:
            self.run = run


SIZES = [[1], [4], [5], [40], [130]]


@pytest.mark.parametrize("counts", SIZES)
@pytest.mark.parametrize("block", [16, 32, 64, 128, 256, 100])
@pytest.mark.parametrize("value", [-1, 10 ** 6])
def test_pages_out_of_range(counts, block, value):
    prefix = 1100
    last = -(-prefix // block) - 1
    for bad in ([0], [last], [1, last // 2]):
        Holes([prefix], counts, block=block, value=value, seed=block,
              bad_pages=[(0, c) for c in bad]).check()


@pytest.mark.parametrize("counts", [[2, 1, 3], [40, 3, 64]])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("out", [None, torch.float32])
def test_types_and_mixed_batches(counts, dtype, out):
    Holes([1000, 300, 4000], counts, dtype=dtype, seed=3,
          bad_pages=[(0, 1), (2, 0), (2, 9), (2, 15)]).check(output_dtype=out)


@pytest.mark.parametrize("counts", [[4], [40]])
def test_nodes_out_of_range(counts):
    Holes([300], counts, seed=4, bad_nodes=[(0, 1), (0, 3)]).check()


@pytest.mark.parametrize("counts", [[1], [3], [40], [130]])
@pytest.mark.parametrize("block", [64, 256, 100])
def test_no_key_left(counts, block):
    """Every page missing: the tree alone; its nodes missing too: zeros."""
    pages = [(0, c) for c in range(-(-600 // block))]
    Holes([600], counts, block=block, seed=5, bad_pages=pages).check()
    nodes = [(0, n) for n in range(counts[0])]
    got = Holes([600], counts, block=block, seed=5, bad_pages=pages, bad_nodes=nodes).check()
    assert (got == 0).all()


@pytest.mark.parametrize("counts", [[1], [64]])
def test_missing_pages_of_a_request_cut_between_multiprocessors(counts):
    Holes([30011], counts, seed=6, bad_pages=[(0, c) for c in range(0, 117, 5)]).check()
