"""Rounds of speculative verification over the 8-bit paged KV cache.

    python examples/fp8_verify_rounds.py

The operators in the order in which a serving loop uses them, with random projections in the
place of a model:

* prefill: ``build_request_maps`` hands out pages and slots for the prompts, and
  ``qk_norm_rope_store`` norms and rotates Q and K and writes K / V in 8 bits;
* a verification round: every request's draft tree goes into scratch slots,
  ``packed_tree_attention_fp8`` attends to prefix and ancestors; the accepted path gets slots
  from ``build_request_maps`` and is moved there by ``copy_accepted_kv_fp8``;
* a decode round: the same on trees of one node.

Each round's attention is compared with a softmax in fp32 over the cache's dequantised rows.
"""
from __future__ import annotations

import sys
from pathlib import Path

import numpy as np
import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
import __graft_entry__  # noqa: E402

jb = __graft_entry__.load_package()


class Rounds:
    def __init__(self, requests=4, layers=2, kv_heads=8, groups=4, dim=128, block=256,
                 longest=1500, seed=0, device="cuda"):
        self.rng = np.random.default_rng(seed)
        self.gen = torch.Generator(device=device).manual_seed(seed)
        self.device, self.layers, self.block = device, layers, block
        self.kv_heads, self.groups, self.dim = kv_heads, groups, dim
        self.cached = self.rng.integers(1, longest + 1, size=requests)
        width = -(-(longest + 256) // block)
        self.arena = list(range(requests))                    # a scratch page per request
        pages = requests * (width + 1)
        self.free = torch.arange(requests, pages, dtype=torch.int32, device=device)
        self.tables = torch.full((requests, width), -1, dtype=torch.int32, device=device)
        self.pool, self.scale = jb.alloc_fp8_kv_cache(layers, pages, block, kv_heads, dim, device)
        self.weights = [1 + 0.1 * self.randn(dim) for _ in range(2)]
        angle = (torch.arange(longest + 512, device=device)[:, None]
                 * 10000.0 ** (-torch.arange(0, dim, 2, device=device) / dim))
        self.cos_sin = torch.cat([angle.cos(), angle.sin()], dim=1)

    def randn(self, *shape):
        return torch.randn(shape, generator=self.gen, device=self.device, dtype=torch.bfloat16)

    def ints(self, values):
        return torch.tensor(np.asarray(values), dtype=torch.int32, device=self.device)

    def maps(self, cached, new):
        """Slots of the round's new tokens; the pages it takes leave the free list."""
        maps = jb.build_request_maps(self.tables, self.ints(cached), self.ints(new), self.free,
                                     self.block, max_tokens=int(np.sum(new)))
        self.free = self.free[int(maps.pages_taken):]
        return maps

    def store(self, layer, positions, slots):
        """A layer's Q, normed and rotated; its K and V are in the cache."""
        rows = positions.shape[0]
        qkv = self.randn(rows, (self.groups + 2) * self.kv_heads, self.dim)
        q, k, v = qkv.split((self.groups * self.kv_heads, self.kv_heads, self.kv_heads), dim=1)
        return jb.qk_norm_rope_store(q, k, v, *self.weights, positions, self.cos_sin,
                                     *self.layer(layer)[:2], slots, k_scale=self.scale[0, layer],
                                     v_scale=self.scale[1, layer])

    def layer(self, layer):
        return (self.pool[0, layer], self.pool[1, layer], self.scale[0, layer],
                self.scale[1, layer])

    def prefill(self):
        maps = self.maps(np.zeros_like(self.cached), self.cached)
        for layer in range(self.layers):
            self.store(layer, maps.positions, maps.slot_mapping)

    def verify(self, nodes):
        """One round on trees of up to ``nodes`` nodes; the attention's largest error."""
        parents, depths = [], []
        for _ in self.cached:
            tree = [-1] + [int(self.rng.integers(0, j)) for j in
                           range(1, int(self.rng.integers(1, nodes + 1)))]
            depth = [0]
            for p in tree[1:]:
                depth.append(depth[p] + 1)
            parents.append(tree)
            depths += depth
        used = -(-self.cached // self.block)
        owned = [row[:n] for row, n in zip(self.tables.tolist(), used)]
        meta = jb.PackedTreeMetadata.from_parents_device(
            self.cached, owned, parents, self.arena, self.block, device=self.device)
        positions = meta.prefix_lens[meta.query_to_request.long()] + self.ints(depths)
        worst = 0.0
        for layer in range(self.layers):
            q = self.store(layer, positions, meta.tree_slots)
            out = jb.packed_tree_attention_fp8(q, *self.layer(layer), meta, self.dim ** -0.5,
                                               self.groups)
            worst = max(worst, self.error(layer, q, out, meta))
        # Accept the path to a random node, and commit it behind the prefix.
        paths = []
        for tree in parents:
            node, path = int(self.rng.integers(0, len(tree))), []
            while node >= 0:
                path.append(node)
                node = tree[node]
            paths.append(path[::-1])
        starts = np.cumsum([0] + [len(t) for t in parents[:-1]])
        source = meta.tree_slots[self.ints(np.concatenate(
            [s + np.array(p) for s, p in zip(starts, paths)])).long()]
        accepted = np.array([len(p) for p in paths])
        maps = self.maps(self.cached, accepted)
        before = self.rows(source)
        jb.copy_accepted_kv_fp8(self.pool, self.scale, source, maps.slot_mapping, self.block)
        if not torch.equal(self.rows(maps.slot_mapping), before):
            raise AssertionError("the commit changed a row")
        self.cached = self.cached + accepted
        return worst

    def rows(self, slots):
        """Dequantised rows [2, layers, slots, kv_heads, dim]."""
        values = jb.dequantize_kv(self.pool, self.scale, torch.float32)
        return values[:, :, slots // self.block, slots % self.block]

    def error(self, layer, q, out, meta):
        """Largest error over sum w |v|, the attention taken in fp32 over the cache's values."""
        worst, starts, biases = 0.0, meta.cu_seqlens_q.tolist(), meta.qq_bias_offsets.tolist()
        for r, prefix in enumerate(self.cached):
            lo, hi = starts[r], starts[r + 1]
            pos = torch.arange(int(prefix), device=self.device)
            slots = torch.cat([self.tables[r].long()[pos // self.block] * self.block
                               + pos % self.block, meta.tree_slots[lo:hi]])
            k, v = self.rows(slots)[:, layer]
            k, v = (x.repeat_interleave(self.groups, dim=1) for x in (k, v))
            bias = torch.zeros((hi - lo, slots.numel()), device=self.device)
            bias[:, int(prefix):] = meta.qq_bias[biases[r]:biases[r + 1]].view(hi - lo, hi - lo)
            scores = torch.einsum("thd,khd->htk", q[lo:hi].float(), k) * self.dim ** -0.5 + bias
            w = scores.softmax(-1)
            want = torch.einsum("htk,khd->thd", w, v)
            spread = torch.einsum("htk,khd->thd", w, v.abs())
            worst = max(worst, ((out[lo:hi].float() - want).abs() / spread).max().item())
        return worst


def main(rounds=3, nodes=24, **sizes):
    """Largest error of any round (P and the output are rounded to bf16: below 2^-6)."""
    state = Rounds(**sizes)
    state.prefill()
    worst = max([state.verify(nodes) for _ in range(rounds)] + [state.verify(1)])
    if jb.read_device_errors():
        raise AssertionError("device error word set")
    return worst, state


if __name__ == "__main__":
    error, state = main()
    print(f"largest attention error {error:.2e} of sum w |v|; cached tokens {state.cached.tolist()}")
